// Norm and rotation of queries and keys, storing keys and values in 4 bits, and
// reading stored tokens back.
//
// Per head vector x of D values, all in fp32:
//   y = x * (1 / sqrt(sum x^2 / D + eps)) * w
//   rotation by the token's position: (a, b) -> (a cos - b sin, b cos + a sin)
// then either rounded once (queries; keys of w4a16_qk_norm_rope) or quantised to 4
// bits in groups of G without a rounding before.  Memory bounds it: a head's
// values are read once and written once, in one launch for queries, keys and
// values together.
//
// Every operation is rounded by itself (no contraction to fma), and the squares
// are summed in one tree -- eight values of a lane by halves, then lanes by
// halves -- so a token's results are the same bits whether it comes alone or in a
// prompt, and can be reproduced by elementwise arithmetic.
//
// Queries and keys: D / 8 lanes to a head, eight consecutive values to a lane.
// A lane's eight key codes are one word of the cache.  Values: a cache word holds
// eight tokens of one value, so a workgroup quantises a chunk of tokens of one
// head into LDS and then writes words.  A word whose eight tokens are all in the
// chunk is stored whole; any other keeps the codes of its other tokens, which
// another workgroup may be writing in the same call: each changes only its own
// bits (an exclusive or with what it read of them), so the order does not matter.
#include "kv4_device.h"
#include "kv4_launch.h"

#pragma clang fp contract(off)

namespace w4a16 {
namespace {

constexpr int kThreads = 256;

struct RopeArgs {
  const uint16_t *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  uint16_t *q_out, *k_out;
  const float *cos, *sin;
  const int32_t* position;
  const uint16_t *q_weight, *k_weight;
  int32_t* pool;
  const int32_t *table, *rows;
  int tokens, positions, q_heads, kv_heads, half;   // half: rotated pairs of a head
  int table_rows, max_pages, pages, page_shift;
  int group_lanes, NG;                              // lanes of D / 8 that share a group
  int chunk, value_blocks, qk_blocks;
  float eps;
  bool interleaved, store;
};

// The lane's values, normed and rotated.  LPH lanes to a head, all of them active.
template <int LPH, bool BF16>
__device__ __forceinline__ void norm_rotate(float y[8], const RopeArgs& a, const uint16_t* w,
                                            int pos, int lane) {
  constexpr int D = 8 * LPH;
  if (w) {
    const float t0 = y[0] * y[0] + y[4] * y[4], t1 = y[1] * y[1] + y[5] * y[5];
    const float t2 = y[2] * y[2] + y[6] * y[6], t3 = y[3] * y[3] + y[7] * y[7];
    float t = (t0 + t2) + (t1 + t3);
#pragma unroll
    for (int m = LPH / 2; m; m /= 2) t = t + __shfl_xor(t, m, LPH);
    const float r = 1.0f / sqrtf(t * (1.0f / D) + a.eps);
    const u32x4 wv = load8(w + 8 * lane);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = (y[i] * r) * to_f32<BF16>((uint16_t)(wv[i / 2] >> (16 * (i & 1))));
  }
  const bool inside = (uint32_t)pos < (uint32_t)a.positions;
  const float* c = a.cos + (int64_t)(inside ? pos : 0) * a.half;
  const float* s = a.sin + (int64_t)(inside ? pos : 0) * a.half;
  const float bad = inside ? 0.0f : __builtin_nanf("");
  if (a.interleaved) {
    if (8 * lane < 2 * a.half) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float cc = c[4 * lane + i] + bad, ss = s[4 * lane + i] + bad;
        const float p = y[2 * i], q = y[2 * i + 1];
        y[2 * i] = p * cc - q * ss;
        y[2 * i + 1] = q * cc + p * ss;
      }
    }
  } else {
    const int hl = a.half >> 3;   // lanes of one half
    const bool low = lane < hl, turn = lane < 2 * hl;
    const int other = low ? lane + hl : turn ? lane - hl : lane;
    const int at = turn ? 8 * (low ? lane : other) : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl(y[i], other, LPH);
      const float cc = c[at + i] + bad, ss = s[at + i] + bad;
      const float r = low ? y[i] * cc - o * ss : y[i] * cc + o * ss;
      y[i] = turn ? r : y[i];
    }
  }
  if (!inside) {   // values that do not rotate as well
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] += bad;
  }
}

// Codes of a lane's eight values with the group's word; group_lanes lanes to a group.
__device__ __forceinline__ uint32_t quantise(const float y[8], int group_lanes, uint32_t code[8]) {
  // (a minimum that keeps NaN: one such value makes its whole group NaN)
  float lo = y[0], hi = y[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = __builtin_elementwise_minimum(lo, y[i]);
    hi = __builtin_elementwise_maximum(hi, y[i]);
  }
  for (int m = 1; m < group_lanes; m *= 2) {
    lo = __builtin_elementwise_minimum(lo, __shfl_xor(lo, m));
    hi = __builtin_elementwise_maximum(hi, __shfl_xor(hi, m));
  }
  const f16 s = (f16)((hi - lo) / 15.0f);
  const f16 c = (f16)(lo + 8.0f * (float)s);
  const float inv = 1.0f / (float)s;
  const bool ok = __builtin_isfinite(inv) && __builtin_isfinite((float)c) &&
                  __builtin_isfinite((float)s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float n = rintf((y[i] - (float)c) * inv);
    code[i] = ok ? (uint32_t)((int)fminf(fmaxf(n, -8.0f), 7.0f) + 8) : 8u;
  }
  return (uint32_t)as_u16(s) | (uint32_t)as_u16(c) << 16;
}

__device__ __forceinline__ void unpack8(u32x4 v, uint16_t h[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[2 * i] = (uint16_t)v[i];
    h[2 * i + 1] = (uint16_t)(v[i] >> 16);
  }
}

template <int LPH, bool BF16>
__device__ __forceinline__ void qk_part(const RopeArgs& a, int block) {
  constexpr int D = 8 * LPH;
  const int heads = a.q_heads + a.kv_heads;
  const int unit = block * (kThreads / LPH) + (int)threadIdx.x / LPH;
  const int lane = threadIdx.x % LPH;
  if (unit >= a.tokens * heads) return;
  const int t = unit / heads, h = unit - t * heads;
  const bool is_q = h < a.q_heads;
  const int kh = h - a.q_heads;
  const uint16_t* src = is_q ? a.q + t * a.q_token + h * a.q_head : a.k + t * a.k_token + kh * a.k_head;
  uint16_t half8[8];
  unpack8(load8(src + 8 * lane), half8);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = to_f32<BF16>(half8[i]);
  const int pos = a.position[t];
  norm_rotate<LPH, BF16>(y, a, is_q ? a.q_weight : a.k_weight, pos, lane);
  if (is_q || !a.store) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = (uint32_t)from_f32<BF16>(y[2 * i]) | (uint32_t)from_f32<BF16>(y[2 * i + 1]) << 16;
    uint16_t* dst = is_q ? a.q_out + ((int64_t)t * a.q_heads + h) * D
                         : a.k_out + ((int64_t)t * a.kv_heads + kh) * D;
    *reinterpret_cast<u32x4*>(dst + 8 * lane) = r;
    return;
  }
  uint32_t code[8];
  const uint32_t group = quantise(y, a.group_lanes, code);
  const int row = a.rows ? a.rows[t] : t;
  const int64_t page = pos < 0 ? -1 : kv4_page(a.table, a.table_rows, a.max_pages, a.pages, row,
                                               pos >> a.page_shift);
  if (page < 0) return;
  const int P = 1 << a.page_shift, tok = pos & (P - 1);
  const Kv4Layout f{P, D, a.NG};
  int32_t* blk = a.pool + (page * a.kv_heads + kh) * f.words();
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) w |= code[i] << kv4_shift(i);
  blk[tok * (D / 8) + kv4_key_word(lane, D)] = (int32_t)w;
  if (lane % a.group_lanes == 0)
    blk[f.key_groups() + lane / a.group_lanes * P + tok] = (int32_t)group;
}

constexpr int kChunk = 32;   // most tokens of a value chunk

template <int LPH, bool BF16>
__device__ __forceinline__ void value_part(const RopeArgs& a, int block) {
  constexpr int D = 8 * LPH;
  __shared__ uint8_t codes[kChunk][D];
  __shared__ int64_t where[kChunk];      // block of the token's page and head, in words; -1: none
  __shared__ int place[kChunk];          // token within the page
  __shared__ uint8_t member[kChunk][8];  // of the octet that a token leads: who holds which place
  __shared__ uint32_t leaders;
  const int kh = block % a.kv_heads, t0 = block / a.kv_heads * a.chunk;
  const int n = min(a.chunk, a.tokens - t0);
  const int P = 1 << a.page_shift;
  const Kv4Layout f{P, D, a.NG};
  const int lane = threadIdx.x % LPH;
  if ((int)threadIdx.x < kChunk) {
    const int c = threadIdx.x;
    int64_t at = -1;
    int tok = 0;
    if (c < n) {
      const int t = t0 + c, pos = a.position[t], row = a.rows ? a.rows[t] : t;
      const int64_t page = pos < 0 ? -1 : kv4_page(a.table, a.table_rows, a.max_pages, a.pages,
                                                   row, pos >> a.page_shift);
      tok = pos & (P - 1);
      if (page >= 0) at = (page * a.kv_heads + kh) * f.words();
    }
    where[c] = at;
    place[c] = tok;
    for (int i = 0; i < 8; ++i) member[c][i] = 255;
  }
  __syncthreads();
  for (int c = threadIdx.x / LPH; c < n; c += kThreads / LPH) {
    const uint16_t* src = a.v + (t0 + c) * a.v_token + kh * a.v_head;
    uint16_t half8[8];
    unpack8(load8(src + 8 * lane), half8);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = to_f32<BF16>(half8[i]);
    uint32_t code[8];
    const uint32_t group = quantise(y, a.group_lanes, code);
#pragma unroll
    for (int i = 0; i < 8; ++i) codes[c][8 * lane + i] = (uint8_t)code[i];
    if (where[c] >= 0 && lane % a.group_lanes == 0)
      a.pool[where[c] + f.value_groups() + lane / a.group_lanes * P + place[c]] = (int32_t)group;
  }
  if (threadIdx.x < 64) {
    // the first token of the chunk in an octet leads it
    const int c = threadIdx.x;
    bool leads = false;
    if (c < n && where[c] >= 0) {
      int lead = c;
      for (int o = 0; o < c; ++o)
        if (where[o] == where[c] && place[o] >> 3 == place[c] >> 3) {
          lead = o;
          break;
        }
      member[lead][place[c] & 7] = (uint8_t)c;
      leads = lead == c;
    }
    const uint64_t all = __ballot(leads);
    if (c == 0) leaders = (uint32_t)all;
  }
  __syncthreads();
  // a wave takes a led octet's D words in rows of 64
  const int wave = threadIdx.x / 64, l = threadIdx.x % 64;
  int turn = 0;
  for (uint32_t left = leaders; left; left &= left - 1) {
    const int c = __builtin_ctz(left);
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += 64, ++turn) {
      if ((turn & 3) != wave) continue;
      const int d = d0 + l;
      uint32_t bits = 0, mask = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int m = member[c][i];
        if (m != 255) {
          bits |= (uint32_t)codes[m][d] << kv4_shift(i);
          mask |= 15u << kv4_shift(i);
        }
      }
      uint32_t* w = reinterpret_cast<uint32_t*>(a.pool) + where[c] + f.values() +
                    (place[c] >> 3) * D + kv4_value_word(d);
      if (mask == ~0u)
        *w = bits;
      else
        atomicXor(w, (*w & mask) ^ bits);
    }
  }
}

template <int LPH, bool BF16>
__global__ __launch_bounds__(kThreads) void kv4_rope_kernel(const RopeArgs a) {
  if ((int)blockIdx.x < a.qk_blocks)
    qk_part<LPH, BF16>(a, blockIdx.x);
  else
    value_part<LPH, BF16>(a, (int)blockIdx.x - a.qk_blocks);
}

struct ReadArgs {
  const int32_t *pool, *table, *rows, *position;
  uint16_t *k, *v;
  int tokens, heads, table_rows, max_pages, pages, page_shift, group_lanes, NG;
};

template <int LPH, bool BF16>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(const ReadArgs a) {
  constexpr int D = 8 * LPH;
  const int unit = (int)blockIdx.x * (kThreads / LPH) + (int)threadIdx.x / LPH;
  const int lane = threadIdx.x % LPH;
  if (unit >= a.tokens * a.heads) return;
  const int t = unit / a.heads, h = unit - t * a.heads;
  const int pos = a.position[t], row = a.rows ? a.rows[t] : t;
  const int64_t page =
      pos < 0 ? -1 : kv4_page(a.table, a.table_rows, a.max_pages, a.pages, row, pos >> a.page_shift);
  u32x4 rk = {0, 0, 0, 0}, rv = {0, 0, 0, 0};
  if (page >= 0) {
    const int P = 1 << a.page_shift, tok = pos & (P - 1), g = lane / a.group_lanes;
    const Kv4Layout f{P, D, a.NG};
    const uint32_t* blk =
        reinterpret_cast<const uint32_t*>(a.pool) + (page * a.heads + h) * f.words();
    const uint32_t kw = blk[tok * (D / 8) + kv4_key_word(lane, D)];
    const uint32_t km = blk[f.key_groups() + g * P + tok];
    const uint32_t vm = blk[f.value_groups() + g * P + tok];
    const uint32_t* vw = blk + f.values() + (tok >> 3) * D;
    const int sh = kv4_shift(tok & 7);
    const float ks = (float)as_h((uint16_t)km), kc = (float)as_h((uint16_t)(km >> 16));
    const float vs = (float)as_h((uint16_t)vm), vc = (float)as_h((uint16_t)(vm >> 16));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = (float)((int)(kw >> kv4_shift(i) & 15) - 8) * ks + kc;
      const float y = (float)((int)(vw[kv4_value_word(8 * lane + i)] >> sh & 15) - 8) * vs + vc;
      rk[i / 2] |= (uint32_t)from_f32<BF16>(x) << (16 * (i & 1));
      rv[i / 2] |= (uint32_t)from_f32<BF16>(y) << (16 * (i & 1));
    }
  }
  *reinterpret_cast<u32x4*>(a.k + (int64_t)unit * D + 8 * lane) = rk;
  *reinterpret_cast<u32x4*>(a.v + (int64_t)unit * D + 8 * lane) = rv;
}

int log2_of(int x) { return __builtin_ctz((unsigned)x); }

template <template <int, bool> class K, class A>
hipError_t by_type(int D, bool bf16, const A& a, unsigned blocks, hipStream_t st) {
  switch (D + bf16) {
    case 64: return K<8, false>::go(a, blocks, st);
    case 65: return K<8, true>::go(a, blocks, st);
    case 128: return K<16, false>::go(a, blocks, st);
    case 129: return K<16, true>::go(a, blocks, st);
    case 256: return K<32, false>::go(a, blocks, st);
    default: return K<32, true>::go(a, blocks, st);
  }
}
template <int LPH, bool BF16>
struct GoRope {
  static hipError_t go(const RopeArgs& a, unsigned blocks, hipStream_t st) {
    kv4_rope_kernel<LPH, BF16><<<dim3(blocks), dim3(kThreads), 0, st>>>(a);
    return hipGetLastError();
  }
};
template <int LPH, bool BF16>
struct GoRead {
  static hipError_t go(const ReadArgs& a, unsigned blocks, hipStream_t st) {
    kv4_read_kernel<LPH, BF16><<<dim3(blocks), dim3(kThreads), 0, st>>>(a);
    return hipGetLastError();
  }
};

}  // namespace

hipError_t launch_rope(const w4a16_rope& t, const w4a16_kv4* kv, const int32_t* rows,
                       hipStream_t st) {
  RopeArgs a{};
  a.q = static_cast<const uint16_t*>(t.q);
  a.k = static_cast<const uint16_t*>(t.k);
  a.q_token = t.q_token;
  a.q_head = t.q_head;
  a.k_token = t.k_token;
  a.k_head = t.k_head;
  a.q_out = static_cast<uint16_t*>(t.q_out);
  a.k_out = static_cast<uint16_t*>(t.k_out);
  a.cos = t.cos;
  a.sin = t.sin;
  a.position = t.token_position;
  a.q_weight = static_cast<const uint16_t*>(t.q_weight);
  a.k_weight = static_cast<const uint16_t*>(t.k_weight);
  a.tokens = (int)t.tokens;
  a.positions = (int)t.positions;
  a.q_heads = t.q_heads;
  a.kv_heads = t.kv_heads;
  a.half = t.rot_dim / 2;
  a.eps = t.eps;
  a.interleaved = (t.flags & W4A16_KV4_INTERLEAVED) != 0;
  const int D = t.head_dim;
  a.group_lanes = 1;
  const int per_block = kThreads / (D / 8);
  a.qk_blocks = (int)((t.tokens * (t.q_heads + t.kv_heads) + per_block - 1) / per_block);
  if (kv) {
    a.store = true;
    a.v = static_cast<const uint16_t*>(t.v);
    a.v_token = t.v_token;
    a.v_head = t.v_head;
    a.pool = kv->pool;
    a.table = kv->table;
    a.rows = rows;
    a.table_rows = (int)kv->rows;
    a.max_pages = (int)kv->max_pages;
    a.pages = (int)kv->pages;
    a.page_shift = log2_of(kv->page_size);
    a.group_lanes = kv->group_size / 8;
    a.NG = D / kv->group_size;
    // short chunks where the long ones leave CUs without a workgroup: a chunk of
    // single tokens of many sequences changes words one by one
    a.chunk = t.tokens * t.kv_heads < 32 * 512 ? 8 : kChunk;
    a.value_blocks = (int)((t.tokens + a.chunk - 1) / a.chunk * t.kv_heads);
  }
  const unsigned blocks = (unsigned)a.qk_blocks + (unsigned)a.value_blocks;
  return by_type<GoRope>(D, t.flags & W4A16_KV4_BF16, a, blocks, st);
}

hipError_t launch_kv4_read(const w4a16_kv4& kv, const int32_t* positions, const int32_t* rows,
                           int64_t tokens, void* k, void* v, bool bf16, hipStream_t st) {
  const int D = kv.head_dim;
  ReadArgs a{kv.pool, kv.table, rows, positions, static_cast<uint16_t*>(k),
             static_cast<uint16_t*>(v), (int)tokens, kv.heads, (int)kv.rows, (int)kv.max_pages,
             (int)kv.pages, log2_of(kv.page_size), kv.group_size / 8, D / kv.group_size};
  const int per_block = kThreads / (D / 8);
  return by_type<GoRead>(D, bf16, a, (unsigned)((tokens * kv.heads + per_block - 1) / per_block),
                         st);
}

}  // namespace w4a16
