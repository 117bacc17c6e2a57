// Attention over the 4-bit cache: the choice of a launch and the joining of splits
// (the kernel: kv4_attn.h).
#include "kv4_attn.h"

namespace w4a16 {
namespace {

// Joins the splits of one query row: D / 4 lanes to a split, a workgroup takes
// 1024 / D splits at a time.  Bounded by the launch and two dependent reads where
// rows are few, by memory where they are many.
template <int D>
__global__ __launch_bounds__(kAttnThreads) void kv4_join_kernel(const AttnArgs a, int tile_rows,
                                                                int max_rows) {
  constexpr int kLanes = D / 4, kAtOnce = kAttnThreads / kLanes;
  __shared__ f32x4 sum[kAtOnce][kLanes];
  __shared__ float den[kAtOnce];
  uint32_t id = blockIdx.x;
  const int h = id % a.heads;
  id /= a.heads;
  const int r = id % max_rows, b = id / max_rows;
  const AttnSpan s = attn_span(a, b, r / tile_rows * tile_rows, tile_rows);
  if (r >= s.nq * a.per_kv) return;
  const int i = r / a.per_kv;
  const int64_t qrow = (int64_t)(s.q0 + i) * a.q_heads + h * a.per_kv + (r - i * a.per_kv);
  const int at = threadIdx.x % kLanes, o = threadIdx.x / kLanes;
  float m = kNoScore;
  for (int k = 0; k < s.active; ++k) m = fmaxf(m, part_ml(a, k, qrow, D)[0]);
  f32x4 v = {0, 0, 0, 0};
  float l = 0.0f;
  for (int k = o; k < s.active; k += kAtOnce) {
    const float* ml = part_ml(a, k, qrow, D);
    const float w = exp2f(ml[0] - m);
    l += ml[1] * w;
    v += *reinterpret_cast<const f32x4*>(part_values(a, k, qrow, D) + 4 * at) * w;
  }
  sum[o][at] = v;
  if (at == 0) den[o] = l;
  __syncthreads();
  if (o) return;
#pragma unroll
  for (int k = 1; k < kAtOnce; ++k) {
    v += sum[k][at];
    l += den[k];
  }
  const bool any = l > 0.0f || l != l;
  const float inv = any ? 1.0f / l : 0.0f;
  float x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = any ? v[j] * inv : 0.0f;
  store4(a.out + qrow * D + 4 * at, x, a.bf16);
  if (a.lse && at == 0) a.lse[qrow] = lse_of(m, l);
}

}  // namespace

Kv4Plan kv4_attention_plan(const w4a16_kv4& kv, const w4a16_kv4_query& q) {
  Kv4Plan p{};
  const int per_kv = q.q_heads / kv.heads;
  const int64_t rows = q.max_q * per_kv;
  p.rows_form = rows > 32;
  p.cols = rows > 16 && kv.head_dim < 256 ? 2 : 1;
  const int64_t tile_rows = p.rows_form ? 64 * p.cols : 16 * p.cols;
  p.tiles = (int)((rows + tile_rows - 1) / tile_rows);
  int64_t span = q.max_context;
  if (q.window > 0) span = span < q.window + q.max_q ? span : q.window + q.max_q;
  const int64_t blocks = (span + 31) / 32 + 1;
  // enough workgroups for every CU to hold a few, and for rows of unlike lengths to
  // even out; a split has at least four blocks a wave
  const int64_t units = q.batch * kv.heads * p.tiles, least = p.rows_form ? 8 : 16;
  int64_t want = (1024 + units - 1) / units;
  const int64_t most = (blocks + least - 1) / least;
  if (want > most) want = most;
  if (want < 1) want = 1;
  p.chunk = (int)((blocks + want - 1) / want);
  if (!p.rows_form) p.chunk = (p.chunk + 3) / 4 * 4;
  p.splits = (int)((blocks + p.chunk - 1) / p.chunk);
  p.workspace = p.splits > 1 ? (size_t)p.splits * (size_t)q.tokens * (size_t)q.q_heads *
                                   (size_t)(kv.head_dim + 2) * sizeof(float)
                             : 0;
  return p;
}

hipError_t launch_kv4_attention(const Kv4Attn& c, hipStream_t st) {
  const w4a16_kv4& kv = c.kv;
  const w4a16_kv4_query& q = c.q;
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q.q);
  a.q_token = q.q_token;
  a.q_head = q.q_head;
  a.out = static_cast<uint16_t*>(q.out);
  a.lse = q.lse;
  a.part = c.part;
  a.pool = reinterpret_cast<const uint32_t*>(kv.pool);
  a.table = kv.table;
  a.lens = q.lens;
  a.starts = q.q_starts;
  a.seqs = q.seqs;
  a.table_rows = (int)kv.rows;
  a.max_pages = (int)kv.max_pages;
  a.pages = (int)kv.pages;
  a.page_shift = __builtin_ctz((unsigned)kv.page_size);
  a.heads = kv.heads;
  a.q_heads = q.q_heads;
  a.per_kv = q.q_heads / kv.heads;
  a.batch = (int)q.batch;
  a.tokens = (int)q.tokens;
  a.tiles = c.tiles;
  a.splits = c.splits;
  a.chunk = c.chunk;
  a.window = q.window;
  a.scale_log2 = q.scale * 1.4426950408889634f;
  a.causal = (q.flags & W4A16_KV4_CAUSAL) != 0;
  a.bf16 = (q.flags & W4A16_KV4_BF16) != 0;
  a.vec = (reinterpret_cast<uintptr_t>(q.q) & 15) == 0 && (q.q_token | q.q_head) % 8 == 0;
  const int D = kv.head_dim, NG = D / kv.group_size;
  const hipError_t e = c.rows_form && D == 256 ? launch_attention_rows256(a, NG, st)
                       : c.rows_form ? launch_attention_rows(a, D, NG, st)
                       : c.cols == 2 ? launch_attention_tokens2(a, D, NG, st)
                                     : launch_attention_tokens1(a, D, NG, st);
  if (e != hipSuccess || c.splits == 1) return e;
  const int tile_rows = c.rows_form ? 64 * c.cols : 16 * c.cols;
  const int max_rows = (int)q.max_q * a.per_kv;
  const dim3 grid((unsigned)a.heads * max_rows * a.batch);
  switch (D) {
    case 64: kv4_join_kernel<64><<<grid, kAttnThreads, 0, st>>>(a, tile_rows, max_rows); break;
    case 128: kv4_join_kernel<128><<<grid, kAttnThreads, 0, st>>>(a, tile_rows, max_rows); break;
    default: kv4_join_kernel<256><<<grid, kAttnThreads, 0, st>>>(a, tile_rows, max_rows); break;
  }
  return hipGetLastError();
}

}  // namespace w4a16
