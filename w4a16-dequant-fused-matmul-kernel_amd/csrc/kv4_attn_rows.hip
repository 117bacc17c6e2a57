// Attention over the 4-bit cache: kv4_attn.h with 32 query rows a wave (16 of heads of 256), each wave with
// rows of its own.
#include "kv4_attn.h"

namespace w4a16 {

hipError_t launch_attention_rows(const AttnArgs& a, int D, int NG, hipStream_t st) {
  return launch_attention_form<2, 1>(a, D, NG, st);
}
hipError_t launch_attention_rows256(const AttnArgs& a, int NG, hipStream_t st) {
  const dim3 grid((unsigned)a.heads * a.splits * a.batch * a.tiles), block(64);
  switch (NG) {
    case 1: kv4_attention_kernel<256, 1, 1, 1><<<grid, block, 0, st>>>(a); break;
    case 2: kv4_attention_kernel<256, 2, 1, 1><<<grid, block, 0, st>>>(a); break;
    default: kv4_attention_kernel<256, 4, 1, 1><<<grid, block, 0, st>>>(a); break;
  }
  return hipGetLastError();
}

}  // namespace w4a16
