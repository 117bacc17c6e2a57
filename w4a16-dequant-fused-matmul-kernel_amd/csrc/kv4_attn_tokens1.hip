// Attention over the 4-bit cache: kv4_attn.h with 16 query rows a wave, tokens split over four
// or eight waves.
#include "kv4_attn.h"

namespace w4a16 {

hipError_t launch_attention_tokens1(const AttnArgs& a, int D, int NG, hipStream_t st) {
  return launch_attention_form<1, 4>(a, D, NG, st);
}
hipError_t launch_attention_tokens1_wide(const AttnArgs& a, int D, int NG, hipStream_t st) {
  return launch_attention_form<1, 8>(a, D, NG, st);
}

}  // namespace w4a16
