// Attention over the 4-bit cache: kv4_attn.h with 32 query rows a wave, tokens split over the waves.
#include "kv4_attn.h"

namespace w4a16 {

hipError_t launch_attention_tokens2(const AttnArgs& a, int D, int NG, hipStream_t st) {
  return launch_attention_form<2, 4>(a, D, NG, st);
}

}  // namespace w4a16
