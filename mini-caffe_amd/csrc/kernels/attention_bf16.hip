#include "attention_launch.h"

int mchip::attention_bf16(const AttentionArgs& a, bool paged, hipStream_t st) {
  return paged ? launch_type<bf16_t, true>(a, st) : launch_type<bf16_t, false>(a, st);
}
