#include "attention_launch.h"

int mchip::attention_f16(const AttentionArgs& a, bool paged, hipStream_t st) {
  return paged ? launch_type<half_t, true>(a, st) : launch_type<half_t, false>(a, st);
}
