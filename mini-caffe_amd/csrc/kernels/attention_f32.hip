#include "attention_launch.h"

int mchip::attention_f32(const AttentionArgs& a, bool paged, hipStream_t st) {
  return paged ? launch_type<float, true>(a, st) : launch_type<float, false>(a, st);
}
