// Constants of the hash dropout (k_train_fused.hip) shared by the kernels that undo it.
#pragma once

// p -> the 16-bit threshold of the keep test and the factor of what is kept
static inline void drop_consts(float p, unsigned* thr, float* scale) {
  unsigned t = (unsigned)(p * 65536.f + 0.5f);
  if (t > 65535u) t = 65535u;
  *thr = t;
  *scale = 65536.f / (float)(65536u - t);                                 // the exact keep probability of the 16-bit threshold
}
