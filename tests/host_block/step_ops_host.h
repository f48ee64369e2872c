// Further host stand-ins, for the kernels of rotary.hip, token_logprobs.hip and accept_path.hip (see
// hip/hip_runtime.h for the execution model). TEST INFRASTRUCTURE ONLY: forced in front of those sources with
// -include. Atomics are atomics (threads of a workgroup are host threads), sincospif is taken in 64 bits and
// rounded.
#pragma once
#include <atomic>
#include <cmath>

#include "hip/hip_runtime.h"

#define FTA_FORGET(x) ((void)(x))
inline int atomicAdd(int* at, int v) { return std::atomic_ref<int>(*at).fetch_add(v); }
inline int atomicMin(int* at, int v) {
  std::atomic_ref<int> ref(*at);
  int old = ref.load();
  while (v < old && !ref.compare_exchange_weak(old, v)) {
  }
  return old;
}
inline void sincospif(float x, float* s, float* c) {
  const double a = 3.14159265358979323846 * static_cast<double>(x);
  *s = static_cast<float>(std::sin(a));
  *c = static_cast<float>(std::cos(a));
}
