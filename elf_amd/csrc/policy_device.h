// What the kernels of the policy-network operators share: element types, sums over a wave, vectors, argument checks.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/goenv.h"
#include "goenv_host.h"

namespace goenv {

__device__ __forceinline__ float load_any(const void* p, int dt, int64_t i) {
  if (dt == GOENV_DT_F32) return static_cast<const float*>(p)[i];
  if (dt == GOENV_DT_BF16) return (float)static_cast<const __bf16*>(p)[i];
  return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_any(void* p, int dt, int64_t i, float v) {
  if (dt == GOENV_DT_F32) static_cast<float*>(p)[i] = v;
  else if (dt == GOENV_DT_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// A wave's lanes joined by f, in the same order every time, for every lane: scans along rows of 16 lanes, then across the rows (the
// last lane has seen all).  Register moves between lanes; an exchange through LDS takes ten times as long.
template <int CTRL, int ROWS, typename F>
__device__ __forceinline__ float join_step(float v, float none, F f) {
  return f(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false)));
}
template <typename F>
__device__ __forceinline__ float wave_join(float v, float none, F f) {
  v = join_step<0x111, 0xf>(v, none, f);   // from 1, 2, 4 and 8 lanes before in the row
  v = join_step<0x112, 0xf>(v, none, f);
  v = join_step<0x114, 0xf>(v, none, f);
  v = join_step<0x118, 0xf>(v, none, f);
  v = join_step<0x142, 0xa>(v, none, f);   // the last lane of rows 0 and 2 to rows 1 and 3
  v = join_step<0x143, 0xc>(v, none, f);   // lane 31 to rows 2 and 3
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_join(v, 0.f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) { return wave_join(v, -INFINITY, fmaxf); }

template <int N>
struct Int {
  static constexpr int value = N;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}

inline bool is_dtype(int dt) { return dt == GOENV_DT_F32 || dt == GOENV_DT_BF16 || dt == GOENV_DT_F16; }
inline bool aligned(const void* p, int dt) { return ((uintptr_t)p & (dt == GOENV_DT_F32 ? 3 : 1)) == 0; }
inline unsigned grid_of(int64_t items, int64_t most = 1 << 20) { return (unsigned)(items < most ? items : most); }

// `bytes` on from p; no array stays none
template <typename P>
P* past(P* p, int64_t bytes) {
  return p ? reinterpret_cast<P*>(reinterpret_cast<uintptr_t>(p) + bytes) : nullptr;
}

#define ON_DEVICE(dev, who)           \
  DeviceScope dev_scope_(dev);        \
  if (dev_scope_.err != hipSuccess) return fail(who ": selecting the device", dev_scope_.err)

// f<element type>() for the dtype
template <typename F>
void by_dtype(int dt, F f) {
  if (dt == GOENV_DT_F32) f(float());
  else if (dt == GOENV_DT_BF16) f(__bf16());
  else f(_Float16());
}

}  // namespace goenv
