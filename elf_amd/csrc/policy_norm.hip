// Group norm with the residual sum and the activation, channels last (a policy network's, behind its convolutions).
// Interface and definitions: include/goenv.h.
#include "policy_device.h"

using namespace goenv;

namespace {

// Sum over a workgroup of WAVES waves, in the same order every time; every thread gets it.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) t += lds[w];
  return t;
}

// ---- group norm ---------------------------------------------------------------------------------
//
// y = act((x - mean) rstd w + b + residual) per sample and group.  Bound by memory: the forward pass has to read x and the residual
// and write y once (2,048 boards of 128 bf16 channels: 568 MB, 120 us = 4.7 TB/s; a large copy reaches 4.9), the
// backward pass reads x, dy and the residual and writes dx and dresidual (the same boards: 227 us = 4.2 TB/s; 256 boards, 118 MB: 26 us
// and 4 us for the channels' sums).
// So a sample's slab of a few groups is held by one workgroup, in LDS, from the first read to the write: the mean and then the
// squared deviations about it (not sums of squares, which lose the variance of data far from zero) are taken from LDS.  The loads
// go to LDS directly, without registers in between: with the slab in registers a thread's loads waited for each other
// and occupancy was three waves a SIMD (159 us for the case above).

// The hardware's exponential and reciprocal are off by about one step of float32 each; a division in full costs ten
// instructions an element.
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

// y = act(z), and dz = dy * act'(z).  (A NaN stays one; -inf and an infinite dy on the flat side of relu give 0.)
template <int ACT>
__device__ __forceinline__ float act_of(float slope, float z) {
  if (ACT == GOENV_ACT_RELU) return z <= 0.f ? 0.f : z;
  if (ACT == GOENV_ACT_LEAKY_RELU) return z > 0.f ? z : z * slope;
  if (ACT == GOENV_ACT_SILU) return z * sigmoid(z);
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float slope, float z, float dy) {
  if (ACT == GOENV_ACT_RELU) return z <= 0.f ? 0.f : dy;
  if (ACT == GOENV_ACT_LEAKY_RELU) return z > 0.f ? dy : dy * slope;
  if (ACT == GOENV_ACT_SILU) {
    const float s = sigmoid(z);
    return dy * (s * (1.f + z * (1.f - s)));
  }
  return dy;
}
// f(activation as a constant): the choice is made once, around a loop
template <typename F>
__host__ __device__ __forceinline__ void by_act(int act, F f) {
  if (act == GOENV_ACT_RELU) f(Int<GOENV_ACT_RELU>());
  else if (act == GOENV_ACT_LEAKY_RELU) f(Int<GOENV_ACT_LEAKY_RELU>());
  else if (act == GOENV_ACT_SILU) f(Int<GOENV_ACT_SILU>());
  else f(Int<GOENV_ACT_NONE>());
}

// `VEC` channels' weights or biases
template <int VEC>
__device__ __forceinline__ void load_params(const void* p, int dt, int c, float missing, float (&to)[VEC]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) to[j] = missing;
  } else if (dt == GOENV_DT_F32) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) to[j] = static_cast<const float*>(p)[c + j];
  } else if (dt == GOENV_DT_BF16) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) to[j] = (float)static_cast<const __bf16*>(p)[c + j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) to[j] = (float)static_cast<const _Float16*>(p)[c + j];
  }
}

// How a launch cuts the work: a workgroup has one sample's slab of slab_groups whole groups (width channels, units vectors of
// VEC channels a position) and the positions of one chunk; its threads are rows x units.
struct NormCut {
  int slab_groups, width, units, rows, slabs, chunks;
  int staged, scratch;    // vectors of a thread that are staged in LDS (of each array), behind this many floats of scratch
  int64_t chunk;          // positions of a chunk (the last one may have fewer)
};

constexpr int NORM_THREADS = 512;   // the most that a workgroup has

enum NormPhase { NORM_WHOLE, NORM_SUMS, NORM_APPLY };

// This thread's place in a launch: `count` positions of the chunk, from `first` on, `rows` apart.
struct NormPlace {
  int64_t sample, first, chunk_size;
  int c0, unit, row, part, count;   // first channel of the slab; the vector of the position; the row; the chunk
  bool on;                          // the thread has a row
};
// Workgroups go to the eight XCDs in turn; each XCD takes a run of neighbours, so that what lies next to each other in memory (the
// slabs of a sample share cache lines) meets in one L2.
__device__ __forceinline__ uint32_t near_block() {
  const uint32_t xcd = blockIdx.x & 7, share = gridDim.x >> 3, over = gridDim.x & 7;
  return xcd * share + (xcd < over ? xcd : over) + (blockIdx.x >> 3);
}
__device__ __forceinline__ NormPlace norm_place(const goenv_norm& P, const NormCut& cut) {
  NormPlace q;
  uint32_t b = near_block();
  q.part = (int)(b % (uint32_t)cut.chunks);
  b /= (uint32_t)cut.chunks;
  q.c0 = (int)(b % (uint32_t)cut.slabs) * cut.width;
  q.sample = b / (uint32_t)cut.slabs;
  const int64_t lo = q.part * cut.chunk;
  q.chunk_size = lo + cut.chunk < P.positions ? cut.chunk : P.positions - lo;
  q.unit = threadIdx.x % cut.units;
  q.row = threadIdx.x / cut.units;
  q.on = q.row < cut.rows;
  q.first = lo + (q.on && q.row < q.chunk_size ? q.row : 0);   // an address inside the sample for every thread
  q.count = q.on && q.row < q.chunk_size ? ((int)q.chunk_size - q.row + cut.rows - 1) / cut.rows : 0;
  return q;
}

__host__ __device__ __forceinline__ bool is_pow2(int v) { return (v & (v - 1)) == 0; }

// Sums over a slab's groups.  Each thread brings its vector's sum: NV = 1 where a vector lies within one group, else a value per
// channel.  Where the vectors of a position and of a group are powers of two that fit a wave, lanes are added up by
// exchanges and a group's sum is one value per wave; elsewhere a wave adds up a group's values from LDS.  Returned
// for the thread's channels (group_of(j) of its own).  lds: threads * NV + groups floats; every thread of the workgroup calls.
template <int VEC, int NV>
__device__ __forceinline__ void slab_sum(const NormCut& cut, int cpg, const NormPlace& q, float (&val)[NV], float* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if (!q.on)
#pragma unroll
    for (int j = 0; j < NV; ++j) val[j] = 0.f;
  const int per = NV == 1 ? cpg / VEC : 0;   // vectors of a group
  if (NV == 1 && cut.units <= 64 && is_pow2(cut.units) && is_pow2(per)) {
    float v = val[0];
    for (int d = 1; d < per; d <<= 1) v += __shfl_xor(v, d);
    for (int d = cut.units; d < 64; d <<= 1) v += __shfl_xor(v, d);
    const int g = q.unit / per;
    if (lane < cut.units && q.unit % per == 0) lds[wave * cut.slab_groups + g] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < waves; ++w) v += lds[w * cut.slab_groups + g];
    val[0] = v;
    __syncthreads();
    return;
  }
  float* total = lds + blockDim.x * NV;
#pragma unroll
  for (int j = 0; j < NV; ++j) lds[threadIdx.x * NV + j] = val[j];
  __syncthreads();
  const int mine = NV == 1 ? per : cpg;     // a group's values per row: they lie next to each other
  const int down = 64 / mine, right = 64 - down * mine, row0 = lane / mine, col0 = lane - row0 * mine;
  for (int g = wave; g < cut.slab_groups; g += waves) {
    float v = 0.f;
    for (int row = row0, col = col0; row < cut.rows;) {
      v += lds[row * cut.units * NV + g * mine + col];
      row += down;
      col += right;
      if (col >= mine) {
        col -= mine;
        ++row;
      }
    }
    v = wave_sum(v);
    if (lane == 0) total[g] = v;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NV; ++j) val[j] = total[NV == 1 ? q.unit / per : (q.unit * VEC + j) / cpg];
  __syncthreads();
}

// Arrays that are read through LDS: a thread's slot k of an area is its own, what it puts there only it reads.  Vectors of 16 bytes go
// there without passing through registers (a wave's 64 slots lie next to each other, as the instruction wants them), so that
// all of a thread's loads are under way at once.
template <typename T, int VEC>
__device__ __forceinline__ void stage(const T* from, Pack<T, VEC>* area, int k) {
  if constexpr (sizeof(Pack<T, VEC>) == 16) {
    Pack<T, VEC>* wave0 = area + k * blockDim.x + __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)wave0, 16, 0, 0);
  } else {
    area[k * blockDim.x + threadIdx.x] = load_pack<T, VEC>(from);
  }
}

// Before the first read of a staged slot: the loads to LDS are counted with the loads from memory, and nothing else waits for them.
__device__ __forceinline__ void staged_here() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> staged_pack(const Pack<T, VEC>* slot) {
  if constexpr (sizeof(Pack<T, VEC>) == 16) {
    typedef uint32_t Quad __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(Pack<T, VEC>, *reinterpret_cast<const Quad*>(slot));   // one 16-byte read
  } else {
    return *slot;
  }
}

// Group norm of a slab's chunk.  x and the residual are read once, into LDS (the first `staged` vectors of a thread; what does not fit
// is read again in each pass, from the caches).  WHOLE: statistics, normalisation, residual and activation in one
// launch.  SUMS: a chunk's mean and sum of squared deviations to the workspace [n][groups][chunks].  APPLY: joins the chunks' and
// applies them.
template <typename T, int VEC, bool ONE, bool RES, int PHASE>
__global__ __launch_bounds__(NORM_THREADS) void k_group_norm(goenv_norm P, NormCut cut, T* y) {
  extern __shared__ __align__(16) float lds[];
  constexpr int NV = ONE ? 1 : VEC;
  const int cpg = P.channels / P.groups;
  const NormPlace q = norm_place(P, cut);
  const int c = q.c0 + q.unit * VEC;
  const T* x = static_cast<const T*>(P.x) + q.sample * P.x_sample + q.first * P.x_position + c;
  const T* r = RES ? static_cast<const T*>(P.residual) + q.sample * P.r_sample + q.first * P.r_position + c : nullptr;
  const int64_t xs = cut.rows * P.x_position, rs = cut.rows * P.r_position, os = (int64_t)cut.rows * P.channels;
  Pack<T, VEC>*area = reinterpret_cast<Pack<T, VEC>*>(lds + cut.scratch), *area2 = area + cut.staged * blockDim.x;
  const int staged = q.count < cut.staged ? q.count : cut.staged;
  for (int k = 0; k < staged; ++k) stage<T, VEC>(x + k * xs, area, k);
  if (RES)
    for (int k = 0; k < staged; ++k) stage<T, VEC>(r + k * rs, area2, k);
  float w[VEC], b[VEC];
  load_params<VEC>(P.weight, P.param_dtype, c, 1.f, w);
  load_params<VEC>(P.bias, P.param_dtype, c, 0.f, b);

  float mean[NV], rstd[NV];
  if (PHASE != NORM_APPLY) {
    staged_here();
    const float inv_m = 1.f / ((float)q.chunk_size * (float)cpg);
#pragma unroll
    for (int j = 0; j < NV; ++j) mean[j] = rstd[j] = 0.f;
    auto add = [&](const Pack<T, VEC>& a) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) mean[ONE ? 0 : j] += (float)a.v[j];
    };
    for (int k = 0; k < staged; ++k) add(staged_pack(&area[k * blockDim.x + threadIdx.x]));
    for (int k = staged; k < q.count; ++k) add(load_pack<T, VEC>(x + k * xs));
    slab_sum<VEC, NV>(cut, cpg, q, mean, lds);
#pragma unroll
    for (int j = 0; j < NV; ++j) mean[j] *= inv_m;
    auto square = [&](const Pack<T, VEC>& a) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = (float)a.v[j] - mean[ONE ? 0 : j];
        rstd[ONE ? 0 : j] += d * d;
      }
    };
    for (int k = 0; k < staged; ++k) square(staged_pack(&area[k * blockDim.x + threadIdx.x]));
    for (int k = staged; k < q.count; ++k) square(load_pack<T, VEC>(x + k * xs));
    slab_sum<VEC, NV>(cut, cpg, q, rstd, lds);
    if (PHASE == NORM_WHOLE)
#pragma unroll
      for (int j = 0; j < NV; ++j) rstd[j] = 1.f / sqrtf(rstd[j] * inv_m + P.eps);
    // one thread per group says what it has
    float2* to = PHASE == NORM_SUMS ? static_cast<float2*>(P.workspace) : reinterpret_cast<float2*>(P.stats);
    if (to && q.on && q.row == 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if ((c + j) % cpg == 0) to[(q.sample * P.groups + (c + j) / cpg) * cut.chunks + q.part] = make_float2(mean[j], rstd[j]);
    }
    if (PHASE == NORM_SUMS) return;
  } else {
    // mean = sum n_k mean_k / n; the deviations about it: sum of M2_k + n_k (mean_k - mean)^2.  A wave takes every eighth group or so,
    // four at a time, with their loads under way together (and with the loads to LDS).
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const float inv_m = 1.f / ((float)P.positions * (float)cpg);
    const float2* parts = static_cast<const float2*>(P.workspace) + (q.sample * P.groups + q.c0 / cpg) * cut.chunks;
    auto size = [&](int k) { return (float)((k + 1) * cut.chunk < P.positions ? cut.chunk : P.positions - k * cut.chunk) * (float)cpg; };
    const float size0 = lane < cut.chunks ? size(lane) : 0.f;
    for (int g0 = wave; g0 < cut.slab_groups; g0 += 4 * waves) {
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int g = g0 + i * waves;
        v[i] = parts[(int64_t)(g < cut.slab_groups ? g : g0) * cut.chunks + (lane < cut.chunks ? lane : 0)];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int g = g0 + i * waves;
        if (g >= cut.slab_groups) break;
        const float2* part = parts + (int64_t)g * cut.chunks;
        float m = size0 * v[i].x, s = lane < cut.chunks ? v[i].y : 0.f;
        for (int k = lane + 64; k < cut.chunks; k += 64) m += size(k) * part[k].x;
        m = wave_sum(m);
        m *= inv_m;
        s += size0 * (v[i].x - m) * (v[i].x - m);
        for (int k = lane + 64; k < cut.chunks; k += 64) {
          const float2 u = part[k];
          s += u.y + size(k) * (u.x - m) * (u.x - m);
        }
        s = wave_sum(s);
        s = 1.f / sqrtf(s * inv_m + P.eps);
        if (lane == 0) {
          lds[2 * g] = m;
          lds[2 * g + 1] = s;
          if (P.stats && q.part == 0) reinterpret_cast<float2*>(P.stats)[q.sample * P.groups + q.c0 / cpg + g] = make_float2(m, s);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int g = (q.unit * VEC + j) / cpg;
      mean[j] = lds[2 * g];
      rstd[j] = lds[2 * g + 1];
    }
    staged_here();
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) w[j] *= rstd[ONE ? 0 : j];
  T* o = y + (q.sample * P.positions + q.first) * P.channels + c;
  by_act(P.act, [&](auto act) {
    auto apply = [&](int k, const Pack<T, VEC>& a, const Pack<T, VEC>& e) {
      Pack<T, VEC> out;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float z = ((float)a.v[j] - mean[ONE ? 0 : j]) * w[j] + b[j];
        if (RES) z += (float)e.v[j];
        out.v[j] = (T)act_of<decltype(act)::value>(P.slope, z);
      }
      *reinterpret_cast<Pack<T, VEC>*>(o + k * os) = out;
    };
    for (int k = 0; k < staged; ++k) {
      const int at = k * blockDim.x + threadIdx.x;
      apply(k, staged_pack(&area[at]), RES ? staged_pack(&area2[at]) : Pack<T, VEC>());
    }
    for (int k = staged; k < q.count; ++k) apply(k, load_pack<T, VEC>(x + k * xs), RES ? load_pack<T, VEC>(r + k * rs) : Pack<T, VEC>());
  });
}

// The gradients of a slab's chunk, cut and staged as above.  WHOLE: the channels' sums of dz and dz xh (to the workspace,
// [n][chunks][channels], for k_group_norm_param_grad), the groups' means from them, dx and dresidual.  SUMS: the sums alone.
// APPLY: joins the chunks' sums; dx and dresidual.
template <typename T, int VEC, bool RES, int PHASE>
__global__ __launch_bounds__(NORM_THREADS) void k_group_norm_grad(goenv_norm P, NormCut cut, const T* dy0, int64_t dy_sample,
                                                                  int64_t dy_position, T* dx, T* dr) {
  extern __shared__ __align__(16) float lds[];
  const int cpg = P.channels / P.groups, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const NormPlace q = norm_place(P, cut);
  const int c = q.c0 + q.unit * VEC;
  const T* x = static_cast<const T*>(P.x) + q.sample * P.x_sample + q.first * P.x_position + c;
  const T* r = RES ? static_cast<const T*>(P.residual) + q.sample * P.r_sample + q.first * P.r_position + c : nullptr;
  const T* dy = dy0 + q.sample * dy_sample + q.first * dy_position + c;
  const int64_t xs = cut.rows * P.x_position, rs = cut.rows * P.r_position, gs = cut.rows * dy_position, os = (int64_t)cut.rows * P.channels;
  Pack<T, VEC>*area = reinterpret_cast<Pack<T, VEC>*>(lds + cut.scratch), *area2 = area + cut.staged * blockDim.x,
             *area3 = area2 + cut.staged * blockDim.x;
  const int staged = q.count < cut.staged ? q.count : cut.staged;
  for (int k = 0; k < staged; ++k) {
    stage<T, VEC>(x + k * xs, area, k);
    stage<T, VEC>(dy + k * gs, area2, k);
    if (RES) stage<T, VEC>(r + k * rs, area3, k);
  }
  float w[VEC], b[VEC], mean[VEC], rstd[VEC];
  load_params<VEC>(P.weight, P.param_dtype, c, 1.f, w);
  load_params<VEC>(P.bias, P.param_dtype, c, 0.f, b);
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float2 st = reinterpret_cast<const float2*>(P.stats)[q.sample * P.groups + (c + j) / cpg];
    mean[j] = st.x;
    rstd[j] = st.y;
  }
  if (PHASE != NORM_APPLY) staged_here();
  // f(j, xh, dz) for every element of the thread's
  auto each = [&](auto f, auto done) {
    by_act(P.act, [&](auto act) {
      auto one = [&](int k, const Pack<T, VEC>& a, const Pack<T, VEC>& g, const Pack<T, VEC>& e) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xh = ((float)a.v[j] - mean[j]) * rstd[j];
          float z = xh * w[j] + b[j];
          if (RES) z += (float)e.v[j];
          f(j, xh, act_grad<decltype(act)::value>(P.slope, z, (float)g.v[j]));
        }
        done(k);
      };
      for (int k = 0; k < staged; ++k) {
        const int at = k * blockDim.x + threadIdx.x;
        one(k, staged_pack(&area[at]), staged_pack(&area2[at]), RES ? staged_pack(&area3[at]) : Pack<T, VEC>());
      }
      for (int k = staged; k < q.count; ++k)
        one(k, load_pack<T, VEC>(x + k * xs), load_pack<T, VEC>(dy + k * gs), RES ? load_pack<T, VEC>(r + k * rs) : Pack<T, VEC>());
    });
  };
  float2* part = static_cast<float2*>(P.workspace);
  float* sum1 = lds;                       // [width] of w dz, then of w dz xh: a channel's
  float* sum2 = lds + cut.width;
  float* group = sum2 + cut.width;         // [slab_groups][2]: a group's means
  float* red = group + 2 * cut.slab_groups;
  if (PHASE != NORM_APPLY) {
    float a1[VEC], a2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a1[j] = a2[j] = 0.f;
    each(
        [&](int j, float xh, float dz) {
          a1[j] += dz;
          a2[j] += dz * xh;
        },
        [](int) {});
    // over the rows: by exchanges where the units of a position are a power of two that fits a wave, then over the waves (or all rows)
    const bool pow2 = cut.units <= 64 && is_pow2(cut.units);
    if (pow2)
      for (int d = cut.units; d < 64; d <<= 1)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          a1[j] += __shfl_xor(a1[j], d);
          a2[j] += __shfl_xor(a2[j], d);
        }
    const int from = pow2 ? wave : q.row;
    int many = pow2 ? waves : cut.rows;
    auto put = [&](int at) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        red[(at * 2) * cut.width + q.unit * VEC + j] = a1[j];
        red[(at * 2 + 1) * cut.width + q.unit * VEC + j] = a2[j];
      }
    };
    for (; many > 8 && !pow2; many -= many / 2) {   // rows in pairs, until eight are left
      const int kept = many - many / 2;
      if (q.on && from >= kept && from < many) put(from - kept);
      __syncthreads();
      if (q.on && from < many / 2)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          a1[j] += red[(from * 2) * cut.width + q.unit * VEC + j];
          a2[j] += red[(from * 2 + 1) * cut.width + q.unit * VEC + j];
        }
      __syncthreads();
    }
    if (pow2 ? lane < cut.units : q.on && from < many) put(from);
    __syncthreads();
    for (int k = threadIdx.x; k < cut.width; k += blockDim.x) {
      float s1 = 0.f, s2 = 0.f;
      for (int i = 0; i < many; ++i) {
        s1 += red[(i * 2) * cut.width + k];
        s2 += red[(i * 2 + 1) * cut.width + k];
      }
      part[(q.sample * cut.chunks + q.part) * P.channels + q.c0 + k] = make_float2(s1, s2);
      const float wk = P.weight ? load_any(P.weight, P.param_dtype, q.c0 + k) : 1.f;
      sum1[k] = wk * s1;
      sum2[k] = wk * s2;
    }
    if (PHASE == NORM_SUMS) return;
  } else {
    // the chunks' sums of a channel, by as many threads as there are for it
    const int each = (int)blockDim.x > cut.width ? (int)blockDim.x / cut.width : 1;
    const float2* from = part + q.sample * cut.chunks * P.channels + q.c0;
    for (int t = threadIdx.x; t < cut.width * each; t += blockDim.x) {
      const int ch = t % cut.width;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll 4
      for (int i = t / cut.width; i < cut.chunks; i += each) {
        const float2 v = from[(int64_t)i * P.channels + ch];
        s1 += v.x;
        s2 += v.y;
      }
      red[2 * t] = s1;
      red[2 * t + 1] = s2;
    }
    __syncthreads();
    for (int ch = threadIdx.x; ch < cut.width; ch += blockDim.x) {
      float s1 = 0.f, s2 = 0.f;
      for (int i = 0; i < each; ++i) {
        s1 += red[2 * (i * cut.width + ch)];
        s2 += red[2 * (i * cut.width + ch) + 1];
      }
      const float wk = P.weight ? load_any(P.weight, P.param_dtype, q.c0 + ch) : 1.f;
      sum1[ch] = wk * s1;
      sum2[ch] = wk * s2;
    }
  }
  __syncthreads();
  for (int g = wave; g < cut.slab_groups; g += waves) {
    float m1 = 0.f, m2 = 0.f;
    for (int k = lane; k < cpg; k += 64) {
      m1 += sum1[g * cpg + k];
      m2 += sum2[g * cpg + k];
    }
    m1 = wave_sum(m1);
    m2 = wave_sum(m2);
    const float inv_m = 1.f / ((float)P.positions * (float)cpg);
    if (lane == 0) {
      group[2 * g] = m1 * inv_m;
      group[2 * g + 1] = m2 * inv_m;
    }
  }
  __syncthreads();
  float m1[VEC], m2[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const int g = (q.unit * VEC + j) / cpg;
    m1[j] = group[2 * g];
    m2[j] = group[2 * g + 1];
  }
  if (PHASE == NORM_APPLY) staged_here();
  const int64_t o = (q.sample * P.positions + q.first) * P.channels + c;
  Pack<T, VEC> ox, orr;
  each(
      [&](int j, float xh, float dz) {
        orr.v[j] = (T)dz;
        ox.v[j] = (T)(rstd[j] * (dz * w[j] - m1[j] - xh * m2[j]));
      },
      [&](int k) {
        if (dx) *reinterpret_cast<Pack<T, VEC>*>(dx + o + k * os) = ox;
        if (dr) *reinterpret_cast<Pack<T, VEC>*>(dr + o + k * os) = orr;
      });
}

// Few positions (a feature vector a sample, a small board): a slab would leave most of a workgroup idle.  A team of 1 to 64
// lanes of one wave takes a sample's group instead, NK vectors a lane, all in registers; sums are exchanges within the team,
// without LDS and barriers (65,536 x 512 bf16 features in 8 groups: 352 -> 26 us, a copy's time; the gradient 910 -> 49 us, 4.1 TB/s).  A workgroup has the teams of slab_groups groups of `slots` samples and takes samples in strides,
// so that the gradient's channel sums stay in registers until the end.
struct FewCut {
  int team, units, rows;         // lanes of a team; its vectors of a position; the positions that it has at a time
  int slab_groups, slabs, slots;
  int64_t strides;               // workgroups of a slab
};
constexpr int FEW_THREADS = 256;

struct FewPlace {
  int lane, unit, group, slab;
  int64_t stride, first;         // the workgroup's number in its slab; the first sample
  bool on;                       // the team has a group
};
__device__ __forceinline__ FewPlace few_place(const goenv_norm& P, const FewCut& cut) {
  FewPlace q;
  const uint32_t b = near_block();
  q.slab = (int)(b % (uint32_t)cut.slabs);
  q.stride = b / (uint32_t)cut.slabs;
  const int team = threadIdx.x / cut.team, slot = team / cut.slab_groups;
  q.lane = threadIdx.x % cut.team;
  q.unit = q.lane % cut.units;
  q.group = q.slab * cut.slab_groups + team % cut.slab_groups;
  q.on = slot < cut.slots && q.group < P.groups;
  q.first = q.on ? q.stride * cut.slots + slot : P.n;
  if (!q.on) q.group = 0;
  return q;
}
// The lane's positions; behind the last one, that one again
template <int NK>
__device__ __forceinline__ void few_positions(const goenv_norm& P, const FewCut& cut, const FewPlace& q, int (&at)[NK], bool (&in)[NK]) {
  const int row = q.lane / cut.units, last = (int)P.positions - 1;
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int p = row + k * cut.rows;
    in[k] = row < cut.rows && p <= last;
    at[k] = p < last ? p : last;
  }
}
__device__ __forceinline__ float team_sum(float v, int team) {
  for (int d = 1; d < team; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

template <typename T, int VEC, int NK, bool RES>
__global__ __launch_bounds__(FEW_THREADS) void k_group_norm_few(goenv_norm P, FewCut cut, T* y) {
  const int cpg = P.channels / P.groups;
  const FewPlace q = few_place(P, cut);
  const int c = q.group * cpg + q.unit * VEC;
  int at[NK];
  bool in[NK];
  few_positions<NK>(P, cut, q, at, in);
  float w[VEC], b[VEC];
  load_params<VEC>(P.weight, P.param_dtype, c, 1.f, w);
  load_params<VEC>(P.bias, P.param_dtype, c, 0.f, b);
  const float inv_m = 1.f / ((float)P.positions * (float)cpg);
  for (int64_t sample = q.first; sample < P.n; sample += cut.strides * cut.slots) {
    const T* x = static_cast<const T*>(P.x) + sample * P.x_sample + c;
    const T* r = RES ? static_cast<const T*>(P.residual) + sample * P.r_sample + c : nullptr;
    T* o = y + sample * P.positions * P.channels + c;
    Pack<T, VEC> a[NK], e[RES ? NK : 1];
#pragma unroll
    for (int k = 0; k < NK; ++k) a[k] = load_pack<T, VEC>(x + at[k] * P.x_position);
    if (RES)
#pragma unroll
      for (int k = 0; k < NK; ++k) e[k] = load_pack<T, VEC>(r + at[k] * P.r_position);
    float mean = 0.f, rstd = 0.f;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) s += (float)a[k].v[j];
      mean += in[k] ? s : 0.f;
    }
    mean = team_sum(mean, cut.team) * inv_m;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = (float)a[k].v[j] - mean;
        s += d * d;
      }
      rstd += in[k] ? s : 0.f;
    }
    rstd = 1.f / sqrtf(team_sum(rstd, cut.team) * inv_m + P.eps);
    if (P.stats && q.lane == 0) reinterpret_cast<float2*>(P.stats)[sample * P.groups + q.group] = make_float2(mean, rstd);
    by_act(P.act, [&](auto act) {
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        Pack<T, VEC> out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float z = ((float)a[k].v[j] - mean) * (w[j] * rstd) + b[j];
          if (RES) z += (float)e[k].v[j];
          out.v[j] = (T)act_of<decltype(act)::value>(P.slope, z);
        }
        if (in[k]) *reinterpret_cast<Pack<T, VEC>*>(o + (int64_t)at[k] * P.channels) = out;
      }
    });
  }
}

// The gradients.  The workspace: [strides][channels] sums of dz and dz xh, for k_group_norm_param_grad.
template <typename T, int VEC, int NK, bool RES>
__global__ __launch_bounds__(FEW_THREADS) void k_group_norm_few_grad(goenv_norm P, FewCut cut, const T* dy0, int64_t dy_sample, int64_t dy_position,
                                                                     T* dx, T* dr) {
  __shared__ float lds[2][VEC][FEW_THREADS];
  const int cpg = P.channels / P.groups;
  const FewPlace q = few_place(P, cut);
  const int c = q.group * cpg + q.unit * VEC;
  int at[NK];
  bool in[NK];
  few_positions<NK>(P, cut, q, at, in);
  float w[VEC], b[VEC], sum1[VEC], sum2[VEC];
  load_params<VEC>(P.weight, P.param_dtype, c, 1.f, w);
  load_params<VEC>(P.bias, P.param_dtype, c, 0.f, b);
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum1[j] = sum2[j] = 0.f;
  const float inv_m = 1.f / ((float)P.positions * (float)cpg);
  for (int64_t sample = q.first; sample < P.n; sample += cut.strides * cut.slots) {
    const T* x = static_cast<const T*>(P.x) + sample * P.x_sample + c;
    const T* r = RES ? static_cast<const T*>(P.residual) + sample * P.r_sample + c : nullptr;
    const T* dy = dy0 + sample * dy_sample + c;
    Pack<T, VEC> a[NK], g[NK], e[RES ? NK : 1];
#pragma unroll
    for (int k = 0; k < NK; ++k) a[k] = load_pack<T, VEC>(x + at[k] * P.x_position);
#pragma unroll
    for (int k = 0; k < NK; ++k) g[k] = load_pack<T, VEC>(dy + at[k] * dy_position);
    if (RES)
#pragma unroll
      for (int k = 0; k < NK; ++k) e[k] = load_pack<T, VEC>(r + at[k] * P.r_position);
    const float2 st = reinterpret_cast<const float2*>(P.stats)[sample * P.groups + q.group];
    const float mean = st.x, rstd = st.y;
    float xh[NK][VEC], dz[NK][VEC], m1 = 0.f, m2 = 0.f;
    by_act(P.act, [&](auto act) {
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float h = ((float)a[k].v[j] - mean) * rstd;
          float z = h * w[j] + b[j];
          if (RES) z += (float)e[k].v[j];
          const float d = act_grad<decltype(act)::value>(P.slope, z, (float)g[k].v[j]);
          xh[k][j] = h;
          dz[k][j] = d;
          sum1[j] += in[k] ? d : 0.f;
          sum2[j] += in[k] ? d * h : 0.f;
          m1 += in[k] ? d * w[j] : 0.f;
          m2 += in[k] ? d * w[j] * h : 0.f;
        }
    });
    m1 = team_sum(m1, cut.team) * inv_m;
    m2 = team_sum(m2, cut.team) * inv_m;
    const int64_t o = sample * P.positions * P.channels + c;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      Pack<T, VEC> ox, orr;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        orr.v[j] = (T)dz[k][j];
        ox.v[j] = (T)(rstd * (dz[k][j] * w[j] - m1 - xh[k][j] * m2));
      }
      if (in[k]) {
        if (dx) *reinterpret_cast<Pack<T, VEC>*>(dx + o + (int64_t)at[k] * P.channels) = ox;
        if (dr) *reinterpret_cast<Pack<T, VEC>*>(dr + o + (int64_t)at[k] * P.channels) = orr;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    lds[0][j][threadIdx.x] = sum1[j];
    lds[1][j][threadIdx.x] = sum2[j];
  }
  __syncthreads();
  float2* part = static_cast<float2*>(P.workspace) + q.stride * P.channels;
  const int left = P.groups - q.slab * cut.slab_groups, width = (left < cut.slab_groups ? left : cut.slab_groups) * cpg;
  for (int ch = threadIdx.x; ch < width; ch += FEW_THREADS) {
    const int group = ch / cpg, in_group = ch % cpg, j = in_group % VEC, from = group * cut.team + in_group / VEC;
    float s1 = 0.f, s2 = 0.f;
    for (int slot = 0; slot < cut.slots; ++slot)
      for (int row = 0; row < cut.rows; ++row) {
        const int t = from + slot * cut.slab_groups * cut.team + row * cut.units;
        s1 += lds[0][j][t];
        s2 += lds[1][j][t];
      }
    part[q.slab * cut.slab_groups * cpg + ch] = make_float2(s1, s2);
  }
}

// dbias and dweight: the sums of the samples' (and chunks') parts, 16 channels (a cache line) a workgroup, 64 rows at a time
__global__ __launch_bounds__(1024) void k_group_norm_param_grad(const float2* part, int64_t rows, int channels, int param_dtype, void* dweight,
                                                                void* dbias) {
  __shared__ float2 lds[64][16];
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float a = 0.f, b = 0.f;
  if (c < channels)
#pragma unroll 4
    for (int64_t i = row; i < rows; i += 64) {
      const float2 v = part[i * channels + c];
      a += v.x;
      b += v.y;
    }
  lds[row][col] = make_float2(a, b);
  __syncthreads();
  if (row != 0 || c >= channels) return;
#pragma unroll 8
  for (int i = 1; i < 64; ++i) {
    a += lds[i][col].x;
    b += lds[i][col].y;
  }
  if (dbias) store_any(dbias, param_dtype, c, a);
  if (dweight) store_any(dweight, param_dtype, c, b);
}

template <typename T>
__global__ __launch_bounds__(256) void k_group_norm_any(goenv_norm P, T* y) {
  __shared__ float lds[4];
  const int cpg = P.channels / P.groups;
  const int64_t m = P.positions * cpg;
  for (int64_t item = blockIdx.x; item < P.n * P.groups; item += gridDim.x) {
    const int64_t i = item / P.groups;
    const int c0 = (int)(item % P.groups) * cpg;
    const T* x = static_cast<const T*>(P.x) + i * P.x_sample + c0;
    const T* r = P.residual ? static_cast<const T*>(P.residual) + i * P.r_sample + c0 : nullptr;
    T* o = y + i * P.positions * P.channels + c0;
    float s = 0.f;
    for (int64_t k = threadIdx.x; k < m; k += 256) s += (float)x[k / cpg * P.x_position + k % cpg];
    const float mean = block_sum<4>(s, lds) / (float)m;
    s = 0.f;
    for (int64_t k = threadIdx.x; k < m; k += 256) {
      const float d = (float)x[k / cpg * P.x_position + k % cpg] - mean;
      s += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum<4>(s, lds) / (float)m + P.eps);
    if (P.stats && threadIdx.x == 0) {
      P.stats[2 * item] = mean;
      P.stats[2 * item + 1] = rstd;
    }
    for (int64_t k = threadIdx.x; k < m; k += 256) {
      const int c = (int)(k % cpg);
      const int64_t p = k / cpg;
      float z = ((float)x[p * P.x_position + c] - mean) * rstd;
      if (P.weight) z *= load_any(P.weight, P.param_dtype, c0 + c);
      if (P.bias) z += load_any(P.bias, P.param_dtype, c0 + c);
      if (r) z += (float)r[p * P.r_position + c];
      by_act(P.act, [&](auto a) { o[p * P.channels + c] = (T)act_of<decltype(a)::value>(P.slope, z); });
    }
  }
}

// dx and dresidual of one sample's group, and its channels' part of dbias and dweight into workspace [n][channels][2]
template <typename T>
__global__ __launch_bounds__(256) void k_group_norm_any_grad(goenv_norm P, const T* dy0, int64_t dy_sample, int64_t dy_position, T* dx0,
                                                         T* dr0) {
  __shared__ float lds[4];
  const int cpg = P.channels / P.groups;
  const int64_t m = P.positions * cpg;
  float2* part = static_cast<float2*>(P.workspace);
  for (int64_t item = blockIdx.x; item < P.n * P.groups; item += gridDim.x) {
    const int64_t i = item / P.groups;
    const int c0 = (int)(item % P.groups) * cpg;
    const T* x = static_cast<const T*>(P.x) + i * P.x_sample + c0;
    const T* r = P.residual ? static_cast<const T*>(P.residual) + i * P.r_sample + c0 : nullptr;
    const T* dy = dy0 + i * dy_sample + c0;
    const float mean = P.stats[2 * item], rstd = P.stats[2 * item + 1];
    float s1 = 0.f, s2 = 0.f;
    for (int c = 0; c < cpg; ++c) {
      const float w = P.weight ? load_any(P.weight, P.param_dtype, c0 + c) : 1.f;
      const float b = P.bias ? load_any(P.bias, P.param_dtype, c0 + c) : 0.f;
      float a1 = 0.f, a2 = 0.f;
      for (int64_t p = threadIdx.x; p < P.positions; p += 256) {
        const float xh = ((float)x[p * P.x_position + c] - mean) * rstd;
        float z = xh * w + b;
        if (r) z += (float)r[p * P.r_position + c];
        float dz;
        by_act(P.act, [&](auto a) { dz = act_grad<decltype(a)::value>(P.slope, z, (float)dy[p * dy_position + c]); });
        a1 += dz;
        a2 += dz * xh;
      }
      a1 = block_sum<4>(a1, lds);
      a2 = block_sum<4>(a2, lds);
      if (threadIdx.x == 0) part[i * P.channels + c0 + c] = make_float2(a1, a2);
      s1 += w * a1;
      s2 += w * a2;
    }
    const float m1 = s1 / (float)m, m2 = s2 / (float)m;
    for (int64_t k = threadIdx.x; k < m; k += 256) {
      const int c = (int)(k % cpg);
      const int64_t p = k / cpg, o = (i * P.positions + p) * P.channels + c0 + c;
      const float w = P.weight ? load_any(P.weight, P.param_dtype, c0 + c) : 1.f;
      const float b = P.bias ? load_any(P.bias, P.param_dtype, c0 + c) : 0.f;
      const float xh = ((float)x[p * P.x_position + c] - mean) * rstd;
      float z = xh * w + b;
      if (r) z += (float)r[p * P.r_position + c];
      float dz;
      by_act(P.act, [&](auto a) { dz = act_grad<decltype(a)::value>(P.slope, z, (float)dy[p * dy_position + c]); });
      if (dr0) dr0[o] = (T)dz;
      if (dx0) dx0[o] = (T)(rstd * (dz * w - m1 - xh * m2));
    }
  }
}

// ---- host: group norm ---------------------------------------------------------------------------

// The widest vector that divides a row of channels
int norm_vec(int channels, int dtype) {
  const int most = dtype == GOENV_DT_F32 ? 4 : 8;
  if (channels % most == 0) return most;
  return dtype != GOENV_DT_F32 && channels % 2 == 0 ? 2 : 1;
}

struct NormPlan {
  NormCut cut;
  int threads, vec;
  size_t lds;      // bytes of the staging launches
  bool split;
  // Of a launch, whose threads are to stay below 2^31; more samples take several, one after the other
  int64_t samples_at_once() const { return INT32_MAX / threads / cut.slabs / cut.chunks; }
};

// `vec` 0: the widest vector; else what the arrays' alignment allows (the cut into slabs and chunks stays the same)
NormPlan norm_plan(int64_t n, int64_t positions, int channels, int groups, int dtype, bool residual, bool grad, int vec = 0) {
  NormPlan p;
  const int cpg = channels / groups, widest = norm_vec(channels, dtype), size = dtype == GOENV_DT_F32 ? 4 : 2;
  // Slabs are whole groups and whole vectors.  Wide ones: full cache lines of a position (128 bytes) where up to 384 bytes give them,
  // else up to 320 bytes (2,048 boards of 128 bf16 channels in 8 groups: 32 bytes 150 us, 64 bytes 124 us, 128 bytes
  // 124 us and the gradient 236 / 227 us; 378 boards of 240 channels in 24 groups: 80 bytes 51 us, 240 bytes 39 us).
  auto fits = [&](int gs) { return groups % gs == 0 && (gs * cpg) % widest == 0; };
  int least = 1;
  while (!fits(least)) ++least;
  int gs = least;
  for (int i = least; i <= groups && i * cpg * size <= 384; ++i) {
    if (!fits(i) || (i * cpg * size > 320 && (i * cpg * size) % 128)) continue;
    gs = i;
    if ((i * cpg * size) % 128 == 0) break;
  }
  auto vectors_at = [&](int threads, int64_t of) {   // of a thread
    const int rows = threads / (gs * cpg / widest);
    return rows ? (of + rows - 1) / rows : of;
  };
  // Fewer workgroups than CUs: slabs get narrower, to half lines at first.  If that leaves them too few or too long, the axis is cut
  // into chunks of eight vectors a thread instead (64 x 100 x 100 positions of 64 bf16 channels: 134 -> 66 us, 250 -> 139 us;
  // two images of 128 x 128 x 256 56 -> 16, 81 -> 26 us; 20 x 45 x 45 x 64, 16 vectors uncut and cut: 9 and 13, 17 and 23 us), or as few as
  // give each CU a workgroup, but three (64 x 64 x 512 with eight and three: 12.1 and 9.5 us, 21 and 16 us).  Half lines are as good while the slab is staged whole,
  // and keep the last round of workgroups short: the forward pass takes them, the gradient while it has few workgroups (512 boards
  // of 256 bf16 channels, forward: 70 us with lines, 67 with half lines; 2,048 boards of 128, the gradient: 227 and 238; 256
  // boards of 128 float32 channels, the gradient: 62 and 57).
  auto narrower = [&](int gs, int bytes) {   // the next one that is not below `bytes`, or the same
    for (int i = gs - 1; i >= least && i * cpg * size >= bytes; --i)
      if (fits(i)) return i;
    return gs;
  };
  auto wgs_of = [&](int gs) { return n * (groups / gs); };
  int64_t chunks = 1;
  if (wgs_of(gs) < 256) {
    const int wide = gs;
    while (wgs_of(gs) < 256 && narrower(gs, 64) != gs) gs = narrower(gs, 64);
    if (vectors_at(NORM_THREADS, positions) > 16) {
      gs = wide;
      const int64_t v = vectors_at(NORM_THREADS, positions), fair = (v * wgs_of(gs) + 255) / 256, each = fair < 3 ? 3 : fair > 8 ? 8 : fair;
      chunks = (v + each - 1) / each;
      const int64_t most = (2047 + wgs_of(gs)) / wgs_of(gs);
      if (chunks > most) chunks = most;
    } else {
      while (wgs_of(gs) < 256 && narrower(gs, 1) != gs) gs = narrower(gs, 1);
    }
  } else if ((!grad || wgs_of(gs) < 2048) && gs * cpg * size % 128 == 0) {
    for (int i = least; i < gs; ++i)
      if (fits(i) && i * cpg * size == 64) gs = i;
  }
  // As many threads as leave each a few vectors: six where there are many workgroups, but three in the forward pass while a vector lies
  // in one group (else the sums over a slab grow with the threads).  LDS for three workgroups of 512 threads on a CU in the
  // forward pass, two in the gradient whose sums need little of it; five or four smaller ones (2,048 boards of 128 bf16
  // channels, forward: 52 KB 123 us, 40 KB 126; the gradient 62 KB 227 us, 52 KB 235, but 1,000 boards of 120 float32 channels 50
  // and 45; 256 boards of 128 bf16 channels with 256 threads: 52 KB 34 us, 40 KB 28 us, with 512 threads 31).
  const int64_t of = (positions + chunks - 1) / chunks, wgs = wgs_of(gs) * chunks;
  const int few = wgs < 64 ? 2 : wgs < 512 || (!grad && cpg % widest == 0) ? 3 : 6;
  p.threads = 64;
  while (p.threads < NORM_THREADS && (p.threads < gs * cpg / widest || vectors_at(p.threads, of) > few)) p.threads *= 2;
  const bool pow2 = is_pow2(gs * cpg / widest);
  const int shared = p.threads == NORM_THREADS ? (grad && pow2 ? 62 << 10 : 52 << 10) : grad ? 40 << 10 : 32 << 10;
  // A CU that has one or two workgroups at most gives them all it has (30 images of 42 x 43 x 128 bf16, 240 workgroups: 52 KB 16 us, 152 KB
  // 14 us, the gradient 27 and 23)
  const int most = wgs <= 256 ? 152 << 10 : wgs <= 512 ? 76 << 10 : shared;
  NormCut& c = p.cut;
  p.vec = vec ? vec : widest;
  c.slab_groups = gs;
  c.width = gs * cpg;
  c.slabs = groups / gs;
  c.chunk = (positions + chunks - 1) / chunks;
  c.chunks = (int)((positions + c.chunk - 1) / c.chunk);
  c.units = c.width / p.vec;
  c.rows = p.threads / c.units;
  p.split = c.chunks > 1;
  if (c.rows == 0) return p;
  if (grad) {
    const int parts = c.units <= 64 && (c.units & (c.units - 1)) == 0 ? p.threads / 64 : c.rows <= 8 ? c.rows : c.rows / 2 > 8 ? c.rows / 2 : 8;
    const int sums = parts * c.width;
    c.scratch = 2 * c.width + 2 * gs + 2 * (sums > p.threads ? sums : p.threads);
  } else {
    c.scratch = p.threads * (cpg % p.vec == 0 ? 1 : p.vec) + 2 * gs;
  }
  c.scratch = (c.scratch + 3) & ~3;
  if (c.scratch * 4 > 64 << 10) {   // (a group of more than 4,090 channels: as one that is wider than a workgroup's vectors)
    c.rows = 0;
    return p;
  }
  const int64_t vectors = (c.chunk + c.rows - 1) / c.rows, row = (int64_t)p.threads * p.vec * size * (1 + grad + residual);
  const int64_t room = most > c.scratch * 4 ? (most - c.scratch * 4) / row : 0;
  c.staged = (int)(vectors < room ? vectors : room);
  p.lds = c.scratch * sizeof(float) + c.staged * row;
  return p;
}

// The cut into teams, or none (team 0).  `vec` 0: the widest vector; else what the arrays' alignment allows.
struct FewPlan {
  FewCut cut;
  int vec, nk;
};
FewPlan few_plan(int64_t n, int64_t positions, int channels, int groups, int dtype, bool grad, int vec = 0) {
  FewPlan p = {};
  const int cpg = channels / groups, most = dtype == GOENV_DT_F32 ? 4 : 8;
  p.vec = cpg % most == 0 ? most : dtype != GOENV_DT_F32 && cpg % 2 == 0 ? 2 : 1;
  if (vec && vec < p.vec) p.vec = vec;
  FewCut& c = p.cut;
  c.units = cpg / p.vec;
  // Vectors of 16 bytes: up to four of a lane in the forward pass, two in the gradient (2,048 boards of 7 x 7 x 128 bf16 channels in 8
  // groups, slabs against teams: 21 -> 15 us, 41 -> 34 us; 9 x 9, 1,024 of them: 17 -> 14, but 34 -> 43 us).  Narrower ones, whose loads
  // use a part of a cache line each: a few positions (16,384 samples of 128 bf16 channels in 32 groups, 16 positions: 123 -> 36 us,
  // 113 -> 91, but 25 of them 69 -> 45, 69 -> 91; of 120 float32 channels in 24 groups, 8 positions: 62 -> 53, 88 -> 86, but 16 of
  // them 72 -> 101, 123 -> 204).
  const int vectors = grad ? 2 : 4;
  if (c.units > 64 || (p.vec < most && positions > (p.vec == 1 ? 8 : 16))) return p;
  auto of_lane = [&](int team) { return (positions + team / c.units - 1) / (team / c.units); };
  int team = 1;
  while (team < c.units) team *= 2;
  const int want = n * groups <= 1024 ? 1 : vectors;   // (few teams: more lanes each; 64 boards of 5 x 5 4.3 -> 3.6 us)
  while (team < 64 && of_lane(team) > want) team *= 2;
  if (of_lane(team) > vectors) return p;
  c.team = team;
  c.rows = team / c.units;
  p.nk = of_lane(team) > 2 ? 4 : (int)of_lane(team);
  const int teams = FEW_THREADS / team;
  c.slab_groups = groups < teams ? groups : teams;
  c.slabs = (groups + c.slab_groups - 1) / c.slab_groups;
  c.slots = teams / c.slab_groups;
  c.strides = (n + c.slots - 1) / c.slots;
  // A workgroup takes several samples where there are many, for its weights (65,536 x 512 bf16 features: 35 -> 25 us) and its channel
  // sums: the more rows of them, the longer k_group_norm_param_grad reads.
  auto most_workgroups = [&](int64_t workgroups) {
    const int64_t strides = (workgroups + c.slabs - 1) / c.slabs;
    if (c.strides > strides) c.strides = strides;
  };
  const int64_t eight_samples = c.strides / 8 * c.slabs;   // workgroups that take eight each
  most_workgroups(!grad ? 4096 : eight_samples > 2048 ? 2048 : eight_samples < 512 ? 512 : eight_samples);
  return p;
}
// f(vectors of a lane)
template <typename F>
void by_vectors(int nk, F f) {
  if (nk == 1) f(Int<1>());
  else if (nk == 2) f(Int<2>());
  else f(Int<4>());
}

// The widest vector that the arrays' alignment allows
int norm_fit(const goenv_norm* a, const void* dy, int64_t dy_sample, int64_t dy_position, const void* o1, const void* o2) {
  const int size = a->dtype == GOENV_DT_F32 ? 4 : 2, vec = norm_vec(a->channels, a->dtype);
  auto fits = [&](int v) {
    int64_t all = (int64_t)(uintptr_t)a->x | (int64_t)(uintptr_t)a->residual | (int64_t)(uintptr_t)dy | (int64_t)(uintptr_t)o1 | (int64_t)(uintptr_t)o2;
    all |= (a->x_sample | a->x_position | dy_sample | dy_position) * size;
    if (a->residual) all |= (a->r_sample | a->r_position) * size;
    return (all & (v * size - 1)) == 0;
  };
  return fits(vec) ? vec : vec > 2 && size == 2 && fits(2) ? 2 : 1;
}

// f(vector width)
template <typename T, typename F>
void by_vec(int vec, F f) {
  if (vec == 1) return f(Int<1>());
  if constexpr (sizeof(T) == 2)
    if (vec == 2) return f(Int<2>());
  f(Int<16 / sizeof(T)>());
}

int check_norm(const goenv_norm* p, bool grad) {
  if (!p) return fail("goenv_group_norm_act: p is NULL");
  if (!is_dtype(p->dtype)) return fail("goenv_group_norm_act: dtype must be GOENV_DT_F32, BF16 or F16");
  if (p->param_dtype != GOENV_DT_F32 && p->param_dtype != p->dtype)
    return fail("goenv_group_norm_act: param_dtype must be GOENV_DT_F32 or dtype");
  if (p->n < 0 || p->positions < 0 || p->channels < 0) return fail("goenv_group_norm_act: a size is negative");
  if (p->positions > INT32_MAX || p->channels > 1 << 24)
    return fail("goenv_group_norm_act: more than 2^31 - 1 positions or 2^24 channels");
  if (p->groups <= 0 || p->channels % p->groups) return fail("goenv_group_norm_act: groups must divide channels");
  if (p->act < GOENV_ACT_NONE || p->act > GOENV_ACT_SILU) return fail("goenv_group_norm_act: act must be a GOENV_ACT_*");
  if (!(p->eps >= 0.f) || isinf(p->eps)) return fail("goenv_group_norm_act: eps must be finite and not negative");
  if (p->act == GOENV_ACT_LEAKY_RELU && !isfinite(p->slope)) return fail("goenv_group_norm_act: slope must be finite");
  if (p->n == 0 || p->positions == 0 || p->channels == 0) return 0;
  if (!p->x) return fail("goenv_group_norm_act: x is required");
  if (grad && !p->stats) return fail("goenv_group_norm_act_grad: the forward pass's stats are required");
  if (!aligned(p->x, p->dtype) || !aligned(p->residual, p->dtype) || !aligned(p->weight, p->param_dtype) ||
      !aligned(p->bias, p->param_dtype) || !aligned(p->stats, GOENV_DT_F32))
    return fail("goenv_group_norm_act: an array is not aligned to its elements");
  const int64_t need = goenv_group_norm_workspace(p->n, p->positions, p->channels, p->groups, p->dtype, grad);
  if (need > 0 && (!p->workspace || (int64_t)p->workspace_bytes < need || ((uintptr_t)p->workspace & 15)))
    return fail("goenv_group_norm_act: the workspace is too small or not 16-byte aligned (goenv_group_norm_workspace)");
  return 0;
}
// `n` samples from `first` on (their workspace apart)
goenv_norm norm_from(const goenv_norm& p, int64_t first, int64_t n) {
  const int64_t size = p.dtype == GOENV_DT_F32 ? 4 : 2;
  goenv_norm q = p;
  q.n = n;
  q.x = past(p.x, first * p.x_sample * size);
  q.residual = past(p.residual, first * p.r_sample * size);
  q.stats = past(p.stats, first * p.groups * 8);
  return q;
}
goenv_norm with_act(const goenv_norm* p) {
  goenv_norm q = *p;
  if (q.act == GOENV_ACT_LEAKY_RELU && q.slope == 0.f) q.act = GOENV_ACT_RELU;
  return q;
}

}  // namespace

extern "C" {

int64_t goenv_group_norm_workspace(int64_t n, int64_t positions, int channels, int groups, int dtype, int grad) {
  if (n <= 0 || positions <= 0 || channels <= 0 || groups <= 0 || channels % groups) return 0;
  const NormPlan plan = norm_plan(n, positions, channels, groups, dtype, true, grad);
  if (grad) {
    int64_t rows = n * plan.cut.chunks;
    for (int vec : {0, 1, 2}) {
      const FewPlan few = few_plan(n, positions, channels, groups, dtype, true, vec);
      if (few.cut.team && few.cut.strides > rows) rows = few.cut.strides;
    }
    return rows * channels * (int64_t)sizeof(float2);
  }
  return plan.split ? n * plan.cut.chunks * groups * (int64_t)sizeof(float2) : 0;
}

int goenv_group_norm_act(const goenv_norm* p, void* y, void* stream) {
  if (check_norm(p, false)) return -1;
  if (p->n == 0 || p->positions == 0 || p->channels == 0) return 0;
  if (!y || !aligned(y, p->dtype)) return fail("goenv_group_norm_act: y is required, aligned to its elements");
  ON_DEVICE(p->device, "goenv_group_norm_act");
  const goenv_norm q = with_act(p);
  const FewPlan few = few_plan(q.n, q.positions, q.channels, q.groups, q.dtype, false, norm_fit(&q, nullptr, 0, 0, y, nullptr));
  if (few.cut.team) {
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      by_vec<T>(few.vec, [&](auto v) {
        by_vectors(few.nk, [&](auto k) {
          constexpr int VEC = decltype(v)::value, NK = decltype(k)::value;
          auto go = [&](auto f) {
            hipLaunchKernelGGL(f, dim3((unsigned)(few.cut.strides * few.cut.slabs)), dim3(FEW_THREADS), 0, S(stream), q, few.cut, static_cast<T*>(y));
          };
          q.residual ? go(k_group_norm_few<T, VEC, NK, true>) : go(k_group_norm_few<T, VEC, NK, false>);
        });
      });
    });
    HIPCHK(hipGetLastError());
    return 0;
  }
  const NormPlan plan = norm_plan(q.n, q.positions, q.channels, q.groups, q.dtype, q.residual != nullptr, false, norm_fit(&q, nullptr, 0, 0, y, nullptr));
  if (plan.cut.rows == 0) {
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL((k_group_norm_any<T>), dim3(grid_of(q.n * q.groups)), dim3(256), 0, S(stream), q, static_cast<T*>(y));
    });
    HIPCHK(hipGetLastError());
    return 0;
  }
  const int64_t each = plan.samples_at_once(), sample = q.positions * q.channels * (q.dtype == GOENV_DT_F32 ? 4 : 2);
  if (each == 0) return fail("goenv_group_norm_act: too many groups for one launch");
  for (int64_t first = 0; first < q.n; first += each) {
    const goenv_norm part = norm_from(q, first, each < q.n - first ? each : q.n - first);
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      by_vec<T>(plan.vec, [&](auto v) {
        constexpr int VEC = decltype(v)::value;
        const dim3 grid((unsigned)(part.n * plan.cut.slabs * plan.cut.chunks)), block(plan.threads);
        const bool one = (q.channels / q.groups) % VEC == 0;
        auto go = [&](auto f) { hipLaunchKernelGGL(f, grid, block, plan.lds, S(stream), part, plan.cut, static_cast<T*>(past(y, first * sample))); };
        auto with = [&](auto o, auto r) {
          constexpr bool ONE = decltype(o)::value, RES = decltype(r)::value;
          if (!plan.split) {
            go(k_group_norm<T, VEC, ONE, RES, NORM_WHOLE>);
          } else {
            go(k_group_norm<T, VEC, ONE, false, NORM_SUMS>);
            go(k_group_norm<T, VEC, ONE, RES, NORM_APPLY>);
          }
        };
        if (one) q.residual ? with(Int<1>(), Int<1>()) : with(Int<1>(), Int<0>());
        else q.residual ? with(Int<0>(), Int<1>()) : with(Int<0>(), Int<0>());
      });
    });
    HIPCHK(hipGetLastError());
  }
  return 0;
}

int goenv_group_norm_act_grad(const goenv_norm* p, const void* dy, int64_t dy_sample, int64_t dy_position, void* dx, void* dresidual,
                              void* dweight, void* dbias, void* stream) {
  if (check_norm(p, true)) return -1;
  if (p->channels == 0) return 0;
  const bool empty = p->n == 0 || p->positions == 0;
  if (!empty && (!dy || !aligned(dy, p->dtype) || !aligned(dx, p->dtype) || !aligned(dresidual, p->dtype)))
    return fail("goenv_group_norm_act_grad: dy is required, and the arrays aligned to their elements");
  ON_DEVICE(p->device, "goenv_group_norm_act_grad");
  const goenv_norm q = with_act(p);
  NormPlan plan = {};
  FewPlan few = {};
  if (!empty) few = few_plan(q.n, q.positions, q.channels, q.groups, q.dtype, true, norm_fit(&q, dy, dy_sample, dy_position, dx, dresidual));
  if (few.cut.team) {
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      by_vec<T>(few.vec, [&](auto v) {
        by_vectors(few.nk, [&](auto k) {
          constexpr int VEC = decltype(v)::value, NK = decltype(k)::value;
          auto go = [&](auto f) {
            hipLaunchKernelGGL(f, dim3((unsigned)(few.cut.strides * few.cut.slabs)), dim3(FEW_THREADS), 0, S(stream), q, few.cut,
                               static_cast<const T*>(dy), dy_sample, dy_position, static_cast<T*>(dx), static_cast<T*>(dresidual));
          };
          q.residual ? go(k_group_norm_few_grad<T, VEC, NK, true>) : go(k_group_norm_few_grad<T, VEC, NK, false>);
        });
      });
    });
    HIPCHK(hipGetLastError());
  } else if (!empty) {
    plan = norm_plan(q.n, q.positions, q.channels, q.groups, q.dtype, q.residual != nullptr, true, norm_fit(&q, dy, dy_sample, dy_position, dx, dresidual));
    if (plan.cut.rows == 0) {
      plan.cut.chunks = 1;
      by_dtype(p->dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((k_group_norm_any_grad<T>), dim3(grid_of(q.n * q.groups)), dim3(256), 0, S(stream), q, static_cast<const T*>(dy),
                           dy_sample, dy_position, static_cast<T*>(dx), static_cast<T*>(dresidual));
      });
      HIPCHK(hipGetLastError());
    } else {
      const int64_t each = plan.samples_at_once(), size = q.dtype == GOENV_DT_F32 ? 4 : 2, sample = q.positions * q.channels * size;
      if (each == 0) return fail("goenv_group_norm_act_grad: too many groups for one launch");
      for (int64_t first = 0; first < q.n; first += each) {
        goenv_norm part = norm_from(q, first, each < q.n - first ? each : q.n - first);
        part.workspace = past(q.workspace, first * plan.cut.chunks * q.channels * (int64_t)sizeof(float2));
        const void* g = past(dy, first * dy_sample * size);
        void *gx = past(dx, first * sample), *gr = past(dresidual, first * sample);
        by_dtype(p->dtype, [&](auto t) {
          using T = decltype(t);
          by_vec<T>(plan.vec, [&](auto v) {
            constexpr int VEC = decltype(v)::value;
            const dim3 grid((unsigned)(part.n * plan.cut.slabs * plan.cut.chunks)), block(plan.threads);
            auto go = [&](auto f) {
              hipLaunchKernelGGL(f, grid, block, plan.lds, S(stream), part, plan.cut, static_cast<const T*>(g), dy_sample, dy_position,
                                 static_cast<T*>(gx), static_cast<T*>(gr));
            };
            auto with = [&](auto r) {
              constexpr bool RES = decltype(r)::value;
              if (!plan.split) {
                go(k_group_norm_grad<T, VEC, RES, NORM_WHOLE>);
              } else {
                go(k_group_norm_grad<T, VEC, RES, NORM_SUMS>);
                if (dx || dresidual) go(k_group_norm_grad<T, VEC, RES, NORM_APPLY>);
              }
            };
            q.residual ? with(Int<1>()) : with(Int<0>());
          });
        });
        HIPCHK(hipGetLastError());
      }
    }
  }
  if (dweight || dbias) {
    hipLaunchKernelGGL(k_group_norm_param_grad, dim3((q.channels + 15) / 16), dim3(1024), 0, S(stream),
                       static_cast<const float2*>(q.workspace), empty ? 0 : few.cut.team ? few.cut.strides : q.n * plan.cut.chunks, q.channels, q.param_dtype, dweight, dbias);
    HIPCHK(hipGetLastError());
  }
  return 0;
}

}  // extern "C"
