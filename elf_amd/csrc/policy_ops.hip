// The policy network's operators around its convolutions: group norm with the residual sum and the activation
// (channels last), dropout from a counter-based generator, masks / penalties / biases on policy logits.
// Interface and definitions: include/goenv.h.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/goenv.h"
#include "goenv_host.h"

using namespace goenv;

namespace {

template <int DT>
struct ElemOf;
template <>
struct ElemOf<GOENV_DT_F32> { using type = float; };
template <>
struct ElemOf<GOENV_DT_BF16> { using type = __bf16; };
template <>
struct ElemOf<GOENV_DT_F16> { using type = _Float16; };

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

// Sum over a workgroup of WAVES waves, in the same order every time; every thread gets it.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float* lds) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) t += lds[w];
  return t;
}
template <int WAVES>
__device__ __forceinline__ float block_max(float v, float* lds) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) t = fmaxf(t, lds[w]);
  return t;
}

// ---- group norm ---------------------------------------------------------------------------------

__device__ __forceinline__ float act_of(int act, float slope, float z) {
  if (act == GOENV_ACT_SILU) return z / (1.f + __expf(-z));
  if (z > 0.f) return z;
  return slope == 0.f ? (z != z ? z : 0.f) : z * slope;
}
__device__ __forceinline__ float act_grad(int act, float slope, float z) {
  if (act == GOENV_ACT_SILU) {
    const float s = 1.f / (1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  return z > 0.f ? 1.f : slope;
}

template <typename T>
__global__ __launch_bounds__(256) void k_group_norm(goenv_norm P, T* y) {
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
      o[p * P.channels + c] = (T)act_of(P.act, P.slope, z);
    }
  }
}

// dx and dresidual of one sample's group, and its channels' part of dbias and dweight into workspace [n][channels][2]
template <typename T>
__global__ __launch_bounds__(256) void k_group_norm_grad(goenv_norm P, const T* dy0, int64_t dy_sample, int64_t dy_position, T* dx0,
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
        const float dz = (float)dy[p * dy_position + c] * act_grad(P.act, P.slope, z);
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
      const float dz = (float)dy[p * dy_position + c] * act_grad(P.act, P.slope, z);
      if (dr0) dr0[o] = (T)dz;
      if (dx0) dx0[o] = (T)(rstd * (dz * w - m1 - xh * m2));
    }
  }
}

__global__ __launch_bounds__(256) void k_group_norm_param_grad(const float2* part, int64_t rows, int channels, int param_dtype, void* dweight,
                                                               void* dbias) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= channels) return;
  float a = 0.f, b = 0.f;
  for (int64_t i = 0; i < rows; ++i) {
    const float2 v = part[i * channels + c];
    a += v.x;
    b += v.y;
  }
  if (dbias) store_any(dbias, param_dtype, c, a);
  if (dweight) store_any(dweight, param_dtype, c, b);
}

// ---- dropout ------------------------------------------------------------------------------------

// Philox4x32-10: ten rounds of two 32 x 32 -> 64 products, crossed over and keyed.
__device__ __forceinline__ uint4 philox(uint64_t block, uint32_t step, uint32_t site, uint64_t seed) {
  uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = step, d = site;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
    a = (uint32_t)(q >> 32) ^ b ^ k0;
    b = (uint32_t)q;
    c = (uint32_t)(p >> 32) ^ d ^ k1;
    d = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(a, b, c, d);
}

template <typename T>
__global__ __launch_bounds__(256) void k_dropout(int64_t n, const T* x, const T* residual, T* y, uint32_t thr, float scale,
                                                 const int64_t* rng, uint32_t site) {
  const uint64_t seed = (uint64_t)rng[0];
  const uint32_t step = (uint32_t)rng[1];
  for (int64_t blk = (int64_t)blockIdx.x * 256 + threadIdx.x; blk < (n + 7) / 8; blk += (int64_t)gridDim.x * 256) {
    const uint4 u = philox((uint64_t)blk, step, site, seed);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t e = blk * 8 + j;
      if (e >= n) break;
      const uint32_t bits = j < 4 ? w[j] & 0xffffu : w[j - 4] >> 16;
      float v = bits >= thr ? (float)x[e] * scale : 0.f;
      if (residual) v += (float)residual[e];
      y[e] = (T)v;
    }
  }
}

// ---- policy logits ------------------------------------------------------------------------------

constexpr int LOGIT_CHUNK = 4096;   // columns whose history counts are in LDS at a time

struct RowRules {
  float inv_rep, rep, presence, frequency, inv_t;
};
__device__ __forceinline__ RowRules rules_of(const goenv_logit_rules& P, int64_t row) {
  RowRules r;
  r.rep = P.row_repetition ? P.row_repetition[row] : P.repetition;
  r.presence = P.row_presence ? P.row_presence[row] : P.presence;
  r.frequency = P.row_frequency ? P.row_frequency[row] : P.frequency;
  r.inv_rep = 1.f / r.rep;
  r.inv_t = 1.f / (P.row_temperature ? P.row_temperature[row] : P.temperature);
  return r;
}
__device__ __forceinline__ bool allowed(const goenv_logit_rules& P, int64_t row, int64_t v) {
  if (P.legal) return P.legal[row * P.legal_row + v] != 0;
  if (P.legal_bits) return (P.legal_bits[row * P.bits_row + (v >> 5)] >> (v & 31)) & 1u;
  return true;
}
// z of a column, and dz / dlogit without the temperature in `slope`
template <typename T>
__device__ __forceinline__ float z_of(const goenv_logit_rules& P, const RowRules& r, int64_t row, int64_t v, int count, float& slope) {
  slope = 1.f;
  if (!allowed(P, row, v)) return -INFINITY;
  float a = (float)static_cast<const T*>(P.logits)[row * P.logits_row + v];
  if (count > 0) {
    slope = a > 0.f ? r.inv_rep : r.rep;
    a = a * slope - r.presence - r.frequency * (float)count;
  }
  if (P.bias) a += load_any(P.bias, P.bias_dtype, row * P.bias_row + v);
  return a * r.inv_t;
}
// counts of columns [v0, v0 + LOGIT_CHUNK) in the row's history
__device__ __forceinline__ void count_chunk(const goenv_logit_rules& P, int64_t row, int64_t v0, int* count) {
  __syncthreads();
  for (int k = threadIdx.x; k < LOGIT_CHUNK; k += 256) count[k] = 0;
  __syncthreads();
  if (P.history) {
    int len = P.history_len ? P.history_len[row] : P.history_max;
    len = len < 0 ? 0 : len > P.history_max ? P.history_max : len;
    for (int k = threadIdx.x; k < len; k += 256) {
      const int64_t at = row * P.history_row + k;
      const int64_t v = P.history_i64 ? static_cast<const int64_t*>(P.history)[at] : static_cast<const int32_t*>(P.history)[at];
      if (v >= v0 && v < v0 + LOGIT_CHUNK && v < P.cols) atomicAdd(&count[v - v0], 1);
    }
  }
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(256) void k_policy_logits(goenv_logit_rules P, void* out) {
  __shared__ int count[LOGIT_CHUNK];
  __shared__ float lds[4];
  for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x) {
    const RowRules r = rules_of(P, row);
    float m = -INFINITY, s = 0.f, slope;
    if (P.out_kind != GOENV_OUT_LOGITS) {
      for (int64_t v0 = 0; v0 < P.cols; v0 += LOGIT_CHUNK) {
        count_chunk(P, row, v0, count);
        for (int64_t v = v0 + threadIdx.x; v < P.cols && v < v0 + LOGIT_CHUNK; v += 256) {
          const float z = z_of<T>(P, r, row, v, count[v - v0], slope);
          if (z == -INFINITY) continue;
          const float top = fmaxf(m, z);
          s = s * (m == -INFINITY ? 0.f : expf(m - top)) + expf(z - top);
          m = top;
        }
      }
      const float top = block_max<4>(m, lds);
      s = block_sum<4>(m == -INFINITY ? s : s * expf(m - top), lds);
      m = top == -INFINITY ? 0.f : top;
      if (P.stats && threadIdx.x == 0) {
        P.stats[2 * row] = m;
        P.stats[2 * row + 1] = s;
      }
    }
    const float log_s = logf(s), inv_s = 1.f / s;
    for (int64_t v0 = 0; v0 < P.cols; v0 += LOGIT_CHUNK) {
      count_chunk(P, row, v0, count);
      for (int64_t v = v0 + threadIdx.x; v < P.cols && v < v0 + LOGIT_CHUNK; v += 256) {
        const float z = z_of<T>(P, r, row, v, count[v - v0], slope);
        float o = z;
        if (P.out_kind == GOENV_OUT_PROBS) o = z == -INFINITY ? 0.f : expf(z - m) * inv_s;
        if (P.out_kind == GOENV_OUT_LOG_PROBS) o = z == -INFINITY ? z : z - m - log_s;
        store_any(out, P.out_dtype, row * P.cols + v, o);
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_policy_logits_grad(goenv_logit_rules P, const void* d_out, int64_t dy_row, T* dlogits, void* dbias,
                                                            float* dz_out) {
  __shared__ int count[LOGIT_CHUNK];
  __shared__ float lds[4];
  for (int64_t row = blockIdx.x; row < P.rows; row += gridDim.x) {
    const RowRules r = rules_of(P, row);
    float total = 0.f, m = 0.f, inv_s = 0.f, slope;
    if (P.out_kind != GOENV_OUT_LOGITS) {
      m = P.stats[2 * row];
      inv_s = 1.f / P.stats[2 * row + 1];
      for (int64_t v0 = 0; v0 < P.cols; v0 += LOGIT_CHUNK) {
        count_chunk(P, row, v0, count);
        for (int64_t v = v0 + threadIdx.x; v < P.cols && v < v0 + LOGIT_CHUNK; v += 256) {
          const float z = z_of<T>(P, r, row, v, count[v - v0], slope);
          if (z == -INFINITY) continue;
          const float dy = load_any(d_out, P.out_dtype, row * dy_row + v);
          total += P.out_kind == GOENV_OUT_PROBS ? dy * expf(z - m) * inv_s : dy;
        }
      }
      total = block_sum<4>(total, lds);
    }
    for (int64_t v0 = 0; v0 < P.cols; v0 += LOGIT_CHUNK) {
      count_chunk(P, row, v0, count);
      for (int64_t v = v0 + threadIdx.x; v < P.cols && v < v0 + LOGIT_CHUNK; v += 256) {
        const float z = z_of<T>(P, r, row, v, count[v - v0], slope);
        float dz = 0.f;
        if (z != -INFINITY) {
          dz = load_any(d_out, P.out_dtype, row * dy_row + v);
          if (P.out_kind == GOENV_OUT_PROBS) dz = expf(z - m) * inv_s * (dz - total);
          if (P.out_kind == GOENV_OUT_LOG_PROBS) dz -= expf(z - m) * inv_s * total;
          dz *= r.inv_t;
        } else {
          slope = 0.f;
        }
        if (dlogits) dlogits[row * P.cols + v] = (T)(z == -INFINITY ? 0.f : dz * slope);
        if (dz_out) dz_out[row * P.cols + v] = dz;
        else if (dbias) store_any(dbias, P.bias_dtype, row * P.cols + v, dz);
      }
    }
  }
}

__global__ __launch_bounds__(256) void k_column_sum(const float* part, int64_t rows, int64_t cols, int dtype, void* out) {
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < cols; v += (int64_t)gridDim.x * 256) {
    float a = 0.f;
    for (int64_t i = 0; i < rows; ++i) a += part[i * cols + v];
    store_any(out, dtype, v, a);
  }
}

// ---- host ---------------------------------------------------------------------------------------

bool is_dtype(int dt) { return dt == GOENV_DT_F32 || dt == GOENV_DT_BF16 || dt == GOENV_DT_F16; }
bool aligned(const void* p, int dt) { return ((uintptr_t)p & (dt == GOENV_DT_F32 ? 3 : 1)) == 0; }
unsigned grid_of(int64_t items, int64_t most = 1 << 20) { return (unsigned)(items < most ? items : most); }

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

int check_norm(const goenv_norm* p, bool grad) {
  if (!p) return fail("goenv_group_norm_act: p is NULL");
  if (!is_dtype(p->dtype)) return fail("goenv_group_norm_act: dtype must be GOENV_DT_F32, BF16 or F16");
  if (p->param_dtype != GOENV_DT_F32 && p->param_dtype != p->dtype)
    return fail("goenv_group_norm_act: param_dtype must be GOENV_DT_F32 or dtype");
  if (p->n < 0 || p->positions < 0 || p->channels < 0) return fail("goenv_group_norm_act: a size is negative");
  if (p->groups <= 0 || p->channels % p->groups) return fail("goenv_group_norm_act: groups must divide channels");
  if (p->act < GOENV_ACT_NONE || p->act > GOENV_ACT_SILU) return fail("goenv_group_norm_act: act must be a GOENV_ACT_*");
  if (!(p->eps >= 0.f) || isinf(p->eps)) return fail("goenv_group_norm_act: eps must be finite and not negative");
  if (p->act == GOENV_ACT_LEAKY_RELU && !isfinite(p->slope)) return fail("goenv_group_norm_act: slope must be finite");
  if (p->n == 0 || p->positions == 0 || p->channels == 0) return 0;
  if (!p->x) return fail("goenv_group_norm_act: x is required");
  if (grad && !p->stats) return fail("goenv_group_norm_act_grad: the forward pass's stats are required");
  if (!aligned(p->x, p->dtype) || !aligned(p->residual, p->dtype) || !aligned(p->weight, p->param_dtype) ||
      !aligned(p->bias, p->param_dtype))
    return fail("goenv_group_norm_act: an array is not aligned to its elements");
  const int64_t need = goenv_group_norm_workspace(p->n, p->positions, p->channels, p->groups, p->dtype, grad);
  if (need > 0 && (!p->workspace || (int64_t)p->workspace_bytes < need || ((uintptr_t)p->workspace & 15)))
    return fail("goenv_group_norm_act: the workspace is too small or not 16-byte aligned (goenv_group_norm_workspace)");
  return 0;
}
goenv_norm with_slope(const goenv_norm* p) {
  goenv_norm q = *p;
  if (q.act == GOENV_ACT_NONE) q.slope = 1.f;
  if (q.act == GOENV_ACT_RELU) q.slope = 0.f;
  return q;
}

int check_logits(const goenv_logit_rules* p, bool grad) {
  if (!p) return fail("goenv_policy_logits: p is NULL");
  if (!is_dtype(p->dtype)) return fail("goenv_policy_logits: dtype must be GOENV_DT_F32, BF16 or F16");
  if (p->out_dtype != GOENV_DT_F32 && p->out_dtype != p->dtype)
    return fail("goenv_policy_logits: out_dtype must be GOENV_DT_F32 or dtype");
  if (p->bias && p->bias_dtype != GOENV_DT_F32 && p->bias_dtype != p->dtype)
    return fail("goenv_policy_logits: bias_dtype must be GOENV_DT_F32 or dtype");
  if (p->out_kind < GOENV_OUT_LOGITS || p->out_kind > GOENV_OUT_PROBS) return fail("goenv_policy_logits: out_kind must be a GOENV_OUT_*");
  if (p->rows < 0 || p->cols < 0 || p->cols > INT32_MAX) return fail("goenv_policy_logits: rows or cols out of range");
  if (p->legal && p->legal_bits) return fail("goenv_policy_logits: legal or legal_bits, not both");
  if (p->history && p->history_max < 0) return fail("goenv_policy_logits: history_max is negative");
  if (!p->row_temperature && !(p->temperature > 0.f && isfinite(p->temperature)))
    return fail("goenv_policy_logits: temperature must be positive and finite");
  if (p->history) {
    if (!p->row_repetition && !(p->repetition > 0.f && isfinite(p->repetition)))
      return fail("goenv_policy_logits: repetition must be positive and finite");
    if ((!p->row_presence && !isfinite(p->presence)) || (!p->row_frequency && !isfinite(p->frequency)))
      return fail("goenv_policy_logits: presence and frequency must be finite");
  }
  if (p->rows == 0 || p->cols == 0) return 0;
  if (!p->logits) return fail("goenv_policy_logits: logits is required");
  if (grad && p->out_kind != GOENV_OUT_LOGITS && !p->stats)
    return fail("goenv_policy_logits_grad: the forward pass's stats are required");
  if (!aligned(p->logits, p->dtype) || !aligned(p->bias, p->bias_dtype) || ((uintptr_t)p->legal_bits & 3) ||
      ((uintptr_t)p->history & (p->history_i64 ? 7 : 3)))
    return fail("goenv_policy_logits: an array is not aligned to its elements");
  const int64_t need = goenv_policy_logits_workspace(p->rows, p->cols, p->out_kind, p->bias && p->bias_row == 0, grad);
  if (need > 0 && (!p->workspace || (int64_t)p->workspace_bytes < need || ((uintptr_t)p->workspace & 15)))
    return fail("goenv_policy_logits: the workspace is too small or not 16-byte aligned (goenv_policy_logits_workspace)");
  return 0;
}

}  // namespace

extern "C" {

int64_t goenv_group_norm_workspace(int64_t n, int64_t positions, int channels, int groups, int dtype, int grad) {
  (void)positions, (void)groups, (void)dtype;
  return grad ? n * channels * (int64_t)sizeof(float2) : 0;
}

int goenv_group_norm_act(const goenv_norm* p, void* y, void* stream) {
  if (check_norm(p, false)) return -1;
  if (p->n == 0 || p->positions == 0 || p->channels == 0) return 0;
  if (!y || !aligned(y, p->dtype)) return fail("goenv_group_norm_act: y is required, aligned to its elements");
  ON_DEVICE(p->device, "goenv_group_norm_act");
  const goenv_norm q = with_slope(p);
  by_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_group_norm<T>), dim3(grid_of(q.n * q.groups)), dim3(256), 0, S(stream), q, static_cast<T*>(y));
  });
  HIPCHK(hipGetLastError());
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
  const goenv_norm q = with_slope(p);
  if (!empty) {
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL((k_group_norm_grad<T>), dim3(grid_of(q.n * q.groups)), dim3(256), 0, S(stream), q, static_cast<const T*>(dy),
                         dy_sample, dy_position, static_cast<T*>(dx), static_cast<T*>(dresidual));
    });
    HIPCHK(hipGetLastError());
  }
  if (dweight || dbias) {
    hipLaunchKernelGGL(k_group_norm_param_grad, dim3((q.channels + 255) / 256), dim3(256), 0, S(stream),
                       static_cast<const float2*>(q.workspace), empty ? 0 : q.n, q.channels, q.param_dtype, dweight, dbias);
    HIPCHK(hipGetLastError());
  }
  return 0;
}

int goenv_dropout(int device, int dtype, int64_t n, const void* x, const void* residual, void* y, double p, const int64_t* rng,
                  uint32_t site, void* stream) {
  if (!is_dtype(dtype)) return fail("goenv_dropout: dtype must be GOENV_DT_F32, BF16 or F16");
  if (n < 0) return fail("goenv_dropout: n is negative");
  if (!(p >= 0. && p <= 1.)) return fail("goenv_dropout: p must be between 0 and 1");
  if (n == 0) return 0;
  if (!x || !y || !rng) return fail("goenv_dropout: x, y and rng are required");
  if (!aligned(x, dtype) || !aligned(residual, dtype) || !aligned(y, dtype) || ((uintptr_t)rng & 7))
    return fail("goenv_dropout: an array is not aligned to its elements");
  ON_DEVICE(device, "goenv_dropout");
  const uint32_t thr = (uint32_t)floor(p * 65536. + 0.5);
  const float scale = thr >= 65536u ? 0.f : (float)(65536. / (65536. - thr));
  by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_dropout<T>), dim3(grid_of(((n + 7) / 8 + 255) / 256)), dim3(256), 0, S(stream), n, static_cast<const T*>(x),
                       static_cast<const T*>(residual), static_cast<T*>(y), thr, scale, rng, site);
  });
  HIPCHK(hipGetLastError());
  return 0;
}

int64_t goenv_policy_logits_workspace(int64_t rows, int64_t cols, int out_kind, int shared_bias, int grad) {
  (void)out_kind;
  return grad && shared_bias ? rows * cols * (int64_t)sizeof(float) : 0;
}

int goenv_policy_logits(const goenv_logit_rules* p, void* out, void* stream) {
  if (check_logits(p, false)) return -1;
  if (p->rows == 0 || p->cols == 0) return 0;
  if (!out || !aligned(out, p->out_dtype)) return fail("goenv_policy_logits: out is required, aligned to its elements");
  ON_DEVICE(p->device, "goenv_policy_logits");
  by_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((k_policy_logits<T>), dim3(grid_of(p->rows)), dim3(256), 0, S(stream), *p, out);
  });
  HIPCHK(hipGetLastError());
  return 0;
}

int goenv_policy_logits_grad(const goenv_logit_rules* p, const void* d_out, int64_t dy_row, void* dlogits, void* dbias, void* stream) {
  if (check_logits(p, true)) return -1;
  if (dbias && !p->bias) return fail("goenv_policy_logits_grad: dbias without a bias");
  if (p->cols == 0) return 0;
  const bool shared = dbias && p->bias_row == 0;
  if (p->rows > 0 && (!d_out || !aligned(d_out, p->out_dtype) || !aligned(dlogits, p->dtype) || !aligned(dbias, p->bias_dtype)))
    return fail("goenv_policy_logits_grad: d_out is required, and the arrays aligned to their elements");
  ON_DEVICE(p->device, "goenv_policy_logits_grad");
  if (p->rows > 0) {
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL((k_policy_logits_grad<T>), dim3(grid_of(p->rows)), dim3(256), 0, S(stream), *p, d_out, dy_row,
                         static_cast<T*>(dlogits), dbias, shared ? static_cast<float*>(p->workspace) : nullptr);
    });
    HIPCHK(hipGetLastError());
  }
  if (shared) {
    hipLaunchKernelGGL(k_column_sum, dim3(grid_of((p->cols + 255) / 256)), dim3(256), 0, S(stream), static_cast<const float*>(p->workspace),
                       p->rows, p->cols, p->bias_dtype, dbias);
    HIPCHK(hipGetLastError());
  }
  return 0;
}

}  // extern "C"
