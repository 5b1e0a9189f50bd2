// Dropout from a counter-based generator, and masks / penalties / biases on policy logits (a policy network's operators).
// Interface and definitions: include/goenv.h.
#include <type_traits>

#include "policy_device.h"

using namespace goenv;

namespace {

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

// Bound by memory (11.8 million bf16 elements and a residual: 71 MB, 13 us; without the residual 47 MB, 11 us) as long as the generator
// stays behind it: 20 products for eight elements of 16 bits each.  32 bits an element would double them, and a stored mask
// would have to be written and read.  Whole 16-byte vectors a thread, and a block's bits are made while its loads are under way.
template <typename T>
struct alignas(16) Eight {
  T v[8];
};

// A block of eight elements a thread and turn; VECTOR: the arrays allow 16-byte accesses.
template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void k_dropout(int64_t n, const T* x, const T* residual, T* y, uint32_t thr, float scale,
                                                 const int64_t* rng, uint32_t site) {
  const uint64_t seed = (uint64_t)rng[0];
  const uint32_t step = (uint32_t)rng[1];
  for (int64_t blk = (int64_t)blockIdx.x * 256 + threadIdx.x; blk < (n + 7) / 8; blk += (int64_t)gridDim.x * 256) {
    const int64_t e = blk * 8;
    const bool whole = VECTOR && e + 8 <= n;
    Eight<T> a, r;
    if (whole) {
      a = *reinterpret_cast<const Eight<T>*>(x + e);
      if (residual) r = *reinterpret_cast<const Eight<T>*>(residual + e);
    }
    const uint4 u = philox((uint64_t)blk, step, site, seed);   // under way while the loads are
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    auto keep = [&](int j) { return (j < 4 ? w[j] & 0xffffu : w[j - 4] >> 16) >= thr; };
    if (whole) {
      Eight<T> o;
      if (residual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = (T)((keep(j) ? (float)a.v[j] * scale : 0.f) + (float)r.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o.v[j] = (T)(keep(j) ? (float)a.v[j] * scale : 0.f);
      }
      *reinterpret_cast<Eight<T>*>(y + e) = o;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (e + j >= n) break;
        float v = keep(j) ? (float)x[e + j] * scale : 0.f;
        if (residual) v += (float)residual[e + j];
        y[e + j] = (T)v;
      }
    }
  }
}

// ---- policy logits ------------------------------------------------------------------------------
//
// A row's columns are cut into slices of threads x NI vectors of VEC columns, one workgroup each, with the slice's columns
// in registers; how often a column stands in the row's history is counted in LDS (integers: the order does not matter).  Bound by
// memory for many rows or long ones, by latency for a short one; so a row that fits one slice takes one launch and reads everything
// once (8,192 rows of 361 bf16 columns with a mask and a history: 7.1 us, bound by instructions, some 285 a wave and row, since a row
// that is no multiple of four columns goes element by element; 64 rows of 131,072 with histories of 2,048, no softmax: 36 MB, 10.9 us =
// 3.3 TB/s, where every slice scans the row's whole history).  Longer rows take a launch for the slices' maxima and sums and one that joins them and computes z again, which costs
// reading the logits a second time (from the caches) instead of writing and reading z in 32 bits (one row of 131,072:
// 4.3 and 4.1 us, of which a launch by itself takes 2).

struct LogitCut {
  int threads;             // of a slice
  int slices, per_group;   // slices of a row; rows that one workgroup takes one after the other
  int64_t groups;          // of rows
};
// The threads that share a slice: a workgroup, or (WAVE) one of its waves -- short rows go four to a workgroup, without barriers.
template <bool WAVE>
struct Team {
  int tid, threads;
  uint32_t index;
  __device__ __forceinline__ explicit Team(const LogitCut& cut) : tid(WAVE ? threadIdx.x & 63 : threadIdx.x), threads(WAVE ? 64 : cut.threads) {
    index = WAVE ? blockIdx.x * 4 + wave() : blockIdx.x;
  }
  // (the same for all lanes, and known to be: a row's addresses and rules are scalars)
  __device__ __forceinline__ static int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
  __device__ __forceinline__ void sync() const {
    if (WAVE) {   // a wave's accesses to LDS keep their order; the compiler has to keep it too
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  }
  // Over the team, the same order every time.  lds: 16 floats.
  __device__ __forceinline__ float sum(float v, float* lds) const {
    v = wave_sum(v);
    return WAVE ? v : across(v, lds, [](float a, float b) { return a + b; });
  }
  __device__ __forceinline__ float max(float v, float* lds) const {
    v = wave_max(v);
    return WAVE ? v : across(v, lds, fmaxf);
  }
  template <typename F>
  __device__ __forceinline__ float across(float v, float* lds, F f) const {
    const int waves = threads >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int w = 1; w < waves; ++w) v = f(v, lds[w]);
    return v;
  }
};
enum LogitMode { LOGIT_MAP, LOGIT_WHOLE, LOGIT_SUMS, LOGIT_APPLY };   // no softmax; softmax in one launch, or in two

struct RowRules {
  float inv_rep, rep, presence, frequency, inv_t;
};
// A scalar argument as a register's value: left as a place in memory, the choice between it and a row's value becomes a choice between
// two addresses, and the arguments are copied to the stack for it.
__device__ __forceinline__ float in_register(float v) {
  asm("" : "+s"(v));
  return v;
}
__device__ __forceinline__ RowRules rules_of(const goenv_logit_rules& P, int64_t row) {
  RowRules r;
  float t;
  if (P.row_repetition && P.row_presence && P.row_frequency && P.row_temperature) {   // the loads are under way together
    r.rep = P.row_repetition[row];
    r.presence = P.row_presence[row];
    r.frequency = P.row_frequency[row];
    t = P.row_temperature[row];
  } else {
    r.rep = in_register(P.repetition);
    r.presence = in_register(P.presence);
    r.frequency = in_register(P.frequency);
    t = in_register(P.temperature);
    if (P.row_repetition) r.rep = P.row_repetition[row];
    if (P.row_presence) r.presence = P.row_presence[row];
    if (P.row_frequency) r.frequency = P.row_frequency[row];
    if (P.row_temperature) t = P.row_temperature[row];
  }
  r.inv_rep = 1.f / r.rep;
  r.inv_t = 1.f / t;
  return r;
}

// A row's start (a scalar) and an offset in bytes below 2^32: one addition to a load
template <typename P>
__device__ __forceinline__ P* in_row(const void* row, uint32_t bytes) {
  return reinterpret_cast<P*>(const_cast<char*>(static_cast<const char*>(row)) + bytes);
}

// NI vectors of an array of type F32 or T, the row at element `at`.  The columns behind the last vector read that one again.
template <typename E, int VEC, int NI>
__device__ __forceinline__ void load_row(const E* row, const uint32_t (&col)[NI], float (&to)[NI][VEC]) {
  Pack<E, VEC> v[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) v[k] = *in_row<const Pack<E, VEC>>(row, col[k] * (uint32_t)sizeof(E));
#pragma unroll
  for (int k = 0; k < NI; ++k)
#pragma unroll
    for (int j = 0; j < VEC; ++j) to[k][j] = (float)v[k].v[j];
}
template <typename T, int VEC, int NI>
__device__ __forceinline__ void load_columns(const void* p, bool f32, int64_t at, const uint32_t (&col)[NI], float (&to)[NI][VEC]) {
  if (f32) load_row<float, VEC, NI>(static_cast<const float*>(p) + at, col, to);
  else load_row<T, VEC, NI>(static_cast<const T*>(p) + at, col, to);
}
template <typename E, int VEC, int NI>
__device__ __forceinline__ void store_row(E* row, const uint32_t (&col)[NI], const bool (&in)[NI], const float (&from)[NI][VEC]) {
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    Pack<E, VEC> v;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v.v[j] = (E)from[k][j];
    if (in[k]) *in_row<Pack<E, VEC>>(row, col[k] * (uint32_t)sizeof(E)) = v;
  }
}
template <typename T, int VEC, int NI>
__device__ __forceinline__ void store_columns(void* p, bool f32, int64_t at, const uint32_t (&col)[NI], const bool (&in)[NI], const float (&from)[NI][VEC]) {
  if (f32) store_row<float, VEC, NI>(static_cast<float*>(p) + at, col, in, from);
  else store_row<T, VEC, NI>(static_cast<T*>(p) + at, col, in, from);
}

// This thread's columns of a slice of a row: z (-inf where it is off or behind the row's end); in `seen` and `up` a bit per column,
// whether it stands in the history and whether its logit is above zero (what dz / dlogit goes by); returns the
// row's rules.  count: LDS, a word per column of the slice; every thread of the team calls.  have_bias: `bias` is loaded already.
// All loads start before anything waits for one: a short row's time is the time of its longest chain of loads.
template <typename T, int VEC, int NI, bool WAVE>
__device__ __forceinline__ RowRules slice_of(const goenv_logit_rules& P, const Team<WAVE>& team, int64_t row, uint32_t v0, const uint32_t (&col)[NI],
                                             const bool (&in)[NI], int* count, float (&z)[NI][VEC], uint32_t& seen, uint32_t& up, bool have_bias,
                                             float (&bias)[NI][VEC]) {
  const T* logits = static_cast<const T*>(P.logits) + row * P.logits_row;
  Pack<T, VEC> raw[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) raw[k] = *in_row<const Pack<T, VEC>>(logits, col[k] * (uint32_t)sizeof(T));
  uint32_t mask[NI];
  if (P.legal) {
    const uint8_t* legal = P.legal + row * P.legal_row;
#pragma unroll
    for (int k = 0; k < NI; ++k) mask[k] = VEC == 4 ? *in_row<const uint32_t>(legal, col[k]) : *in_row<const uint8_t>(legal, col[k]);
  } else if (P.legal_bits) {
    const uint32_t* bits = P.legal_bits + row * P.bits_row;
#pragma unroll
    for (int k = 0; k < NI; ++k) mask[k] = *in_row<const uint32_t>(bits, (col[k] >> 5) * 4);
  }
  if (P.bias && !have_bias) load_columns<T, VEC, NI>(P.bias, P.bias_dtype == GOENV_DT_F32, row * P.bias_row, col, bias);
  seen = up = 0;
  const bool past = P.history && P.history_max > 0;
  const uint32_t width = (uint32_t)(NI * VEC * team.threads), left = (uint32_t)P.cols - v0, most = width < left ? width : left;
  RowRules r;
  if (past) {
    auto scan = [&](auto* h) {
      using I = std::remove_const_t<std::remove_pointer_t<decltype(h)>>;
      using U = std::make_unsigned_t<I>;
      I v[4];
      auto load = [&](int k) {   // four entries at a time
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = k + i * team.threads;
          v[i] = *in_row<const I>(h, (uint32_t)(at < P.history_max ? at : P.history_max - 1) * (uint32_t)sizeof(I));
        }
      };
      load(team.tid);            // before the row's length is here
      int len = P.history_len ? P.history_len[row] : P.history_max;
      len = len < 0 ? 0 : len > P.history_max ? P.history_max : len;
      r = rules_of(P, row);
      team.sync();               // the row before has read its counts
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) count[(k * team.threads + team.tid) * VEC + j] = 0;
      team.sync();
      for (int k = team.tid; k < len;) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const U at = (U)v[i] - (U)v0;   // (negative entries are far beyond every column)
          if (k + i * team.threads < len && at < most) atomicAdd(&count[at], 1);
        }
        k += 4 * team.threads;
        if (k < len) load(k);
      }
    };
    if (P.history_i64) scan(static_cast<const int64_t*>(P.history) + row * P.history_row);
    else scan(static_cast<const int32_t*>(P.history) + row * P.history_row);
    team.sync();
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int c = count[(k * team.threads + team.tid) * VEC + j];
        const float l = (float)raw[k].v[j], f = l > 0.f ? r.inv_rep : r.rep;
        seen |= (uint32_t)(c > 0) << (k * VEC + j);
        up |= (uint32_t)(l > 0.f) << (k * VEC + j);
        z[k][j] = c > 0 ? l * f - r.presence - r.frequency * (float)c : l;
      }
  } else {
    r = rules_of(P, row);
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) z[k][j] = (float)raw[k].v[j];
  }
  if (P.bias)
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) z[k][j] += bias[k][j];
  auto finish = [&](auto allowed) {
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) z[k][j] = (int)allowed(k, j) & (int)in[k] ? z[k][j] * r.inv_t : -INFINITY;
  };
  if (P.legal) finish([&](int k, int j) { return (mask[k] & (0xffu << (8 * j))) != 0; });
  else if (P.legal_bits) finish([&](int k, int j) { return ((mask[k] >> ((col[k] + j) & 31)) & 1u) != 0; });
  else finish([](int, int) { return true; });
  return r;
}

template <int VEC, int NI, bool WAVE>
__device__ __forceinline__ void columns_of(const goenv_logit_rules& P, const Team<WAVE>& team, int v0, uint32_t (&col)[NI], bool (&in)[NI]) {
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const uint32_t v = (uint32_t)v0 + (uint32_t)(k * team.threads + team.tid) * VEC, cols = (uint32_t)P.cols;
    in[k] = v < cols;
    col[k] = in[k] ? v : cols - VEC;
  }
}

// The workspace of the two launches: a row's slices' (largest z, sum exp(z - largest)).
template <typename T, int VEC, int NI, bool WAVE, int MODE>
__global__ __launch_bounds__(1024) void k_policy_logits(goenv_logit_rules P, LogitCut cut, void* out) {
  extern __shared__ __align__(16) int counts[];
  __shared__ float lds[16];
  const Team<WAVE> team(cut);
  const uint32_t slices = cut.slices, at = team.index / slices;
  const int64_t row = at;
  if (WAVE && row >= P.rows) return;
  const int slice = (int)(team.index - at * slices), v0 = slice * NI * VEC * team.threads;
  int* count = counts + (WAVE ? team.wave() * NI * VEC * 64 : 0);
  uint32_t col[NI];
  bool in[NI];
  columns_of<VEC, NI>(P, team, v0, col, in);
  float z[NI][VEC], bias[NI][VEC];
  uint32_t seen, up;
  slice_of<T, VEC, NI>(P, team, row, v0, col, in, count, z, seen, up, false, bias);
  if (MODE != LOGIT_MAP) {
    float m = -INFINITY, s = 0.f;
    if (MODE != LOGIT_APPLY) {
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = fmaxf(m, z[k][j]);
      m = team.max(m, lds);
      if (m == -INFINITY) m = 0.f;    // nothing left: every exponential is 0
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += __expf(z[k][j] - m);
      s = team.sum(s, lds);
    }
    float2* part = static_cast<float2*>(P.workspace) + row * cut.slices;
    if (MODE == LOGIT_SUMS) {
      if (team.tid == 0) part[slice] = make_float2(s == 0.f ? -INFINITY : m, s);
      return;
    }
    if (MODE == LOGIT_APPLY) {
      // every wave joins the slices by itself
      const int lane = threadIdx.x & 63;
      for (int k = lane; k < cut.slices; k += 64) m = fmaxf(m, part[k].x);
      m = wave_max(m);
      if (m == -INFINITY) m = 0.f;
      for (int k = lane; k < cut.slices; k += 64) s += part[k].y == 0.f ? 0.f : part[k].y * __expf(part[k].x - m);
      s = wave_sum(s);
    }
    if (P.stats && slice == 0 && team.tid == 0) {
      P.stats[2 * row] = m;
      P.stats[2 * row + 1] = s;
    }
    if (P.out_kind == GOENV_OUT_PROBS) {
      const float inv_s = 1.f / s;
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[k][j] = z[k][j] == -INFINITY ? 0.f : __expf(z[k][j] - m) * inv_s;
    } else {
      const float log_s = logf(s);
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) z[k][j] = z[k][j] == -INFINITY ? -INFINITY : z[k][j] - m - log_s;
    }
  }
  store_columns<T, VEC, NI>(out, P.out_dtype == GOENV_DT_F32, row * P.cols, col, in, z);
}

// The gradients.  SHARED: of a bias that all rows share too -- a workgroup then takes several rows one after the other and
// keeps the sums of dz.  The workspace: a row's slices' sums of dy (log probabilities) or p dy (probabilities), then the
// row groups' sums of dz.
template <typename T, int VEC, int NI, bool WAVE, bool SHARED, int MODE>
__global__ __launch_bounds__(1024) void k_policy_logits_grad(goenv_logit_rules P, LogitCut cut, const void* d_out, int64_t dy_row, T* dlogits,
                                                             void* dbias, float* shared) {
  extern __shared__ __align__(16) int counts[];
  __shared__ float lds[16];
  const Team<WAVE> team(cut);
  const uint32_t slices = cut.slices, at = team.index / slices;
  const int64_t group = at;
  if (WAVE && group >= cut.groups) return;
  const int slice = (int)(team.index - at * slices), v0 = slice * NI * VEC * team.threads;
  int* count = counts + (WAVE ? team.wave() * NI * VEC * 64 : 0);
  uint32_t col[NI];
  bool in[NI];
  columns_of<VEC, NI>(P, team, v0, col, in);
  float sum[SHARED ? NI : 1][VEC], bias[NI][VEC];
  if (SHARED) {
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[k][j] = 0.f;
    load_columns<T, VEC, NI>(P.bias, P.bias_dtype == GOENV_DT_F32, 0, col, bias);
  }
  const int64_t first = SHARED ? group * cut.per_group : group;
  const int64_t end = !SHARED ? first + 1 : first + cut.per_group < P.rows ? first + cut.per_group : P.rows;
  for (int64_t row = first; row < end; ++row) {
    float z[NI][VEC], dz[NI][VEC];
    uint32_t seen, up;
    load_columns<T, VEC, NI>(d_out, P.out_dtype == GOENV_DT_F32, row * dy_row, col, dz);
    const RowRules r = slice_of<T, VEC, NI>(P, team, row, v0, col, in, count, z, seen, up, SHARED, bias);
    if (MODE != LOGIT_MAP) {
      const float m = P.stats[2 * row], inv_s = 1.f / P.stats[2 * row + 1];
      const bool probs = P.out_kind == GOENV_OUT_PROBS;
      float total = 0.f;
      float* part = static_cast<float*>(P.workspace) + row * cut.slices;
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {   // z becomes p
          const bool off = z[k][j] == -INFINITY;
          dz[k][j] = off ? 0.f : dz[k][j];
          z[k][j] = off ? 0.f : __expf(z[k][j] - m) * inv_s;
        }
      if (MODE != LOGIT_APPLY) {
        if (probs) {
#pragma unroll
          for (int k = 0; k < NI; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) total += z[k][j] * dz[k][j];
        } else {
#pragma unroll
          for (int k = 0; k < NI; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j) total += dz[k][j];
        }
        total = team.sum(total, lds);
      } else {
        for (int k = threadIdx.x & 63; k < cut.slices; k += 64) total += part[k];
        total = wave_sum(total);
      }
      if (MODE == LOGIT_SUMS) {
        if (team.tid == 0) part[slice] = total;
        continue;
      }
      if (probs) {
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int j = 0; j < VEC; ++j) dz[k][j] = z[k][j] * (dz[k][j] - total);
      } else {
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int j = 0; j < VEC; ++j) dz[k][j] -= z[k][j] * total;
      }
    } else {
#pragma unroll
      for (int k = 0; k < NI; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) dz[k][j] = z[k][j] == -INFINITY ? 0.f : dz[k][j];
    }
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        dz[k][j] *= r.inv_t;
        if (SHARED) sum[k][j] += dz[k][j];
      }
    if (dbias && !SHARED) store_columns<T, VEC, NI>(dbias, P.bias_dtype == GOENV_DT_F32, row * P.cols, col, in, dz);
    if (dlogits) {
      if (seen)
#pragma unroll
        for (int k = 0; k < NI; ++k)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const uint32_t bit = 1u << (k * VEC + j);
            if (dz[k][j] != 0.f) dz[k][j] *= (seen & bit) == 0 ? 1.f : (up & bit) ? r.inv_rep : r.rep;   // (0 stays 0 whatever the factor)
          }
      store_columns<T, VEC, NI>(dlogits, sizeof(T) == 4, row * P.cols, col, in, dz);
    }
  }
  if constexpr (SHARED)
    if (MODE != LOGIT_SUMS) store_columns<float, VEC, NI>(shared, true, group * P.cols, col, in, sum);
}

// Column sums of [rows][cols]: 1 << log_wide columns a workgroup, as many rows at a time as its threads are for.
__global__ __launch_bounds__(1024) void k_column_sum(const float* part, int64_t rows, int64_t cols, int log_wide, int dtype, void* out) {
  __shared__ float lds[1024];
  const int wide = 1 << log_wide, down = (int)blockDim.x >> log_wide, row = (int)threadIdx.x >> log_wide;
  const int64_t v = (int64_t)blockIdx.x * wide + (threadIdx.x & (wide - 1));
  float a = 0.f;
  if (v < cols)
#pragma unroll 4
    for (int64_t i = row; i < rows; i += down) a += part[i * cols + v];
  lds[threadIdx.x] = a;
  __syncthreads();
  if (row != 0 || v >= cols) return;
  for (int i = 1; i < down; ++i) a += lds[threadIdx.x + i * wide];
  store_any(out, dtype, v, a);
}

__device__ __forceinline__ int64_t row_of(int64_t i, uint32_t width) {   // (64-bit divisions take ten times as long)
  return i >> 32 ? i / width : (uint32_t)i / width;
}

// Dense copies of the rules that a gradient reads again: the mask as bits, the histories and their lengths.  Bound by the launch for a batch
// of boards, by memory for long rows (768 x 361 bytes and four moves a row 2.9 us, 8,192 x 361 and eight moves 3.5, 64 x 131,072 and 2,048 moves
// 4.2).  A thread makes a word of 32 bytes, loaded by 16 from wherever they start (a wave that makes two words of 64 bytes took 7.3 us for
// the second case).
__global__ __launch_bounds__(256) void k_keep_rules(goenv_logit_rules P, int64_t mask_rows, int64_t past_rows, uint32_t* bits, void* history,
                                                    int32_t* history_len) {
  const int64_t thread = (int64_t)blockIdx.x * 256 + threadIdx.x, threads = (int64_t)gridDim.x * 256;
  const uint32_t words = (uint32_t)(P.cols + 31) / 32;
  if (bits && P.legal) {
    for (int64_t i = thread; i < mask_rows * words; i += threads) {
      const int64_t row = row_of(i, words);
      const uint32_t w = (uint32_t)(i - row * words), cols = (uint32_t)P.cols - w * 32;
      const uint32_t before = cols < 32 && w ? 32 - cols : 0;   // the last word takes the row's last 32 bytes
      const uint8_t* from = P.legal + row * P.legal_row + w * 32 - before;
      uint32_t b[8] = {}, word = 0;
      if (P.cols >= 32) {
        __builtin_memcpy(b, from, 32);
      } else {
        for (uint32_t k = 0; k < cols; ++k) word |= (uint32_t)(from[k] != 0) << k;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t v = b[k] | (b[k] >> 4 & 0x0f0f0f0fu);   // a byte's lowest bit: whether any of its bits is set
        v |= v >> 2 & 0x03030303u;
        v = (v | v >> 1) & 0x01010101u;
        word |= ((v | v >> 7 | v >> 14 | v >> 21) & 15u) << (4 * k);
      }
      bits[i] = word >> before;
    }
  } else if (bits) {
    for (int64_t i = thread; i < mask_rows * words; i += threads) {
      const int64_t row = row_of(i, words);
      bits[i] = P.legal_bits[row * P.bits_row + (i - row * words)];
    }
  }
  if (history) {
    auto copy = [&](auto* from, auto* to) {
      for (int64_t i = thread; i < past_rows * P.history_max; i += threads) {
        const int64_t row = row_of(i, (uint32_t)P.history_max);
        to[i] = from[row * P.history_row + (i - row * P.history_max)];
      }
    };
    if (P.history_i64) copy(static_cast<const int64_t*>(P.history), static_cast<int64_t*>(history));
    else copy(static_cast<const int32_t*>(P.history), static_cast<int32_t*>(history));
  }
  if (history_len)
    for (int64_t i = thread; i < P.rows; i += threads) history_len[i] = P.history_len[i];
}

// ---- host: policy logits --------------------------------------------------------------------------

struct LogitPlan {
  LogitCut cut;
  int threads, vec, ni;
  bool split, wave;   // wave: a wave a slice, four a workgroup
  unsigned blocks(int64_t teams) const { return (unsigned)(wave ? (teams + 3) / 4 : teams); }
  // Of a launch, whose threads are to stay below 2^31; more rows take several, one after the other (and the workspace in turn)
  int64_t rows_at_once() const { return (int64_t)(INT32_MAX / threads) * (wave ? 4 : 1) / cut.slices; }
};

// The cut for vectors of `vec` columns (which goes by the arrays' alignment: a workspace is sized for either).
LogitPlan logit_plan(int64_t rows, int64_t cols, bool softmax, bool shared, int vec) {
  LogitPlan p;
  p.vec = vec;
  p.ni = vec == 1 ? 6 : shared ? 2 : 4;   // (the sums of a shared bias's gradient and the bias itself are in registers too)
  if (vec == 1 && softmax && !shared && cols > 6 * 1024 && cols <= 12 * 1024) p.ni = 12;
  // (one launch instead of two: 498 rows of 12,001 bf16 columns 24 -> 16 us, 243 of 6,702 float32 ones 12.5 -> 7.6, the gradient 14 -> 10;
  // with the sums of a shared bias besides they would not fit the registers)
  const int each = p.ni * vec;             // columns of a thread
  p.split = softmax && cols > 1024 * each;
  // As few slices as there can be, all of about the same length (1,732 rows of 3,307 float32 columns: slices of a power of two of
  // threads 37 us, of 576 threads 24 us)
  const int most = p.split || !softmax ? 256 : 1024;
  const int64_t fewest = (cols + (int64_t)most * each - 1) / ((int64_t)most * each), length = (cols + fewest - 1) / fewest;
  p.threads = (int)((length + 64 * each - 1) / (64 * each)) * 64;
  p.cut.threads = p.threads;
  p.wave = p.threads == 64;
  if (p.wave) p.threads = 256;
  p.cut.slices = (int)((cols + (int64_t)p.cut.threads * each - 1) / ((int64_t)p.cut.threads * each));
  p.cut.per_group = 1;
  if (shared) {
    // no more rows in a group than leave half a million threads at work
    const int64_t teams = rows * p.cut.slices, want = (1 << 19) / p.cut.threads, per = (teams + want - 1) / want;
    p.cut.per_group = (int)(per < 1 ? 1 : per > rows ? rows : per);
  }
  p.cut.groups = (rows + p.cut.per_group - 1) / p.cut.per_group;
  return p;
}

int64_t size_of(int dt) { return dt == GOENV_DT_F32 ? 4 : 2; }
// The rules of `rows` rows from `first` on
goenv_logit_rules rules_from(const goenv_logit_rules& p, int64_t first, int64_t rows) {
  goenv_logit_rules q = p;
  q.rows = rows;
  q.logits = past(p.logits, first * p.logits_row * size_of(p.dtype));
  q.legal = past(p.legal, first * p.legal_row);
  q.legal_bits = past(p.legal_bits, first * p.bits_row * 4);
  q.bias = past(p.bias, first * p.bias_row * size_of(p.bias_dtype));
  q.history = past(p.history, first * p.history_row * (p.history_i64 ? 8 : 4));
  q.history_len = past(p.history_len, first * 4);
  q.row_repetition = past(p.row_repetition, first * 4);
  q.row_presence = past(p.row_presence, first * 4);
  q.row_frequency = past(p.row_frequency, first * 4);
  q.row_temperature = past(p.row_temperature, first * 4);
  q.stats = past(p.stats, first * 8);
  return q;
}

// Whether all arrays allow vectors of four columns
bool logit_fours(const goenv_logit_rules* p, const void* d_out, int64_t dy_row, const void* o1, int o1_dtype, const void* o2, int o2_dtype) {
  auto fits = [](const void* a, int dt, int64_t row) {
    const int64_t size = dt == GOENV_DT_F32 ? 4 : 2;
    return a == nullptr || ((((int64_t)(uintptr_t)a) | (row * size)) & (4 * size - 1)) == 0;
  };
  return p->cols % 4 == 0 && fits(p->logits, p->dtype, p->logits_row) && fits(p->bias, p->bias_dtype, p->bias_row) &&
         fits(d_out, p->out_dtype, dy_row) && fits(o1, o1_dtype, p->cols) && fits(o2, o2_dtype, p->cols) &&
         (p->legal == nullptr || (((uintptr_t)p->legal | (uintptr_t)p->legal_row) & 3) == 0);
}

int check_logits(const goenv_logit_rules* p, bool grad) {
  if (!p) return fail("goenv_policy_logits: p is NULL");
  if (!is_dtype(p->dtype)) return fail("goenv_policy_logits: dtype must be GOENV_DT_F32, BF16 or F16");
  if (p->out_dtype != GOENV_DT_F32 && p->out_dtype != p->dtype)
    return fail("goenv_policy_logits: out_dtype must be GOENV_DT_F32 or dtype");
  if (p->bias && p->bias_dtype != GOENV_DT_F32 && p->bias_dtype != p->dtype)
    return fail("goenv_policy_logits: bias_dtype must be GOENV_DT_F32 or dtype");
  if (p->out_kind < GOENV_OUT_LOGITS || p->out_kind > GOENV_OUT_PROBS) return fail("goenv_policy_logits: out_kind must be a GOENV_OUT_*");
  if (p->rows < 0 || p->cols < 0 || p->cols > (1 << 28)) return fail("goenv_policy_logits: rows or cols out of range");
  if (p->legal && p->legal_bits) return fail("goenv_policy_logits: legal or legal_bits, not both");
  if (p->history && (p->history_max < 0 || p->history_max > (1 << 28))) return fail("goenv_policy_logits: history_max out of range");
  auto divides = [](float v) { return v > 0.f && isfinite(v) && isfinite(1.f / v); };   // (the kernels multiply by the inverse)
  if (!p->row_temperature && !divides(p->temperature))
    return fail("goenv_policy_logits: temperature must be positive and finite, with a finite inverse");
  if (p->history) {
    if (!p->row_repetition && !divides(p->repetition))
      return fail("goenv_policy_logits: repetition must be positive and finite, with a finite inverse");
    if ((!p->row_presence && !isfinite(p->presence)) || (!p->row_frequency && !isfinite(p->frequency)))
      return fail("goenv_policy_logits: presence and frequency must be finite");
  }
  if (p->rows == 0 || p->cols == 0) return 0;
  if (!p->logits) return fail("goenv_policy_logits: logits is required");
  if (grad && p->out_kind != GOENV_OUT_LOGITS && !p->stats)
    return fail("goenv_policy_logits_grad: the forward pass's stats are required");
  const uintptr_t words = (uintptr_t)p->legal_bits | (uintptr_t)p->history_len | (uintptr_t)p->stats | (uintptr_t)p->row_repetition |
                          (uintptr_t)p->row_presence | (uintptr_t)p->row_frequency | (uintptr_t)p->row_temperature;
  if (!aligned(p->logits, p->dtype) || !aligned(p->bias, p->bias_dtype) || (words & 3) ||
      ((uintptr_t)p->history & (p->history_i64 ? 7 : 3)))
    return fail("goenv_policy_logits: an array is not aligned to its elements");
  const int64_t need = goenv_policy_logits_workspace(p->rows, p->cols, p->out_kind, p->bias && p->bias_row == 0, grad);
  if (need > 0 && (!p->workspace || (int64_t)p->workspace_bytes < need || ((uintptr_t)p->workspace & 15)))
    return fail("goenv_policy_logits: the workspace is too small or not 16-byte aligned (goenv_policy_logits_workspace)");
  return 0;
}

}  // namespace

extern "C" {

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
    const bool vector = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & 15) == 0;
    auto go = [&](auto f) {
      hipLaunchKernelGGL(f, dim3(grid_of(((n + 7) / 8 + 255) / 256)), dim3(256), 0, S(stream), n, static_cast<const T*>(x),
                         static_cast<const T*>(residual), static_cast<T*>(y), thr, scale, rng, site);
    };
    vector ? go(k_dropout<T, true>) : go(k_dropout<T, false>);
  });
  HIPCHK(hipGetLastError());
  return 0;
}

int64_t goenv_policy_logits_workspace(int64_t rows, int64_t cols, int out_kind, int shared_bias, int grad) {
  if (rows <= 0 || cols <= 0) return 0;
  const bool softmax = out_kind != GOENV_OUT_LOGITS;
  int64_t most = 0;
  for (int vec : {1, 4}) {
    const LogitPlan p = logit_plan(rows, cols, softmax, grad && shared_bias, vec);
    int64_t need = p.split ? rows * p.cut.slices * (int64_t)(grad ? sizeof(float) : sizeof(float2)) : 0;
    if (grad && shared_bias) need = ((need + 15) & ~15) + p.cut.groups * cols * (int64_t)sizeof(float);
    most = need > most ? need : most;
  }
  return most;
}

int goenv_policy_logits(const goenv_logit_rules* p, void* out, void* stream) {
  if (check_logits(p, false)) return -1;
  if (p->rows == 0 || p->cols == 0) return 0;
  if (!out || !aligned(out, p->out_dtype)) return fail("goenv_policy_logits: out is required, aligned to its elements");
  const bool softmax = p->out_kind != GOENV_OUT_LOGITS;
  const LogitPlan plan = logit_plan(p->rows, p->cols, softmax, false, logit_fours(p, nullptr, 0, out, p->out_dtype, nullptr, 0) ? 4 : 1);
  ON_DEVICE(p->device, "goenv_policy_logits");
  for (int64_t first = 0, each = plan.rows_at_once(); first < p->rows; first += each) {
    const goenv_logit_rules q = rules_from(*p, first, each < p->rows - first ? each : p->rows - first);
    void* to = past(out, first * p->cols * size_of(p->out_dtype));
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      auto with = [&](auto v, auto n) {
        constexpr int VEC = decltype(v)::value, NI = decltype(n)::value;
        const size_t lds = p->history ? (size_t)plan.threads * VEC * NI * sizeof(int) : 0;
        auto go = [&](auto f) {
          hipLaunchKernelGGL(f, dim3(plan.blocks(q.rows * plan.cut.slices)), dim3(plan.threads), lds, S(stream), q, plan.cut, to);
        };
        if constexpr (VEC == 1 && NI == 12) {
          go(k_policy_logits<T, VEC, NI, false, LOGIT_WHOLE>);
        } else if (!softmax) {
          plan.wave ? go(k_policy_logits<T, VEC, NI, true, LOGIT_MAP>) : go(k_policy_logits<T, VEC, NI, false, LOGIT_MAP>);
        } else if (!plan.split) {
          plan.wave ? go(k_policy_logits<T, VEC, NI, true, LOGIT_WHOLE>) : go(k_policy_logits<T, VEC, NI, false, LOGIT_WHOLE>);
        } else {
          go(k_policy_logits<T, VEC, NI, false, LOGIT_SUMS>);
          go(k_policy_logits<T, VEC, NI, false, LOGIT_APPLY>);
        }
      };
      plan.vec == 4 ? with(Int<4>(), Int<4>()) : plan.ni == 12 ? with(Int<1>(), Int<12>()) : with(Int<1>(), Int<6>());
    });
    HIPCHK(hipGetLastError());
  }
  return 0;
}

int goenv_policy_logits_grad(const goenv_logit_rules* p, const void* d_out, int64_t dy_row, void* dlogits, void* dbias, void* stream) {
  if (check_logits(p, true)) return -1;
  if (dbias && !p->bias) return fail("goenv_policy_logits_grad: dbias without a bias");
  if (p->cols == 0) return 0;
  const bool shared = dbias && p->bias_row == 0, softmax = p->out_kind != GOENV_OUT_LOGITS;
  if (p->rows > 0 && (!d_out || !aligned(d_out, p->out_dtype) || !aligned(dlogits, p->dtype) || !aligned(dbias, p->bias_dtype)))
    return fail("goenv_policy_logits_grad: d_out is required, and the arrays aligned to their elements");
  const LogitPlan plan = logit_plan(p->rows, p->cols, softmax, shared,
                                    logit_fours(p, d_out, dy_row, dlogits, p->dtype, shared ? nullptr : dbias, p->bias_dtype) ? 4 : 1);
  ON_DEVICE(p->device, "goenv_policy_logits_grad");
  const int64_t sums = plan.split ? (p->rows * plan.cut.slices * (int64_t)sizeof(float) + 15) & ~15 : 0;
  float* parts = shared ? reinterpret_cast<float*>(static_cast<char*>(p->workspace) + sums) : nullptr;
  // (the gradient of a shared bias takes all rows in one launch: a workgroup has as many as it takes)
  for (int64_t first = 0, each = shared ? p->rows : plan.rows_at_once(); first < p->rows; first += each) {
    const goenv_logit_rules q = rules_from(*p, first, each < p->rows - first ? each : p->rows - first);
    LogitCut cut = plan.cut;
    if (!shared) cut.groups = q.rows;
    const void* dy = past(d_out, first * dy_row * size_of(p->out_dtype));
    void* dl = past(dlogits, first * p->cols * size_of(p->dtype));
    void* db = past(dbias, first * p->cols * size_of(p->bias_dtype));
    by_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      auto with = [&](auto v, auto n, auto b) {
        constexpr int VEC = decltype(v)::value, NI = decltype(n)::value;
        constexpr bool SHARED = decltype(b)::value;
        const size_t lds = p->history ? (size_t)plan.threads * VEC * NI * sizeof(int) : 0;
        auto go = [&](auto f) {
          hipLaunchKernelGGL(f, dim3(plan.blocks(cut.groups * cut.slices)), dim3(plan.threads), lds, S(stream), q, cut, dy, dy_row,
                             static_cast<T*>(dl), db, parts);
        };
        auto launch = [&](auto w) {
          constexpr bool WAVE = decltype(w)::value;
          if constexpr (VEC == 1 && NI == 12) {
            if constexpr (!WAVE) go(k_policy_logits_grad<T, VEC, NI, WAVE, SHARED, LOGIT_WHOLE>);
          } else if (!softmax) {
            go(k_policy_logits_grad<T, VEC, NI, WAVE, SHARED, LOGIT_MAP>);
          } else if (!plan.split) {
            go(k_policy_logits_grad<T, VEC, NI, WAVE, SHARED, LOGIT_WHOLE>);
          } else if constexpr (!WAVE) {
            go(k_policy_logits_grad<T, VEC, NI, WAVE, SHARED, LOGIT_SUMS>);
            go(k_policy_logits_grad<T, VEC, NI, WAVE, SHARED, LOGIT_APPLY>);
          }
        };
        plan.wave ? launch(Int<1>()) : launch(Int<0>());
      };
      if (plan.vec == 4) shared ? with(Int<4>(), Int<2>(), Int<1>()) : with(Int<4>(), Int<4>(), Int<0>());
      else if (plan.ni == 12) with(Int<1>(), Int<12>(), Int<0>());
      else shared ? with(Int<1>(), Int<6>(), Int<1>()) : with(Int<1>(), Int<6>(), Int<0>());
    });
    HIPCHK(hipGetLastError());
  }
  if (shared) {
    // wide enough to be read in whole lines, narrow enough for a workgroup on every CU, and rows for the threads that are left (32 rows of
    // 131,072: 16 columns a workgroup 20 us, 256 columns 5 us)
    const int64_t rows = p->rows > 0 ? plan.cut.groups : 0;
    int log_wide = 8, down = 1;
    while (log_wide > 4 && p->cols < ((int64_t)256 << log_wide)) --log_wide;
    const int wide = 1 << log_wide;
    while (wide * down < 1024 && 4 * down < rows) down *= 2;
    if (wide * down < 64) down = 64 / wide;
    hipLaunchKernelGGL(k_column_sum, dim3((unsigned)((p->cols + wide - 1) / wide)), dim3(wide * down), 0, S(stream), parts, rows, p->cols, log_wide,
                       p->bias_dtype, dbias);
    HIPCHK(hipGetLastError());
  }
  return 0;
}

int goenv_policy_logits_keep(const goenv_logit_rules* p, uint32_t* legal_bits, void* history, int32_t* history_len, void* stream) {
  if (!p) return fail("goenv_policy_logits_keep: p is NULL");
  if (p->rows < 0 || p->cols < 0 || p->cols > (1 << 28)) return fail("goenv_policy_logits_keep: rows or cols out of range");
  if (p->legal && p->legal_bits) return fail("goenv_policy_logits_keep: legal or legal_bits, not both");
  if (p->history && (p->history_max < 0 || p->history_max > (1 << 28))) return fail("goenv_policy_logits_keep: history_max out of range");
  if ((legal_bits && !p->legal && !p->legal_bits) || (history && !p->history) || (history_len && !p->history_len))
    return fail("goenv_policy_logits_keep: a copy of an array that p does not have");
  const uintptr_t entry = p->history_i64 ? 7 : 3;
  if ((((uintptr_t)legal_bits | (uintptr_t)p->legal_bits | (uintptr_t)history_len | (uintptr_t)p->history_len) & 3) ||
      (((uintptr_t)history | (uintptr_t)p->history) & entry))
    return fail("goenv_policy_logits_keep: an array is not aligned to its elements");
  const int64_t mask_rows = legal_bits ? ((p->legal ? p->legal_row : p->bits_row) == 0 && p->rows > 0 ? 1 : p->rows) : 0;
  const int64_t past_rows = history ? (p->history_row == 0 && p->rows > 0 ? 1 : p->rows) : 0;
  const int64_t mask = mask_rows * ((p->cols + 31) / 32);
  const int64_t past = past_rows * p->history_max, lens = history_len ? p->rows : 0;
  const int64_t most = mask > past ? mask : past, threads = most > lens ? most : lens;
  if (threads == 0) return 0;
  ON_DEVICE(p->device, "goenv_policy_logits_keep");
  hipLaunchKernelGGL(k_keep_rules, dim3(grid_of((threads + 255) / 256, 1 << 14)), dim3(256), 0, S(stream), *p, mask_rows, past_rows, legal_bits,
                     history, history_len);
  HIPCHK(hipGetLastError());
  return 0;
}

}  // extern "C"
