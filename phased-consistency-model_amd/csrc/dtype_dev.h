// Element formats named by the caller (PCM_DT_*), independent of the 16-bit format this build's contractions use: the alignment losses and the
// gradient-norm kernels take 32-bit, bfloat16 and IEEE-half tensors in every build of the library.
#pragma once
#include "pcm_common.h"

// VEC: elements of a 16-byte access.  The vector types below have the alignment of one element only: rows of odd length and slices of flat buffers
// start anywhere, and gfx950 takes a 16-byte global access at any element address (hipcc emits global_load_dwordx4 for them).
struct DtF32 {
  typedef float raw;
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float ld(raw r) { return r; }
  static __device__ __forceinline__ raw st(float f) { return f; }
};
struct DtBf16 {
  typedef unsigned short raw;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float ld(raw r) { return __uint_as_float(((unsigned)r) << 16); }
  static __device__ __forceinline__ raw st(float f) {        // round to nearest even, NaN kept quiet
#ifdef PCM_HOST_EMU
    unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (raw)((u >> 16) | 0x40);
    return (raw)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
#else
    return __builtin_bit_cast(raw, (__bf16)f);
#endif
  }
};
struct DtF16 {
  typedef unsigned short raw;
  static constexpr int VEC = 8;
#ifdef PCM_HOST_EMU
  static __device__ __forceinline__ float ld(raw r) { return pcm_emu::half_to_float(r); }
  static __device__ __forceinline__ raw st(float f) { return pcm_emu::float_to_half(f); }
#else
  static __device__ __forceinline__ float ld(raw r) { return (float)__builtin_bit_cast(_Float16, r); }
  static __device__ __forceinline__ raw st(float f) { return __builtin_bit_cast(raw, (_Float16)f); }
#endif
};
// f(Dt{}) for the format a PCM_DT_* code names (checked by the caller)
template <typename F>
static inline void pcm_with_dtype(int dt, F&& f) {
  if (dt == PCM_DT_F32) f(DtF32{});
  else if (dt == PCM_DT_BF16) f(DtBf16{});
  else f(DtF16{});
}
static inline bool pcm_dt_ok(int dt) { return dt == PCM_DT_F32 || dt == PCM_DT_BF16 || dt == PCM_DT_F16; }
static inline size_t pcm_dt_size(int dt) { return dt == PCM_DT_F32 ? 4 : 2; }

// a group of N elements at p (N deduced from v): all of them in one access, or the first `left` and 0 for the others
// NT: a nontemporal load, for data that one launch reads once (large reads reach 6.8 TB/s with it against 6.0 without)
template <typename Dt, bool NT = false, int N>
__device__ __forceinline__ void pcm_ld_group(const typename Dt::raw* p, float (&v)[N]) {
  typedef typename Dt::raw vec __attribute__((ext_vector_type(N), aligned(sizeof(typename Dt::raw))));
  const vec r = NT ? __builtin_nontemporal_load((const vec*)p) : *(const vec*)p;
#pragma unroll
  for (int j = 0; j < N; j++) v[j] = Dt::ld(r[j]);
}
template <typename Dt, bool NT = false, int N>
__device__ __forceinline__ void pcm_ld_group(const typename Dt::raw* p, long left, float (&v)[N]) {
  if (left >= N) { pcm_ld_group<Dt, NT>(p, v); return; }
#pragma unroll
  for (int j = 0; j < N; j++) v[j] = j < left ? Dt::ld(p[j]) : 0.f;
}
template <typename Dt, bool NT = false, int N>
__device__ __forceinline__ void pcm_st_group(typename Dt::raw* p, long left, const float (&v)[N]) {
  if (left >= N) {
    typedef typename Dt::raw vec __attribute__((ext_vector_type(N), aligned(sizeof(typename Dt::raw))));
    vec r;
#pragma unroll
    for (int j = 0; j < N; j++) r[j] = Dt::st(v[j]);
    if (NT) __builtin_nontemporal_store(r, (vec*)p);
    else *(vec*)p = r;
    return;
  }
#pragma unroll
  for (int j = 0; j < N; j++)
    if (j < left) p[j] = Dt::st(v[j]);
}

// ---- work of one team (a wave or a workgroup of NT threads) on elements [i0, i1) of a row, U groups of 16 bytes per thread in flight ----
// f(idx, left): the group of VEC elements at idx, `left` of them inside the range (>= VEC: all)
template <typename Dt, int NT, int U, typename Load, typename Use>
__device__ __forceinline__ void pcm_groups(long i0, long i1, int tid, Load&& load, Use&& use) {
  constexpr long STEP = (long)NT * Dt::VEC;
  long i = i0 + (long)tid * Dt::VEC;
  for (; i + (U - 1) * STEP + Dt::VEC <= i1; i += U * STEP) {
#pragma unroll
    for (int u = 0; u < U; u++) load(u, i + u * STEP, (long)Dt::VEC);
#pragma unroll
    for (int u = 0; u < U; u++) use(u, i + u * STEP, (long)Dt::VEC);
  }
  if (i < i1) {                    // at most U groups are left, the last one perhaps partly outside
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i + u * STEP < i1) load(u, i + u * STEP, i1 - i - u * STEP);
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i + u * STEP < i1) use(u, i + u * STEP, i1 - i - u * STEP);
  }
}

// sum over a workgroup of NT threads in a fixed order (wave tree, then the wave sums in wave order), returned to every thread.  `red` holds one
// value per wave; the barriers at both ends let one buffer serve several sums.
template <typename V>
__device__ __forceinline__ V pcm_lane_sum(V v) {      // over the lanes of a wave
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <int NT, typename V>
__device__ __forceinline__ V pcm_block_sum(V v, V* red) {
  v = pcm_lane_sum(v);
  if constexpr (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  V t = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; w++) t += red[w];
  return t;
}
// the same for K values with one exchange
template <int NT, int K>
__device__ __forceinline__ void pcm_block_sums(double (&v)[K], double* red /* [NT / 64 * K] */) {
#pragma unroll
  for (int k = 0; k < K; k++) v[k] = pcm_lane_sum(v[k]);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; k++) red[(threadIdx.x >> 6) * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
      double t = red[k];
#pragma unroll
      for (int w = 1; w < NT / 64; w++) t += red[w * K + k];
      v[k] = t;
    }
  }
}
