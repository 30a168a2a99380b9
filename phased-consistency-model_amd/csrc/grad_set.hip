// pcm-build-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// The global norm of the gradients held in many tensors, and their clipping:  N = sqrt(sum g^2),  g' = g * min(1, c / (N + 1e-6)).
// A table in device memory cuts tensors of any mix of formats into pieces of at most PCM_GRAD_CHUNK elements; one launch covers all of them, a
// piece to a workgroup at a time.  Squares and sums in fp64 (no overflow for any fp32 value), partial sums added in piece order: bitwise the same run
// to run.  Bound by memory: 4 bytes in for one multiply-add, then 4 in and 4 out for one product.
#include "dtype_dev.h"

template <typename Dt, int NT>
__device__ __forceinline__ double piece_sumsq(const void* src, int n, int tid) {
  const typename Dt::raw* p = (const typename Dt::raw*)src;
  float v[4][Dt::VEC];
  double acc = 0.0;
  pcm_groups<Dt, NT, 4>(0, n, tid, [&](int u, long i, long left) { pcm_ld_group<Dt, true>(p + i, left, v[u]); },
    [&](int u, long i, long left) {
#pragma unroll
      for (int j = 0; j < Dt::VEC; j++) acc += (double)v[u][j] * (double)v[u][j];
    });
  return acc;
}
template <typename S, typename D, int NT>
__device__ __forceinline__ void piece_scale(const void* src, void* dst, float f, int n, int tid) {
  constexpr int N = S::VEC < D::VEC ? S::VEC : D::VEC;      // elements of a thread's group: 16 bytes of the wider format, at most 8 of the other
  typedef typename std::conditional<S::VEC == N, S, D>::type W;
  const typename S::raw* p = (const typename S::raw*)src;
  typename D::raw* q = (typename D::raw*)dst;
  float v[4][N];
  pcm_groups<W, NT, 4>(0, n, tid, [&](int u, long i, long left) { pcm_ld_group<S, true>(p + i, left, v[u]); },
    [&](int u, long i, long left) {
#pragma unroll
      for (int j = 0; j < N; j++) v[u][j] *= f;
      pcm_st_group<D, true>(q + i, left, v[u]);
    });
}
template <int NT>
__device__ __forceinline__ double chunk_sumsq(const pcm_grad_chunk& c, int tid) {
  if (c.src_dtype == PCM_DT_F32) return piece_sumsq<DtF32, NT>(c.src, c.n, tid);
  if (c.src_dtype == PCM_DT_BF16) return piece_sumsq<DtBf16, NT>(c.src, c.n, tid);
  return piece_sumsq<DtF16, NT>(c.src, c.n, tid);
}
template <typename S, int NT>
__device__ __forceinline__ void chunk_scale_from(const pcm_grad_chunk& c, float f, int tid) {
  if (c.dst_dtype == PCM_DT_F32) piece_scale<S, DtF32, NT>(c.src, c.dst, f, c.n, tid);
  else if (c.dst_dtype == PCM_DT_BF16) piece_scale<S, DtBf16, NT>(c.src, c.dst, f, c.n, tid);
  else piece_scale<S, DtF16, NT>(c.src, c.dst, f, c.n, tid);
}
template <int NT>
__device__ __forceinline__ void chunk_scale(const pcm_grad_chunk& c, float f, int tid) {
  if (f == 1.0f && c.src == c.dst) return;                              // in place and nothing to clip
  if (c.src_dtype == PCM_DT_F32) chunk_scale_from<DtF32, NT>(c, f, tid);
  else if (c.src_dtype == PCM_DT_BF16) chunk_scale_from<DtBf16, NT>(c, f, tid);
  else chunk_scale_from<DtF16, NT>(c, f, tid);
}
__device__ __forceinline__ float clip_factor(double sumsq, double max_norm) {
  const double c = max_norm / (sqrt(sumsq) + 1e-6);
  return c < 1.0 ? (float)c : (c == c ? 1.0f : (float)c);               // a norm that is not a number reaches the gradients, as the formula has it
}
__global__ __launch_bounds__(256) void grad_sumsq_kernel(const pcm_grad_chunk* chunks, int nchunks, double* part) {
  __shared__ double red[4];
  double acc = 0.0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) acc += chunk_sumsq<256>(chunks[c], threadIdx.x);
  acc = pcm_block_sum<256>(acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}
__device__ __forceinline__ double grad_total(const double* part, int n, double* red) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) acc += part[i];
  return pcm_block_sum<256>(acc, red);
}
__global__ __launch_bounds__(256) void grad_norm_finish_kernel(const double* part, int n, float* norm, double* sumsq) {
  __shared__ double red[4];
  const double t = grad_total(part, n, red);
  if (threadIdx.x == 0) { sumsq[0] = t; norm[0] = (float)sqrt(t); }
}
// Every workgroup adds up the partial sums again (8 KB out of L2) instead of waiting for a launch that does it once.  At 285 MB in and out: a piece to a
// workgroup 155 us against 162 with 4096 workgroups (the sum: 1024 are as fast as 4096, and fewer partial sums), nontemporal stores 147.
__global__ __launch_bounds__(256) void grad_scale_kernel(const pcm_grad_chunk* chunks, int nchunks, const double* part, int nparts, double max_norm, float* norm,
                                                         double* sumsq) {
  __shared__ double red[4];
  const double t = grad_total(part, nparts, red);
  if (blockIdx.x == 0 && threadIdx.x == 0) { sumsq[0] = t; norm[0] = (float)sqrt(t); }
  const float f = clip_factor(t, max_norm);
  for (int c = (int)blockIdx.x; c < nchunks; c += gridDim.x) chunk_scale<256>(chunks[c], f, threadIdx.x);
}
// few elements in few pieces: one workgroup does it all in one launch, its 16 waves taking pieces in turn (max_norm <= 0: the norm alone).  The pieces'
// records are read once, into LDS, so that a piece waits for its data only.
#define GRAD_SMALL_CHUNKS 64
__global__ __launch_bounds__(1024) void grad_small_kernel(const pcm_grad_chunk* chunks, int nchunks, double max_norm, float* norm, double* sumsq) {
  __shared__ pcm_grad_chunk tab[GRAD_SMALL_CHUNKS];
  __shared__ double red[16];
  if ((int)threadIdx.x < nchunks) tab[threadIdx.x] = chunks[threadIdx.x];
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  double acc = 0.0;
  for (int c = wave; c < nchunks; c += 16) acc += chunk_sumsq<64>(tab[c], lane);
  acc = pcm_block_sum<1024>(acc, red);
  if (threadIdx.x == 0) { sumsq[0] = acc; norm[0] = (float)sqrt(acc); }
  if (max_norm > 0.0) {
    const float f = clip_factor(acc, max_norm);
    for (int c = wave; c < nchunks; c += 16) chunk_scale<64>(tab[c], f, lane);
  }
}
// One workgroup against two launches: the second launch costs about 4 us, a round of 16 pieces of 1024 elements about 1 us each way.
#define GRAD_SMALL_ELEMENTS 32768
static bool grad_small(int nchunks, long total) { return total <= GRAD_SMALL_ELEMENTS && nchunks <= GRAD_SMALL_CHUNKS; }
static int grad_blocks(int nchunks, int cap) { return nchunks < cap ? nchunks : cap; }
#define GRAD_PARTS PCM_GRID_CAP(1024)
extern "C" size_t pcm_grad_norm_workspace_bytes(int nchunks, long total) {
  return nchunks > 0 && !grad_small(nchunks, total) ? (size_t)grad_blocks(nchunks, GRAD_PARTS) * sizeof(double) : 0;
}
static int grad_run(const char* who, const pcm_grad_chunk* chunks, int nchunks, long total, double max_norm, float* norm, double* sumsq, void* workspace,
                    size_t workspace_bytes, void* stream) {
  PCM_CHECK(chunks && nchunks > 0 && total > 0 && norm && sumsq, PCM_EINVAL, "%s: null/empty", who);
  const size_t need = pcm_grad_norm_workspace_bytes(nchunks, total);
  PCM_CHECK(need == 0 || (workspace && ((uintptr_t)workspace % 8) == 0 && workspace_bytes >= need), PCM_EINVAL,
            "%s: workspace too small or not 8-byte aligned", who);
  if (need == 0) {
    PCM_LAUNCH(grad_small_kernel, dim3(1), dim3(1024), 0, stream, chunks, nchunks, max_norm, norm, sumsq);
    return pcm_post_launch(who);
  }
  const int nb = grad_blocks(nchunks, GRAD_PARTS);
  PCM_LAUNCH(grad_sumsq_kernel, dim3(nb), dim3(256), 0, stream, chunks, nchunks, (double*)workspace);
  if (max_norm > 0.0)
    PCM_LAUNCH(grad_scale_kernel, dim3(grad_blocks(nchunks, PCM_GRID_CAP(16384))), dim3(256), 0, stream, chunks, nchunks, (const double*)workspace, nb, max_norm, norm, sumsq);
  else
    PCM_LAUNCH(grad_norm_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)workspace, nb, norm, sumsq);
  return pcm_post_launch(who);
}
extern "C" int pcm_grad_norm(const pcm_grad_chunk* chunks, int nchunks, long total, float* norm, double* sumsq, void* workspace, size_t workspace_bytes,
                             void* stream) {
  return grad_run("pcm_grad_norm", chunks, nchunks, total, 0.0, norm, sumsq, workspace, workspace_bytes, stream);
}
extern "C" int pcm_grad_clip(const pcm_grad_chunk* chunks, int nchunks, long total, double max_norm, float* norm, double* sumsq, void* workspace,
                             size_t workspace_bytes, void* stream) {
  PCM_CHECK(max_norm > 0.0, PCM_EINVAL, "pcm_grad_clip: max_norm must be positive");
  return grad_run("pcm_grad_clip", chunks, nchunks, total, max_norm, norm, sumsq, workspace, workspace_bytes, stream);
}
