// pcm-build-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// The global norm of the gradients held in many tensors, and their clipping:  N = sqrt(sum g^2),  g' = g * min(1, c / (N + 1e-6)).
// Tensors of any mix of formats are described by a table in device memory; the work is cut into chunks of PCM_GRAD_CHUNK elements, so that one launch
// covers all of them.  Squares and sums in fp64 (no overflow for any fp32 value), partial sums added in chunk order: bitwise the same run to run.
#include "dtype_dev.h"

template <typename Dt>
__device__ __forceinline__ double chunk_sumsq(const void* src, long i0, long i1) {
  const typename Dt::raw* p = (const typename Dt::raw*)src;
  double acc = 0.0;
  for (long i = i0 + threadIdx.x; i < i1; i += 256) { const double v = (double)Dt::ld(p[i]); acc += v * v; }
  return acc;
}
__global__ __launch_bounds__(256) void grad_sumsq_kernel(const pcm_grad_desc* descs, const pcm_grad_chunk* chunks, int nchunks, double* part) {
  __shared__ double red[4];
  double acc = 0.0;
  for (int c = blockIdx.x; c < nchunks; c += gridDim.x) {
    const pcm_grad_chunk ch = chunks[c];
    const pcm_grad_desc d = descs[ch.tensor];
    const long i1 = ch.start + PCM_GRAD_CHUNK < d.n ? ch.start + PCM_GRAD_CHUNK : d.n;
    acc += d.src_dtype == PCM_DT_F32 ? chunk_sumsq<DtF32>(d.src, ch.start, i1)
                                     : (d.src_dtype == PCM_DT_BF16 ? chunk_sumsq<DtBf16>(d.src, ch.start, i1) : chunk_sumsq<DtF16>(d.src, ch.start, i1));
  }
  acc = pcm_block_sum<256>(acc, red);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}
__global__ __launch_bounds__(256) void grad_norm_finish_kernel(const double* part, int n, float* norm, double* sumsq) {
  __shared__ double red[4];
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) acc += part[i];
  acc = pcm_block_sum<256>(acc, red);
  if (threadIdx.x == 0) { sumsq[0] = acc; norm[0] = (float)sqrt(acc); }
}
template <typename S, typename D>
__device__ __forceinline__ void chunk_scale(const void* src, void* dst, float f, long i0, long i1) {
  const typename S::raw* p = (const typename S::raw*)src;
  typename D::raw* q = (typename D::raw*)dst;
  for (long i = i0 + threadIdx.x; i < i1; i += 256) q[i] = D::st(S::ld(p[i]) * f);
}
template <typename S>
__device__ __forceinline__ void chunk_scale_to(const pcm_grad_desc& d, float f, long i0, long i1) {
  if (d.dst_dtype == PCM_DT_F32) chunk_scale<S, DtF32>(d.src, d.dst, f, i0, i1);
  else if (d.dst_dtype == PCM_DT_BF16) chunk_scale<S, DtBf16>(d.src, d.dst, f, i0, i1);
  else chunk_scale<S, DtF16>(d.src, d.dst, f, i0, i1);
}
__global__ __launch_bounds__(256) void grad_scale_kernel(const pcm_grad_desc* descs, const pcm_grad_chunk* chunks, int nchunks, const double* sumsq, double max_norm) {
  const double c = max_norm / (sqrt(sumsq[0]) + 1e-6);
  const float f = c < 1.0 ? (float)c : (c == c ? 1.0f : (float)c);      // a norm that is not a number reaches the gradients, as the formula has it
  for (int k = blockIdx.x; k < nchunks; k += gridDim.x) {
    const pcm_grad_chunk ch = chunks[k];
    const pcm_grad_desc d = descs[ch.tensor];
    if (f == 1.0f && d.src == d.dst) continue;                          // in place and nothing to clip
    const long i1 = ch.start + PCM_GRAD_CHUNK < d.n ? ch.start + PCM_GRAD_CHUNK : d.n;
    if (d.src_dtype == PCM_DT_F32) chunk_scale_to<DtF32>(d, f, ch.start, i1);
    else if (d.src_dtype == PCM_DT_BF16) chunk_scale_to<DtBf16>(d, f, ch.start, i1);
    else chunk_scale_to<DtF16>(d, f, ch.start, i1);
  }
}
static int grad_blocks(int nchunks) { const int cap = PCM_GRID_CAP(2048); return nchunks < cap ? nchunks : cap; }
extern "C" size_t pcm_grad_norm_workspace_bytes(int nchunks) { return nchunks > 0 ? (size_t)grad_blocks(nchunks) * sizeof(double) : 0; }
static int grad_norm(const char* who, const pcm_grad_desc* descs, const pcm_grad_chunk* chunks, int nchunks, float* norm, double* sumsq, void* workspace,
                     size_t workspace_bytes, void* stream) {
  PCM_CHECK(descs && chunks && nchunks > 0 && norm && sumsq, PCM_EINVAL, "%s: null/empty", who);
  PCM_CHECK(workspace && ((uintptr_t)workspace % 8) == 0 && workspace_bytes >= pcm_grad_norm_workspace_bytes(nchunks), PCM_EINVAL,
            "%s: workspace too small or not 8-byte aligned", who);
  const int nb = grad_blocks(nchunks);
  PCM_LAUNCH(grad_sumsq_kernel, dim3(nb), dim3(256), 0, stream, descs, chunks, nchunks, (double*)workspace);
  PCM_LAUNCH(grad_norm_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)workspace, nb, norm, sumsq);
  return pcm_post_launch(who);
}
extern "C" int pcm_grad_norm(const pcm_grad_desc* descs, const pcm_grad_chunk* chunks, int nchunks, float* norm, double* sumsq, void* workspace,
                             size_t workspace_bytes, void* stream) {
  return grad_norm("pcm_grad_norm", descs, chunks, nchunks, norm, sumsq, workspace, workspace_bytes, stream);
}
extern "C" int pcm_grad_clip(const pcm_grad_desc* descs, const pcm_grad_chunk* chunks, int nchunks, double max_norm, float* norm, double* sumsq, void* workspace,
                             size_t workspace_bytes, void* stream) {
  PCM_CHECK(max_norm > 0.0, PCM_EINVAL, "pcm_grad_clip: max_norm must be positive");
  const int rc = grad_norm("pcm_grad_clip", descs, chunks, nchunks, norm, sumsq, workspace, workspace_bytes, stream);
  if (rc != PCM_OK) return rc;
  PCM_LAUNCH(grad_scale_kernel, dim3(grad_blocks(nchunks)), dim3(256), 0, stream, descs, chunks, nchunks, (const double*)sumsq, max_norm);
  return pcm_post_launch("pcm_grad_clip");
}
