// pcm-build-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Alignment of a distilled student: preference losses over paired log ratios, the clipped policy loss with its KL term, and the log-probability
// of a noisy sampler transition, each with its gradient.  Everything here is bound by memory: a few operations per element read.
//
// Elements are formed in fp32; every sum over elements, rows or tokens is carried in fp64 and in an order fixed by the launch (partial sums in the
// caller's workspace, added up by index), so results are bitwise the same run to run.
#include "dtype_dev.h"

#define AL_LOOP(i, n) for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < (n); i += (long)gridDim.x * blockDim.x)
static inline int al_blocks(long n) { long b = (n + 255) / 256; return (int)(b > PCM_GRID_CAP(2048) ? PCM_GRID_CAP(2048) : (b < 1 ? 1 : b)); }

// ---- log-probability of x ~ N(mean, std^2) per row:  -1/2 sum ((x - mean) / std)^2 - n log std - n/2 log 2 pi   (/ n) ----
#define LOG_2PI 1.8378770664093454836
template <typename Dt>
__global__ __launch_bounds__(256) void transition_fwd_kernel(const typename Dt::raw* x, const typename Dt::raw* mean, const float* std, float* logp,
                                                             long n, int mean_reduce) {
  __shared__ double red[4];
  const long row = blockIdx.x;
  x += row * n; mean += row * n;
  double acc = 0.0;
  for (long i = threadIdx.x; i < n; i += 256) { const float d = Dt::ld(x[i]) - Dt::ld(mean[i]); acc += (double)(d * d); }
  acc = pcm_block_sum<256>(acc, red);
  if (threadIdx.x == 0) {
    const double s = (double)std[row];
    const double per = -0.5 * acc / (s * s * (double)n) - log(s) - 0.5 * LOG_2PI;
    logp[row] = (float)(mean_reduce ? per : per * (double)n);
  }
}
template <typename Dt>
__global__ __launch_bounds__(256) void transition_bwd_kernel(const typename Dt::raw* x, const typename Dt::raw* mean, const float* std,
                                                             const float* dlogp, typename Dt::raw* dmean, long rows, long n, int mean_reduce) {
  AL_LOOP(i, rows * n) {
    const long row = i / n;
    const double s = (double)std[row];
    const float f = (float)((double)dlogp[row] / (s * s * (mean_reduce ? (double)n : 1.0)));
    dmean[i] = Dt::st((Dt::ld(x[i]) - Dt::ld(mean[i])) * f);
  }
}

// ---- preference losses.  rows [0, P) are the preferred side, [P, 2P) the rejected side; rho = log ratio of a row ----
struct PairLoss { double beta, eps; int kind; };
// loss of one pair and its derivative by the preferred row's rho (the rejected row's is its negative)
__device__ __forceinline__ void pair_loss(const PairLoss p, double h, double* loss, double* slope) {
  if (p.kind == PCM_PAIR_SIGMOID) {
    const double s = p.beta * h, e = exp(-fabs(s)), soft = log1p(e);             // -log sig(s) = soft + max(-s, 0)
    *loss = (1.0 - p.eps) * (soft + fmax(-s, 0.0)) + p.eps * (soft + fmax(s, 0.0));
    *slope = p.beta * ((s >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e)) - (1.0 - p.eps));
    if (!(s == s)) *loss = s;                                                     // fmax drops a NaN
  } else if (p.kind == PCM_PAIR_HINGE) {
    const double s = p.beta * h;
    *loss = s < 1.0 ? 1.0 - s : (s == s ? 0.0 : s);
    *slope = s < 1.0 ? -p.beta : (s == s ? 0.0 : s);
  } else {
    const double gap = h - 0.5 / p.beta;
    *loss = gap * gap;
    *slope = 2.0 * gap;
  }
}
__global__ __launch_bounds__(256) void pair_finish_kernel(const double* rho, PairLoss pl, long pairs, float* loss, float* log_ratio) {
  __shared__ double red[4];
  double acc = 0.0;
  for (long p = threadIdx.x; p < pairs; p += 256) {
    double l, s;
    pair_loss(pl, rho[p] - rho[pairs + p], &l, &s);
    acc += l;
    log_ratio[p] = (float)rho[p];
    log_ratio[pairs + p] = (float)rho[pairs + p];
  }
  acc = pcm_block_sum<256>(acc, red);
  if (threadIdx.x == 0) loss[0] = (float)(acc / (double)pairs);
}
// rho of one row of denoising errors: -w k sum ((t - p)^2 - (t - r)^2)
template <typename Dt>
__global__ __launch_bounds__(256) void denoise_rho_kernel(const typename Dt::raw* pred, const typename Dt::raw* ref, const typename Dt::raw* target,
                                                          const float* weight, double k, double* rho, long n) {
  __shared__ double red[4];
  const long row = blockIdx.x;
  double acc = 0.0;
  for (long i = row * n + threadIdx.x; i < (row + 1) * n; i += 256) {
    const float t = Dt::ld(target[i]), a = t - Dt::ld(pred[i]), b = t - Dt::ld(ref[i]);
    acc += (double)(a * a - b * b);
  }
  acc = pcm_block_sum<256>(acc, red);
  if (threadIdx.x == 0) rho[row] = -acc * k * (weight ? (double)weight[row] : 1.0);
}
template <typename Dt>
__global__ __launch_bounds__(256) void denoise_grad_kernel(const typename Dt::raw* pred, const typename Dt::raw* target, const float* weight, double k,
                                                           const double* rho, PairLoss pl, double gscale, typename Dt::raw* dpred, long pairs, long n) {
  const long row = blockIdx.x, p = row < pairs ? row : row - pairs;
  double l, s;
  pair_loss(pl, rho[p] - rho[pairs + p], &l, &s);
  const float f = (float)((row < pairs ? 2.0 : -2.0) * s * k * gscale / (double)pairs * (weight ? (double)weight[row] : 1.0));
  for (long i = row * n + threadIdx.x; i < (row + 1) * n; i += 256) dpred[i] = Dt::st((Dt::ld(target[i]) - Dt::ld(pred[i])) * f);
}

// places that count: mask[row][col] != 0 (or no mask) and col < lengths[row] (or no lengths)
struct Places {
  const unsigned char* mask; long ld_mask;
  const void* lengths; int i64;
  long cols;
  __device__ __forceinline__ long len(long row) const {
    if (!lengths) return cols;
    const long v = i64 ? (long)((const int64_t*)lengths)[row] : (long)((const int32_t*)lengths)[row];
    return v < 0 ? 0 : (v > cols ? cols : v);
  }
};
template <typename Dt>
__global__ __launch_bounds__(256) void preference_rho_kernel(const typename Dt::raw* logp, long ld_logp, const typename Dt::raw* ref, long ld_ref, Places pc,
                                                             int mean_reduce, double* rho, double* share) {
  __shared__ double red[4];
  __shared__ long redl[4];
  const long row = blockIdx.x, len = pc.len(row);
  double acc = 0.0;
  long cnt = 0;
  for (long c = threadIdx.x; c < len; c += 256) {
    if (pc.mask && !pc.mask[row * pc.ld_mask + c]) continue;
    acc += (double)(Dt::ld(logp[row * ld_logp + c]) - Dt::ld(ref[row * ld_ref + c]));
    cnt++;
  }
  acc = pcm_block_sum<256>(acc, red);
  cnt = pcm_block_sum<256>(cnt, redl);
  if (threadIdx.x == 0) {
    const double sh = mean_reduce ? 1.0 / (double)(cnt > 0 ? cnt : 1) : 1.0;
    rho[row] = acc * sh;
    share[row] = sh;
  }
}
template <typename Dt>
__global__ __launch_bounds__(256) void preference_grad_kernel(Places pc, const double* rho, const double* share, PairLoss pl, double gscale,
                                                              typename Dt::raw* dlogp, long ld_d, long pairs) {
  const long row = blockIdx.x, len = pc.len(row), p = row < pairs ? row : row - pairs;
  double l, s;
  pair_loss(pl, rho[p] - rho[pairs + p], &l, &s);
  const float f = (float)((row < pairs ? 1.0 : -1.0) * s * share[row] * gscale / (double)pairs);
  for (long c = threadIdx.x; c < pc.cols; c += 256)
    dlogp[row * ld_d + c] = Dt::st(c < len && (!pc.mask || pc.mask[row * pc.ld_mask + c]) ? f : 0.f);
}

// ---- clipped policy loss with a KL term ----
// exp(d) - d - 1 to full relative accuracy: below 1/2 the power series d^2/2 (1 + d/3 (1 + d/4 (...))) -- the difference itself would leave
// nothing of a small d -- with terms to d^10 (the first one left out is 2^-10 * 2 / 12! of the sum); above, the difference.
__device__ __forceinline__ float kl_term(float d) {
  if (fabsf(d) < 0.5f) {
    float s = 1.0f + d * (1.0f / 10.0f);
    s = 1.0f + d * (1.0f / 9.0f) * s; s = 1.0f + d * (1.0f / 8.0f) * s; s = 1.0f + d * (1.0f / 7.0f) * s; s = 1.0f + d * (1.0f / 6.0f) * s;
    s = 1.0f + d * (1.0f / 5.0f) * s; s = 1.0f + d * (1.0f / 4.0f) * s; s = 1.0f + d * (1.0f / 3.0f) * s;
    return 0.5f * d * d * s;
  }
  return (expf(d) - 1.0f) - d;
}
struct PolicyConst { double log_over, log_under; float over, under, kl; };     // log(1 + hi), log(1 - lo), 1 + hi, 1 - lo, KL coefficient
// one place: the clipped objective, the KL estimate, the derivative of objective + kl * KL by logp.  The border of the clipping is decided in fp64:
// the difference of two fp32 numbers is exact there.
__device__ __forceinline__ void policy_place(const PolicyConst c, float lp, float old, bool has_ref, float ref, float a, float* obj, float* kl,
                                             float* slope, bool* clipped) {
  const double x = (double)lp - (double)old;
  const bool over = a > 0.f && x > c.log_over, under = a < 0.f && x < c.log_under;
  // (an advantage of zero adds nothing, also where exp leaves fp32; a NaN stays one)
  const float r = a == 0.f && x == x ? 0.f : expf((float)x);
  *clipped = over || under;
  *obj = -a * (over ? c.over : (under ? c.under : r));
  *slope = *clipped ? 0.f : -a * r;
  *kl = 0.f;
  if (has_ref) {
    const float d = ref - lp, k = kl_term(d);
    *kl = k;
    *slope -= c.kl * (k + d);        // exp(d) - 1 = k + d
  }
}
// counts per row
__global__ __launch_bounds__(256) void policy_count_kernel(Places pc, double* count) {
  __shared__ long red[4];
  const long row = blockIdx.x, len = pc.len(row);
  long cnt = 0;
  for (long c = threadIdx.x; c < len; c += 256) cnt += (!pc.mask || pc.mask[row * pc.ld_mask + c]) ? 1 : 0;
  cnt = pcm_block_sum<256>(cnt, red);
  if (threadIdx.x == 0) count[row] = (double)cnt;
}
// total[0] = sum of the counts
__global__ __launch_bounds__(256) void policy_total_kernel(const double* count, long rows, double* total) {
  __shared__ double red[4];
  double acc = 0.0;
  for (long r = threadIdx.x; r < rows; r += 256) acc += count[r];
  acc = pcm_block_sum<256>(acc, red);
  if (threadIdx.x == 0) total[0] = acc;
}
template <typename Dt>
__global__ __launch_bounds__(256) void policy_main_kernel(const typename Dt::raw* logp, long ld_logp, const typename Dt::raw* old, long ld_old,
                                                          const typename Dt::raw* ref, long ld_ref, const float* adv, long ld_adv, int adv_row, Places pc,
                                                          PolicyConst con, int reduce, float gscale, const double* count, const double* total,
                                                          typename Dt::raw* dlogp, long ld_d, long rows, double* part) {
  __shared__ double red[4];
  const double inv_total = 1.0 / fmax(total[0], 1.0);
  double so = 0.0, sk = 0.0, sc = 0.0;
  AL_LOOP(i, rows * pc.cols) {
    const long row = i / pc.cols, c = i - row * pc.cols;
    float g = 0.f;
    if (c < pc.len(row) && (!pc.mask || pc.mask[row * pc.ld_mask + c])) {
      const double w = reduce == PCM_POLICY_TOKEN ? inv_total : (reduce == PCM_POLICY_ROW ? 1.0 / (count[row] * (double)rows) : 1.0);
      const float lp = Dt::ld(logp[row * ld_logp + c]);
      float obj, kl, slope;
      bool clipped;
      policy_place(con, lp, old ? Dt::ld(old[row * ld_old + c]) : lp, ref != nullptr, ref ? Dt::ld(ref[row * ld_ref + c]) : 0.f,
                   adv[adv_row ? row : row * ld_adv + c], &obj, &kl, &slope, &clipped);
      so += w * (double)obj; sk += w * (double)kl; sc += clipped ? 1.0 : 0.0;
      g = slope * (float)(w * (double)gscale);
    }
    if (dlogp) dlogp[row * ld_d + c] = Dt::st(g);
  }
  so = pcm_block_sum<256>(so, red); sk = pcm_block_sum<256>(sk, red); sc = pcm_block_sum<256>(sc, red);
  if (threadIdx.x == 0) { part[3 * blockIdx.x] = so; part[3 * blockIdx.x + 1] = sk; part[3 * blockIdx.x + 2] = sc; }
}
__global__ __launch_bounds__(256) void policy_finish_kernel(const double* part, int nparts, const double* total, double kl, float* loss, float* stats) {
  __shared__ double red[4];
  double so = 0.0, sk = 0.0, sc = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) { so += part[3 * i]; sk += part[3 * i + 1]; sc += part[3 * i + 2]; }
  so = pcm_block_sum<256>(so, red); sk = pcm_block_sum<256>(sk, red); sc = pcm_block_sum<256>(sc, red);
  if (threadIdx.x == 0) {
    loss[0] = (float)(so + kl * sk);
    stats[0] = (float)so; stats[1] = (float)sk; stats[2] = (float)(sc / fmax(total[0], 1.0)); stats[3] = (float)total[0];
  }
}

// ---- entry points ----
#define AL_MAX_ROWS 2147483647L
extern "C" size_t pcm_transition_logprob_workspace_bytes(long rows, long n) { return rows > 0 && n > 0 ? 8 : 0; }
extern "C" int pcm_transition_logprob(const void* x, const void* mean, const float* std, int dtype, int mean_reduce, float* logp, long rows, long n,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  PCM_CHECK(x && mean && std && logp && pcm_dt_ok(dtype) && rows > 0 && rows <= AL_MAX_ROWS && n > 0, PCM_EINVAL, "pcm_transition_logprob: null/empty or unknown format");
  PCM_CHECK(workspace && ((uintptr_t)workspace % 8) == 0 && workspace_bytes >= pcm_transition_logprob_workspace_bytes(rows, n), PCM_EINVAL,
            "pcm_transition_logprob: workspace too small or not 8-byte aligned");
  pcm_with_dtype(dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    PCM_LAUNCH(transition_fwd_kernel<Dt>, dim3((unsigned)rows), dim3(256), 0, stream, (cp)x, (cp)mean, std, logp, n, mean_reduce);
  });
  return pcm_post_launch("pcm_transition_logprob");
}
extern "C" int pcm_transition_logprob_bwd(const void* x, const void* mean, const float* std, const float* dlogp, int dtype, int mean_reduce, void* dmean,
                                          long rows, long n, void* stream) {
  PCM_CHECK(x && mean && std && dlogp && dmean && pcm_dt_ok(dtype) && rows > 0 && rows <= AL_MAX_ROWS && n > 0, PCM_EINVAL,
            "pcm_transition_logprob_bwd: null/empty or unknown format");
  pcm_with_dtype(dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    PCM_LAUNCH(transition_bwd_kernel<Dt>, dim3(al_blocks(rows * n)), dim3(256), 0, stream, (cp)x, (cp)mean, std, dlogp, (typename Dt::raw*)dmean, rows, n, mean_reduce);
  });
  return pcm_post_launch("pcm_transition_logprob_bwd");
}

static int pair_args_ok(const char* who, int dtype, long pairs, double beta, int kind, double eps) {
  PCM_CHECK(pcm_dt_ok(dtype), PCM_EINVAL, "%s: unknown element format %d", who, dtype);
  PCM_CHECK(pairs > 0 && pairs <= AL_MAX_ROWS / 2, PCM_EINVAL, "%s: number of pairs %ld", who, pairs);
  PCM_CHECK(beta > 0.0 && beta < 1e30, PCM_EINVAL, "%s: beta must be positive and finite", who);
  PCM_CHECK(kind == PCM_PAIR_SIGMOID || kind == PCM_PAIR_HINGE || kind == PCM_PAIR_SQUARE, PCM_EINVAL, "%s: unknown kind %d", who, kind);
  PCM_CHECK(eps >= 0.0 && eps < 0.5 && (eps == 0.0 || kind == PCM_PAIR_SIGMOID), PCM_EINVAL, "%s: label smoothing must be in [0, 0.5) and needs the sigmoid kind", who);
  return PCM_OK;
}
extern "C" size_t pcm_denoise_preference_loss_workspace_bytes(long pairs, long n) { return pairs > 0 && n > 0 ? 2 * (size_t)pairs * sizeof(double) : 0; }
extern "C" int pcm_denoise_preference_loss(const pcm_denoise_preference_args* a, void* stream) {
  PCM_CHECK(a && a->pred && a->ref && a->target && a->loss && a->log_ratio && a->n > 0, PCM_EINVAL, "pcm_denoise_preference_loss: null/empty");
  const int rc = pair_args_ok("pcm_denoise_preference_loss", a->dtype, a->pairs, a->beta, a->kind, a->label_smoothing);
  if (rc != PCM_OK) return rc;
  PCM_CHECK(a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= pcm_denoise_preference_loss_workspace_bytes(a->pairs, a->n), PCM_EINVAL,
            "pcm_denoise_preference_loss: workspace too small or not 8-byte aligned");
  const PairLoss pl = {a->beta, a->label_smoothing, a->kind};
  const double k = a->mean_reduce ? 1.0 / (double)a->n : 1.0;
  double* rho = (double*)a->workspace;
  pcm_with_dtype(a->dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    PCM_LAUNCH(denoise_rho_kernel<Dt>, dim3((unsigned)(2 * a->pairs)), dim3(256), 0, stream, (cp)a->pred, (cp)a->ref, (cp)a->target, a->weight, k, rho, a->n);
    PCM_LAUNCH(pair_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)rho, pl, a->pairs, a->loss, a->log_ratio);
    if (a->dpred)
      PCM_LAUNCH(denoise_grad_kernel<Dt>, dim3((unsigned)(2 * a->pairs)), dim3(256), 0, stream, (cp)a->pred, (cp)a->target, a->weight, k, (const double*)rho, pl,
                 a->grad_scale, (typename Dt::raw*)a->dpred, a->pairs, a->n);
  });
  return pcm_post_launch("pcm_denoise_preference_loss");
}
extern "C" size_t pcm_preference_loss_workspace_bytes(long pairs, long cols) { return pairs > 0 && cols > 0 ? 4 * (size_t)pairs * sizeof(double) : 0; }
extern "C" int pcm_preference_loss(const pcm_preference_args* a, void* stream) {
  PCM_CHECK(a && a->logp && a->ref_logp && a->loss && a->log_ratio && a->cols > 0, PCM_EINVAL, "pcm_preference_loss: null/empty");
  const int rc = pair_args_ok("pcm_preference_loss", a->dtype, a->pairs, a->beta, a->kind, a->label_smoothing);
  if (rc != PCM_OK) return rc;
  PCM_CHECK(a->ld_logp >= a->cols && a->ld_ref >= a->cols && (!a->mask || a->ld_mask >= a->cols) && (!a->dlogp || a->ld_dlogp >= a->cols), PCM_EINVAL,
            "pcm_preference_loss: row stride below the row length");
  PCM_CHECK(a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= pcm_preference_loss_workspace_bytes(a->pairs, a->cols), PCM_EINVAL,
            "pcm_preference_loss: workspace too small or not 8-byte aligned");
  const PairLoss pl = {a->beta, a->label_smoothing, a->kind};
  const Places pc = {a->mask, a->ld_mask, a->lengths, a->lengths_i64, a->cols};
  double* rho = (double*)a->workspace;
  double* share = rho + 2 * a->pairs;
  pcm_with_dtype(a->dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    PCM_LAUNCH(preference_rho_kernel<Dt>, dim3((unsigned)(2 * a->pairs)), dim3(256), 0, stream, (cp)a->logp, a->ld_logp, (cp)a->ref_logp, a->ld_ref, pc,
               a->mean_reduce, rho, share);
    PCM_LAUNCH(pair_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)rho, pl, a->pairs, a->loss, a->log_ratio);
    if (a->dlogp)
      PCM_LAUNCH(preference_grad_kernel<Dt>, dim3((unsigned)(2 * a->pairs)), dim3(256), 0, stream, pc, (const double*)rho, (const double*)share, pl,
                 a->grad_scale, (typename Dt::raw*)a->dlogp, a->ld_dlogp, a->pairs);
  });
  return pcm_post_launch("pcm_preference_loss");
}
extern "C" size_t pcm_policy_loss_workspace_bytes(long rows, long cols) {
  return rows > 0 && cols > 0 ? ((size_t)rows + 1 + 3 * (size_t)al_blocks(rows * cols)) * sizeof(double) : 0;
}
extern "C" int pcm_policy_loss(const pcm_policy_args* a, void* stream) {
  PCM_CHECK(a && a->logp && a->advantages && a->loss && a->stats && a->rows > 0 && a->rows <= AL_MAX_ROWS && a->cols > 0, PCM_EINVAL, "pcm_policy_loss: null/empty");
  PCM_CHECK(pcm_dt_ok(a->dtype), PCM_EINVAL, "pcm_policy_loss: unknown element format %d", a->dtype);
  PCM_CHECK(a->reduce == PCM_POLICY_TOKEN || a->reduce == PCM_POLICY_ROW || a->reduce == PCM_POLICY_SUM, PCM_EINVAL, "pcm_policy_loss: unknown reduce %d", a->reduce);
  PCM_CHECK(a->clip_low >= 0.0 && a->clip_low < 1.0 && a->clip_high >= 0.0 && a->clip_high < 1e30, PCM_EINVAL, "pcm_policy_loss: clip_low must be in [0, 1), clip_high >= 0");
  PCM_CHECK(a->kl_coef == 0.0 || a->ref_logp, PCM_EINVAL, "pcm_policy_loss: a KL term needs the reference log-probabilities");
  PCM_CHECK(a->ld_logp >= a->cols && (!a->old_logp || a->ld_old >= a->cols) && (!a->ref_logp || a->ld_ref >= a->cols) && (a->adv_per_row || a->ld_adv >= a->cols) &&
                (!a->mask || a->ld_mask >= a->cols) && (!a->dlogp || a->ld_dlogp >= a->cols), PCM_EINVAL, "pcm_policy_loss: row stride below the row length");
  PCM_CHECK(a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= pcm_policy_loss_workspace_bytes(a->rows, a->cols), PCM_EINVAL,
            "pcm_policy_loss: workspace too small or not 8-byte aligned");
  const Places pc = {a->mask, a->ld_mask, a->lengths, a->lengths_i64, a->cols};
  const PolicyConst con = {log1p(a->clip_high), log1p(-a->clip_low), (float)(1.0 + a->clip_high), (float)(1.0 - a->clip_low), (float)a->kl_coef};
  double *count = (double*)a->workspace, *total = count + a->rows, *part = total + 1;
  const int nb = al_blocks(a->rows * a->cols);
  PCM_LAUNCH(policy_count_kernel, dim3((unsigned)a->rows), dim3(256), 0, stream, pc, count);
  PCM_LAUNCH(policy_total_kernel, dim3(1), dim3(256), 0, stream, (const double*)count, a->rows, total);
  pcm_with_dtype(a->dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    PCM_LAUNCH(policy_main_kernel<Dt>, dim3(nb), dim3(256), 0, stream, (cp)a->logp, a->ld_logp, (cp)a->old_logp, a->ld_old, (cp)a->ref_logp, a->ld_ref,
               a->advantages, a->ld_adv, a->adv_per_row, pc, con, a->reduce, (float)a->grad_scale, (const double*)count, (const double*)total,
               (typename Dt::raw*)a->dlogp, a->ld_dlogp, a->rows, part);
  });
  PCM_LAUNCH(policy_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)part, nb, (const double*)total, a->kl_coef, a->loss, a->stats);
  return pcm_post_launch("pcm_policy_loss");
}
