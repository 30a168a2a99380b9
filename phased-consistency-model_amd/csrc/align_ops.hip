// pcm-build-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Alignment of a distilled student: preference losses over paired log ratios, the clipped policy loss with its KL term, and the log-probability
// of a noisy sampler transition, each with its gradient.  Everything here is bound by memory: a few operations per element read.
//
// Elements are formed in fp32; every sum over elements, rows or tokens is carried in fp64 and in an order fixed by the launch (partial sums in the
// caller's workspace, added up by index), so results are bitwise the same run to run.
#include "dtype_dev.h"

#define AL_LOOP(i, n) for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < (n); i += (long)gridDim.x * blockDim.x)
static inline int al_blocks(long n) { long b = (n + 255) / 256; return (int)(b > PCM_GRID_CAP(2048) ? PCM_GRID_CAP(2048) : (b < 1 ? 1 : b)); }

// ---- work of one team (a wave or a workgroup of NT threads) on elements [i0, i1) of a row, U groups of 16 bytes per thread in flight ----
// f(idx, left): the group of VEC elements at idx, `left` of them inside the range (>= VEC: all)
template <typename Dt, int NT, int U, typename Load, typename Use>
__device__ __forceinline__ void al_groups(long i0, long i1, int tid, Load&& load, Use&& use) {
  constexpr long STEP = (long)NT * Dt::VEC;
  long i = i0 + (long)tid * Dt::VEC;
  for (; i + (U - 1) * STEP + Dt::VEC <= i1; i += U * STEP) {
#pragma unroll
    for (int u = 0; u < U; u++) load(u, i + u * STEP, (long)Dt::VEC);
#pragma unroll
    for (int u = 0; u < U; u++) use(u, i + u * STEP, (long)Dt::VEC);
  }
  for (; i < i1; i += STEP) { load(0, i, i1 - i); use(0, i, i1 - i); }
}
// how a launch cuts rows of n elements: teams of 64 (four rows to a workgroup) for short rows, else `chunks` workgroups of 256 per row, so that some
// 2048 workgroups (8 per CU) share the work; at most 64 chunks, whose partial sums one wave adds up with one load per lane.
struct RowCut { int team, chunks; long len; };
static RowCut row_cut(long rows, long n, int vec) {
  RowCut c = {256, 1, n};
  if (n <= 1024) { c.team = 64; return c; }
  const long unit = 256L * vec, most = (n + unit - 1) / unit, want = 2048 / rows;
  long k = want < 1 ? 1 : (want < most ? want : most);
  if (k > 64) k = 64;
  c.len = ((n + k - 1) / k + unit - 1) / unit * unit;
  c.chunks = (int)((n + c.len - 1) / c.len);
  return c;
}
static inline unsigned row_cut_blocks(const RowCut& c, long rows) { return (unsigned)(c.team == 64 ? (rows + 3) / 4 : rows * c.chunks); }
// (row, chunk, thread of the team) of a thread; false: a team past the last row
template <int TEAM>
__device__ __forceinline__ bool row_cut_place(long block, long rows, int chunks, long* row, int* chunk, int* tid) {
  if (TEAM == 64) { *row = block * 4 + (threadIdx.x >> 6); *chunk = 0; *tid = threadIdx.x & 63; return *row < rows; }
  *row = block / chunks; *chunk = (int)(block - *row * chunks); *tid = threadIdx.x;
  return true;
}

// ---- log-probability of x ~ N(mean, std^2) per row:  -1/2 sum ((x - mean) / std)^2 - n log std - n/2 log 2 pi   (/ n) ----
#define LOG_2PI 1.8378770664093454836
__device__ __forceinline__ float transition_value(double acc, double s, long n, int mean_reduce) {
  const double per = -0.5 * acc / (s * s * (double)n) - log(s) - 0.5 * LOG_2PI;
  return (float)(mean_reduce ? per : per * (double)n);
}
template <typename Dt, int TEAM>
__global__ __launch_bounds__(256) void transition_fwd_kernel(const typename Dt::raw* x, const typename Dt::raw* mean, const float* std, float* logp, double* part,
                                                             long rows, long n, int chunks, long len, int mean_reduce) {
  __shared__ double red[4];
  long row; int chunk, tid;
  if (!row_cut_place<TEAM>(blockIdx.x, rows, chunks, &row, &chunk, &tid)) return;
  const long i0 = chunk * len, i1 = i0 + len < n ? i0 + len : n;
  const typename Dt::raw *xr = x + row * n, *mr = mean + row * n;
  float a[4][Dt::VEC], b[4][Dt::VEC];
  double acc = 0.0;
  al_groups<Dt, TEAM, 4>(i0, i1, tid,
    [&](int u, long i, long left) { pcm_ld_group<Dt>(xr + i, left, a[u]); pcm_ld_group<Dt>(mr + i, left, b[u]); },
    [&](int u, long i, long left) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < Dt::VEC; j++) { const float d = a[u][j] - b[u][j]; t += d * d; }
      acc += (double)t;
    });
  acc = pcm_block_sum<TEAM>(acc, red);
  if (tid == 0) {
    if (chunks == 1) logp[row] = transition_value(acc, (double)std[row], n, mean_reduce);
    else part[row * chunks + chunk] = acc;
  }
}
__global__ __launch_bounds__(256) void transition_finish_kernel(const double* part, const float* std, float* logp, long rows, long n, int chunks, int mean_reduce) {
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  const double acc = pcm_lane_sum(lane < chunks ? part[row * chunks + lane] : 0.0);
  if (lane == 0) logp[row] = transition_value(acc, (double)std[row], n, mean_reduce);
}
template <typename Dt, int TEAM>
__global__ __launch_bounds__(256) void transition_bwd_kernel(const typename Dt::raw* x, const typename Dt::raw* mean, const float* std,
                                                             const float* dlogp, typename Dt::raw* dmean, long rows, long n, int chunks, long len, int mean_reduce) {
  long row; int chunk, tid;
  if (!row_cut_place<TEAM>(blockIdx.x, rows, chunks, &row, &chunk, &tid)) return;
  const long i0 = chunk * len, i1 = i0 + len < n ? i0 + len : n;
  const typename Dt::raw *xr = x + row * n, *mr = mean + row * n;
  typename Dt::raw* dr = dmean + row * n;
  const double s = (double)std[row];
  const float f = (float)((double)dlogp[row] / (s * s * (mean_reduce ? (double)n : 1.0)));
  float a[4][Dt::VEC], b[4][Dt::VEC];
  al_groups<Dt, TEAM, 4>(i0, i1, tid,
    [&](int u, long i, long left) { pcm_ld_group<Dt>(xr + i, left, a[u]); pcm_ld_group<Dt>(mr + i, left, b[u]); },
    [&](int u, long i, long left) {
#pragma unroll
      for (int j = 0; j < Dt::VEC; j++) a[u][j] = (a[u][j] - b[u][j]) * f;
      pcm_st_group<Dt>(dr + i, left, a[u]);
    });
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
// A source of log ratios gives, for a range of a row: sums() -- what the thread adds to the row's sums; and grad() -- its part of the gradient, f being
// the row's factor.  rho() and factor() turn a row's sums into its log ratio and into what multiplies the pair's slope in f.
// Denoising errors: rho = -w k sum ((t - p)^2 - (t - r)^2);  d rho / d p = 2 w k (t - p)
template <typename Dt_>
struct DenoiseRows {
  typedef Dt_ Dt;
  typedef typename Dt::raw raw;
  const raw *pred, *ref, *target;
  const float* weight;
  raw* dpred;
  double k;
  long n;
  static constexpr int SUMS = 1;
  template <int NT>
  __device__ __forceinline__ void sums(long row, long i0, long i1, int tid, double (&acc)[SUMS]) const {
    const long o = row * n;
    float t[4][Dt::VEC], p[4][Dt::VEC], r[4][Dt::VEC];
    double s = 0.0;
    al_groups<Dt, NT, 4>(i0, i1, tid,
      [&](int u, long i, long left) {
        pcm_ld_group<Dt>(target + o + i, left, t[u]); pcm_ld_group<Dt>(pred + o + i, left, p[u]); pcm_ld_group<Dt>(ref + o + i, left, r[u]);
      },
      [&](int u, long i, long left) {
        float e = 0.f;
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) { const float a = t[u][j] - p[u][j], b = t[u][j] - r[u][j]; e += a * a - b * b; }
        s += (double)e;
      });
    acc[0] = s;
  }
  template <int NT>
  __device__ __forceinline__ void grad(long row, long i0, long i1, int tid, float f) const {
    const long o = row * n;
    float t[4][Dt::VEC], p[4][Dt::VEC];
    al_groups<Dt, NT, 4>(i0, i1, tid,
      [&](int u, long i, long left) { pcm_ld_group<Dt>(target + o + i, left, t[u]); pcm_ld_group<Dt>(pred + o + i, left, p[u]); },
      [&](int u, long i, long left) {
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) t[u][j] = (t[u][j] - p[u][j]) * f;
        pcm_st_group<Dt>(dpred + o + i, left, t[u]);
      });
  }
  __device__ __forceinline__ double scale(long row) const { return k * (weight ? (double)weight[row] : 1.0); }
  __device__ __forceinline__ double rho(long row, const double (&s)[SUMS]) const { return -s[0] * scale(row); }
  __device__ __forceinline__ double factor(long row, const double (&s)[SUMS]) const { return 2.0 * scale(row); }
  bool wants_grad() const { return dpred != nullptr; }
};
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
  // bit j: place c + j of the row counts, c + j < c + left and < len
  template <int VEC>
  __device__ __forceinline__ unsigned bits(long row, long c, long len) const {
    const long left = len - c;
    if (left <= 0) return 0u;
    unsigned in = left >= VEC ? (1u << VEC) - 1u : (1u << left) - 1u;
    if (mask) {
      const unsigned char* m = mask + row * ld_mask + c;
      unsigned got = 0u;
      if (left >= VEC) {
        typedef unsigned char mv __attribute__((ext_vector_type(VEC), aligned(1)));
        const mv b = *(const mv*)m;
#pragma unroll
        for (int j = 0; j < VEC; j++) got |= b[j] ? 1u << j : 0u;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++)
          if (j < left) got |= m[j] ? 1u << j : 0u;
      }
      in &= got;
    }
    return in;
  }
};
// log-probabilities: rho = sum (mean) over the places that count of logp - ref;  d rho / d logp = 1 (1 / count) there
template <typename Dt_>
struct TokenRows {
  typedef Dt_ Dt;
  typedef typename Dt::raw raw;
  const raw* logp; long ld_logp;
  const raw* ref; long ld_ref;
  Places pc;
  raw* dlogp; long ld_d;
  int mean_reduce;
  static constexpr int SUMS = 2;
  template <int NT>
  __device__ __forceinline__ void sums(long row, long i0, long i1, int tid, double (&acc)[SUMS]) const {
    const raw *lr = logp + row * ld_logp, *rr = ref + row * ld_ref;
    const long len = pc.len(row);
    float a[2][Dt::VEC], b[2][Dt::VEC];
    unsigned in[2];
    double s = 0.0;
    int cnt = 0;
    al_groups<Dt, NT, 2>(i0, len < i1 ? len : i1, tid,
      [&](int u, long i, long left) {
        in[u] = pc.bits<Dt::VEC>(row, i, len);
        pcm_ld_group<Dt>(lr + i, left, a[u]); pcm_ld_group<Dt>(rr + i, left, b[u]);
      },
      [&](int u, long i, long left) {
        float e = 0.f;
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) { e += in[u] >> j & 1u ? a[u][j] - b[u][j] : 0.f; cnt += in[u] >> j & 1u; }
        s += (double)e;
      });
    acc[0] = s; acc[1] = (double)cnt;
  }
  template <int NT>
  __device__ __forceinline__ void grad(long row, long i0, long i1, int tid, float f) const {
    const long len = pc.len(row);
    unsigned in[2];
    al_groups<Dt, NT, 2>(i0, i1, tid,
      [&](int u, long i, long left) { in[u] = pc.bits<Dt::VEC>(row, i, len); },
      [&](int u, long i, long left) {
        float g[Dt::VEC];
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) g[j] = in[u] >> j & 1u ? f : 0.f;
        pcm_st_group<Dt>(dlogp + row * ld_d + i, left, g);
      });
  }
  __device__ __forceinline__ double share(const double (&s)[SUMS]) const { return mean_reduce ? 1.0 / fmax(s[1], 1.0) : 1.0; }
  __device__ __forceinline__ double rho(long row, const double (&s)[SUMS]) const { return s[0] * share(s); }
  __device__ __forceinline__ double factor(long row, const double (&s)[SUMS]) const { return share(s); }
  bool wants_grad() const { return dlogp != nullptr; }
};
// Two launches: (1) partial sums of every (row, chunk); (2) the gradient, where each team adds up the partial sums of its pair again instead of
// waiting for a launch that does it once -- at most 2 x 64 numbers out of L2 -- and the first workgroup forms the mean loss.
template <typename R, int TEAM>
__global__ __launch_bounds__(256) void pair_sums_kernel(R rows_, double* part, long rows, long n, int chunks, long len) {
  __shared__ double red[4];
  long row; int chunk, tid;
  if (!row_cut_place<TEAM>(blockIdx.x, rows, chunks, &row, &chunk, &tid)) return;
  const long i0 = chunk * len, i1 = i0 + len < n ? i0 + len : n;
  double acc[R::SUMS];
  rows_.template sums<TEAM>(row, i0, i1, tid, acc);
#pragma unroll
  for (int a = 0; a < R::SUMS; a++) acc[a] = pcm_block_sum<TEAM>(acc[a], red);
  if (tid == 0)
#pragma unroll
    for (int a = 0; a < R::SUMS; a++) part[(row * chunks + chunk) * R::SUMS + a] = acc[a];
}
template <typename R>
__device__ __forceinline__ void pair_row_total(const double* part, long row, int chunks, int lane, double (&s)[R::SUMS]) {
#pragma unroll
  for (int a = 0; a < R::SUMS; a++) s[a] = pcm_lane_sum(lane < chunks ? part[(row * chunks + lane) * R::SUMS + a] : 0.0);
}
template <typename R, int TEAM>
__global__ __launch_bounds__(256) void pair_grad_kernel(R rows_, const double* part, PairLoss pl, double gscale, float* loss, float* log_ratio, long pairs,
                                                        long n, int chunks, long len) {
  __shared__ double red[4];
  if (blockIdx.x == 0) {
    double acc = 0.0;
    for (long p = threadIdx.x; p < pairs; p += 256) {
      double rho[2], l, s;
      for (int side = 0; side < 2; side++) {
        const long row = p + side * pairs;
        double t[R::SUMS];
#pragma unroll
        for (int a = 0; a < R::SUMS; a++) t[a] = 0.0;
        for (int c = 0; c < chunks; c++)
#pragma unroll
          for (int a = 0; a < R::SUMS; a++) t[a] += part[(row * chunks + c) * R::SUMS + a];
        rho[side] = rows_.rho(row, t);
        log_ratio[row] = (float)rho[side];
      }
      pair_loss(pl, rho[0] - rho[1], &l, &s);
      acc += l;
    }
    acc = pcm_block_sum<256>(acc, red);
    if (threadIdx.x == 0) loss[0] = (float)(acc / (double)pairs);
    return;
  }
  long row; int chunk, tid;
  if (!row_cut_place<TEAM>(blockIdx.x - 1, 2 * pairs, chunks, &row, &chunk, &tid)) return;
  const long i0 = chunk * len, i1 = i0 + len < n ? i0 + len : n, p = row < pairs ? row : row - pairs;
  double up[R::SUMS], down[R::SUMS], l, s;
  pair_row_total<R>(part, p, chunks, threadIdx.x & 63, up);
  pair_row_total<R>(part, pairs + p, chunks, threadIdx.x & 63, down);
  pair_loss(pl, rows_.rho(p, up) - rows_.rho(pairs + p, down), &l, &s);
  const double f = (row < pairs ? s * rows_.factor(row, up) : -s * rows_.factor(row, down)) * gscale / (double)pairs;
  rows_.template grad<TEAM>(row, i0, i1, tid, (float)f);
}
// bytes of the partial sums
static size_t pair_ws_bytes(long rows, long n, int vec, int sums) { const RowCut c = row_cut(rows, n, vec); return (size_t)rows * c.chunks * sums * sizeof(double); }
template <typename R>
static void pair_launch(const R& r, double* part, const PairLoss& pl, double gscale, float* loss, float* log_ratio, long pairs, long n, void* stream) {
  const long rows = 2 * pairs;
  const RowCut c = row_cut(rows, n, R::Dt::VEC);
  const unsigned nb = row_cut_blocks(c, rows), ng = r.wants_grad() ? nb + 1 : 1;
  if (c.team == 64) {
    PCM_LAUNCH((pair_sums_kernel<R, 64>), dim3(nb), dim3(256), 0, stream, r, part, rows, n, c.chunks, c.len);
    PCM_LAUNCH((pair_grad_kernel<R, 64>), dim3(ng), dim3(256), 0, stream, r, (const double*)part, pl, gscale, loss, log_ratio, pairs, n, c.chunks, c.len);
  } else {
    PCM_LAUNCH((pair_sums_kernel<R, 256>), dim3(nb), dim3(256), 0, stream, r, part, rows, n, c.chunks, c.len);
    PCM_LAUNCH((pair_grad_kernel<R, 256>), dim3(ng), dim3(256), 0, stream, r, (const double*)part, pl, gscale, loss, log_ratio, pairs, n, c.chunks, c.len);
  }
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
#define AL_MAX_ROWS 16777216L       /* 64 chunks of a row at the most: a grid stays below 2^31 workgroups */
extern "C" size_t pcm_transition_logprob_workspace_bytes(long rows, long n) {
  if (rows <= 0 || n <= 0) return 0;
  const RowCut c = row_cut(rows, n, 4);      // (the 16-bit formats cut into no more chunks than fp32)
  return c.chunks > 1 ? (size_t)rows * c.chunks * sizeof(double) : 0;
}
#define TRANSITION_LAUNCH(kernel, ...)                                                                                       \
  do {                                                                                                                       \
    if (c.team == 64) PCM_LAUNCH((kernel<Dt, 64>), dim3(row_cut_blocks(c, rows)), dim3(256), 0, stream, __VA_ARGS__);        \
    else PCM_LAUNCH((kernel<Dt, 256>), dim3(row_cut_blocks(c, rows)), dim3(256), 0, stream, __VA_ARGS__);                    \
  } while (0)
extern "C" int pcm_transition_logprob(const void* x, const void* mean, const float* std, int dtype, int mean_reduce, float* logp, long rows, long n,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  PCM_CHECK(x && mean && std && logp && pcm_dt_ok(dtype) && rows > 0 && rows <= AL_MAX_ROWS && n > 0, PCM_EINVAL, "pcm_transition_logprob: null/empty or unknown format");
  const size_t need = pcm_transition_logprob_workspace_bytes(rows, n);
  PCM_CHECK(need == 0 || (workspace && ((uintptr_t)workspace % 8) == 0 && workspace_bytes >= need), PCM_EINVAL,
            "pcm_transition_logprob: workspace too small or not 8-byte aligned");
  pcm_with_dtype(dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    const RowCut c = row_cut(rows, n, Dt::VEC);
    TRANSITION_LAUNCH(transition_fwd_kernel, (cp)x, (cp)mean, std, logp, (double*)workspace, rows, n, c.chunks, c.len, mean_reduce);
    if (c.chunks > 1)
      PCM_LAUNCH(transition_finish_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, (const double*)workspace, std, logp, rows, n, c.chunks, mean_reduce);
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
    const RowCut c = row_cut(rows, n, Dt::VEC);
    TRANSITION_LAUNCH(transition_bwd_kernel, (cp)x, (cp)mean, std, dlogp, (typename Dt::raw*)dmean, rows, n, c.chunks, c.len, mean_reduce);
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
extern "C" size_t pcm_denoise_preference_loss_workspace_bytes(long pairs, long n) { return pairs > 0 && n > 0 ? pair_ws_bytes(2 * pairs, n, 4, DenoiseRows<DtF32>::SUMS) : 0; }
extern "C" int pcm_denoise_preference_loss(const pcm_denoise_preference_args* a, void* stream) {
  PCM_CHECK(a && a->pred && a->ref && a->target && a->loss && a->log_ratio && a->n > 0, PCM_EINVAL, "pcm_denoise_preference_loss: null/empty");
  const int rc = pair_args_ok("pcm_denoise_preference_loss", a->dtype, a->pairs, a->beta, a->kind, a->label_smoothing);
  if (rc != PCM_OK) return rc;
  PCM_CHECK(a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= pcm_denoise_preference_loss_workspace_bytes(a->pairs, a->n), PCM_EINVAL,
            "pcm_denoise_preference_loss: workspace too small or not 8-byte aligned");
  const PairLoss pl = {a->beta, a->label_smoothing, a->kind};
  const double k = a->mean_reduce ? 1.0 / (double)a->n : 1.0;
  pcm_with_dtype(a->dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    const DenoiseRows<Dt> r = {(cp)a->pred, (cp)a->ref, (cp)a->target, a->weight, (typename Dt::raw*)a->dpred, k, a->n};
    pair_launch(r, (double*)a->workspace, pl, a->grad_scale, a->loss, a->log_ratio, a->pairs, a->n, stream);
  });
  return pcm_post_launch("pcm_denoise_preference_loss");
}
extern "C" size_t pcm_preference_loss_workspace_bytes(long pairs, long cols) { return pairs > 0 && cols > 0 ? pair_ws_bytes(2 * pairs, cols, 4, TokenRows<DtF32>::SUMS) : 0; }
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
  pcm_with_dtype(a->dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    const TokenRows<Dt> r = {(cp)a->logp, a->ld_logp, (cp)a->ref_logp, a->ld_ref, pc, (typename Dt::raw*)a->dlogp, a->ld_dlogp, a->mean_reduce};
    pair_launch(r, (double*)a->workspace, pl, a->grad_scale, a->loss, a->log_ratio, a->pairs, a->cols, stream);
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
