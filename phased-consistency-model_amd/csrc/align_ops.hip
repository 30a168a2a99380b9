// pcm-build-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Alignment of a distilled student: preference losses over paired log ratios, the clipped policy loss with its KL term, and the log-probability
// of a noisy sampler transition, each with its gradient.  Everything here is bound by memory: a few operations per element read.
//
// Elements are formed in fp32; every sum over elements, rows or tokens is carried in fp64 and in an order fixed by the launch (partial sums in the
// caller's workspace, added up by index), so results are bitwise the same run to run.
#include "dtype_dev.h"

static inline int al_blocks(long n) { long b = (n + 255) / 256; return (int)(b > PCM_GRID_CAP(2048) ? PCM_GRID_CAP(2048) : (b < 1 ? 1 : b)); }

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
  pcm_groups<Dt, TEAM, 4>(i0, i1, tid,
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
  pcm_groups<Dt, TEAM, 4>(i0, i1, tid,
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
    pcm_groups<Dt, NT, 4>(i0, i1, tid,
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
    pcm_groups<Dt, NT, 4>(i0, i1, tid,
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
    pcm_groups<Dt, NT, 2>(i0, len < i1 ? len : i1, tid,
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
    pcm_groups<Dt, NT, 2>(i0, i1, tid,
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
template <typename Dt_>
struct PolicyRows {
  typedef Dt_ Dt;
  typedef typename Dt::raw raw;
  const raw *logp, *old, *ref;      // old / ref may be NULL
  long ld_logp, ld_old, ld_ref;
  const float* adv;
  long ld_adv;                      // 0: one per row
  Places pc;
  PolicyConst con;
  raw* dlogp;                       // NULL: no gradient
  long ld_d, rows;
  float gscale;
  int reduce;
};
struct PolicySums { double obj, kl, held, count; };
// Groups of VEC places inside a row, numbered row by row; the thread takes g, g + step, ... and keeps (row, group of the row) by addition.  Groups in which
// nothing counts read nothing.  weight(row, len) is the row's weight in the loss.
template <typename Dt, typename W>
__device__ __forceinline__ void policy_groups(const PolicyRows<Dt>& a, long g, long step, W&& weight, PolicySums& s) {
  constexpr int V = Dt::VEC;
  const long cols = a.pc.cols, gpr = (cols + V - 1) / V, drow = step / gpr, dcol = step - drow * gpr;
  long row = g / gpr, col = g - row * gpr;
  while (row < a.rows) {
    const long c = col * V, left = cols - c, len = a.pc.len(row);
    const unsigned in = a.pc.template bits<V>(row, c, len);
    float out[V];
#pragma unroll
    for (int j = 0; j < V; j++) out[j] = 0.f;
    if (in) {
      float lp[V], old[V], ref[V], adv[V];
      pcm_ld_group<Dt>(a.logp + row * a.ld_logp + c, left, lp);
      if (a.old) pcm_ld_group<Dt>(a.old + row * a.ld_old + c, left, old);
      if (a.ref) pcm_ld_group<Dt>(a.ref + row * a.ld_ref + c, left, ref);
      if (a.ld_adv) pcm_ld_group<DtF32>(a.adv + row * a.ld_adv + c, left, adv);
      else {
        const float one = a.adv[row];
#pragma unroll
        for (int j = 0; j < V; j++) adv[j] = one;
      }
      const double w = weight(row, len);
      const float wg = (float)(w * (double)a.gscale);
      float so = 0.f, sk = 0.f;
      int held = 0;
#pragma unroll
      for (int j = 0; j < V; j++) {
        float obj, kl, slope;
        bool clipped;
        policy_place(a.con, lp[j], a.old ? old[j] : lp[j], a.ref != nullptr, a.ref ? ref[j] : 0.f, adv[j], &obj, &kl, &slope, &clipped);
        const bool counts = in >> j & 1u;
        so += counts ? obj : 0.f;
        sk += counts ? kl : 0.f;
        held += counts && clipped ? 1 : 0;
        out[j] = counts ? slope * wg : 0.f;
      }
      s.obj += w * (double)so; s.kl += w * (double)sk; s.held += (double)held; s.count += (double)__builtin_popcount(in);
    }
    if (a.dlogp) pcm_st_group<Dt>(a.dlogp + row * a.ld_d + c, left, out);
    col += dcol; row += drow;
    if (col >= gpr) { col -= gpr; row++; }
  }
}
// how many places count, where the launch has to find out: per row (mean of row means) or in all, as partial sums over groups of 16 places
__device__ __forceinline__ long count_groups(const Places& pc, long rows, long g, long step) {
  const long gpr = (pc.cols + 15) / 16, drow = step / gpr, dcol = step - drow * gpr;
  long row = g / gpr, col = g - row * gpr, n = 0;
  while (row < rows) {
    n += __builtin_popcount(pc.bits<16>(row, col * 16, pc.len(row)));
    col += dcol; row += drow;
    if (col >= gpr) { col -= gpr; row++; }
  }
  return n;
}
__global__ __launch_bounds__(256) void policy_count_kernel(Places pc, long rows, double* part) {
  __shared__ long red[4];
  long n = 0;
  if (pc.mask) n = count_groups(pc, rows, (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256);
  else for (long r = (long)blockIdx.x * 256 + threadIdx.x; r < rows; r += (long)gridDim.x * 256) n += pc.len(r);
  n = pcm_block_sum<256>(n, red);
  if (threadIdx.x == 0) part[blockIdx.x] = (double)n;
}
template <int TEAM>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void policy_count_rows_kernel(Places pc, long rows, double* count) {
  __shared__ long red[16];
  const long row = TEAM == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= rows) return;
  const int tid = TEAM == 64 ? threadIdx.x & 63 : threadIdx.x;
  const long len = pc.len(row);
  long n = 0;
  for (long c = tid * 16L; c < len; c += TEAM * 16L) n += __builtin_popcount(pc.bits<16>(row, c, len));
  n = pcm_block_sum<TEAM>(n, red);
  if (tid == 0) count[row] = (double)n;
}
// where the number of places comes from: the launch's arguments, partial sums of a launch before, or the lengths themselves
struct PolicyCount { double known; const double* part; int nparts; const double* per_row; };
template <typename Dt, int NT>
__device__ __forceinline__ void policy_part(const PolicyRows<Dt>& a, const PolicyCount& pn, long g, long step, double* red, PolicySums& s) {
  s.obj = s.kl = s.held = s.count = 0.0;
  if (a.reduce == PCM_POLICY_TOKEN) {
    double n = pn.known;
    if (pn.part) {
      n = 0.0;
      for (int i = threadIdx.x; i < pn.nparts; i += NT) n += pn.part[i];
      n = pcm_block_sum<NT>(n, red);
    } else if (n < 0.0) {
      long t = 0;
      for (long r = threadIdx.x; r < a.rows; r += NT) t += a.pc.len(r);
      n = pcm_block_sum<NT>((double)t, red);
    }
    const double w = 1.0 / fmax(n, 1.0);
    policy_groups(a, g, step, [&](long, long) { return w; }, s);
  } else if (a.reduce == PCM_POLICY_ROW) {
    policy_groups(a, g, step, [&](long row, long len) { return 1.0 / ((pn.per_row ? pn.per_row[row] : (double)len) * (double)a.rows); }, s);
  } else {
    policy_groups(a, g, step, [&](long, long) { return 1.0; }, s);
  }
  s.obj = pcm_block_sum<NT>(s.obj, red); s.kl = pcm_block_sum<NT>(s.kl, red);
  s.held = pcm_block_sum<NT>(s.held, red); s.count = pcm_block_sum<NT>(s.count, red);
}
__device__ __forceinline__ void policy_result(const PolicySums& s, double kl, float* loss, float* stats) {
  loss[0] = (float)(s.obj + kl * s.kl);
  stats[0] = (float)s.obj; stats[1] = (float)s.kl; stats[2] = (float)(s.held / fmax(s.count, 1.0)); stats[3] = (float)s.count;
}
template <typename Dt>
__global__ __launch_bounds__(256) void policy_main_kernel(PolicyRows<Dt> a, PolicyCount pn, double* part) {
  __shared__ double red[4];
  PolicySums s;
  policy_part<Dt, 256>(a, pn, (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256, red, s);
  if (threadIdx.x == 0) { double* q = part + 4 * (long)blockIdx.x; q[0] = s.obj; q[1] = s.kl; q[2] = s.held; q[3] = s.count; }
}
__global__ __launch_bounds__(256) void policy_finish_kernel(const double* part, int nparts, double kl, float* loss, float* stats) {
  __shared__ double red[4];
  PolicySums s = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < nparts; i += 256) { s.obj += part[4 * i]; s.kl += part[4 * i + 1]; s.held += part[4 * i + 2]; s.count += part[4 * i + 3]; }
  s.obj = pcm_block_sum<256>(s.obj, red); s.kl = pcm_block_sum<256>(s.kl, red);
  s.held = pcm_block_sum<256>(s.held, red); s.count = pcm_block_sum<256>(s.count, red);
  if (threadIdx.x == 0) policy_result(s, kl, loss, stats);
}
// few places: one workgroup counts, forms loss and gradient, and adds up, in one launch
#define POLICY_SMALL_PLACES 16384
#define POLICY_SMALL_ROWS 2048
template <typename Dt>
__global__ __launch_bounds__(1024) void policy_small_kernel(PolicyRows<Dt> a, double kl, float* loss, float* stats) {
  __shared__ double red[16];
  __shared__ double per_row[POLICY_SMALL_ROWS];
  PolicyCount pn = {-1.0, nullptr, 0, nullptr};
  if (a.pc.mask && a.reduce == PCM_POLICY_TOKEN) {
    pn.known = pcm_block_sum<1024>((double)count_groups(a.pc, a.rows, threadIdx.x, 1024), red);
  } else if (a.pc.mask && a.reduce == PCM_POLICY_ROW) {
    for (long row = threadIdx.x >> 6; row < a.rows; row += 16) {
      const long len = a.pc.len(row);
      long n = 0;
      for (long c = (threadIdx.x & 63) * 16L; c < len; c += 64 * 16L) n += __builtin_popcount(a.pc.template bits<16>(row, c, len));
      n = pcm_lane_sum(n);
      if ((threadIdx.x & 63) == 0) per_row[row] = (double)n;
    }
    __syncthreads();
    pn.per_row = per_row;
  }
  PolicySums s;
  policy_part<Dt, 1024>(a, pn, threadIdx.x, 1024, red, s);
  if (threadIdx.x == 0) policy_result(s, kl, loss, stats);
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
static bool policy_small(long rows, long cols) { return rows <= POLICY_SMALL_ROWS && rows * cols <= POLICY_SMALL_PLACES; }
static int policy_blocks(long rows, long cols, int vec) { return al_blocks(rows * ((cols + vec - 1) / vec)); }
#define POLICY_COUNT_PARTS 512
extern "C" size_t pcm_policy_loss_workspace_bytes(long rows, long cols) {
  if (rows <= 0 || cols <= 0 || policy_small(rows, cols)) return 0;
  return ((size_t)(rows > POLICY_COUNT_PARTS ? rows : POLICY_COUNT_PARTS) + 4 * (size_t)policy_blocks(rows, cols, 4)) * sizeof(double);
}
extern "C" int pcm_policy_loss(const pcm_policy_args* a, void* stream) {
  PCM_CHECK(a && a->logp && a->advantages && a->loss && a->stats && a->rows > 0 && a->rows <= AL_MAX_ROWS && a->cols > 0, PCM_EINVAL, "pcm_policy_loss: null/empty");
  PCM_CHECK(pcm_dt_ok(a->dtype), PCM_EINVAL, "pcm_policy_loss: unknown element format %d", a->dtype);
  PCM_CHECK(a->reduce == PCM_POLICY_TOKEN || a->reduce == PCM_POLICY_ROW || a->reduce == PCM_POLICY_SUM, PCM_EINVAL, "pcm_policy_loss: unknown reduce %d", a->reduce);
  PCM_CHECK(a->clip_low >= 0.0 && a->clip_low < 1.0 && a->clip_high >= 0.0 && a->clip_high < 1e30, PCM_EINVAL, "pcm_policy_loss: clip_low must be in [0, 1), clip_high >= 0");
  PCM_CHECK(a->kl_coef == 0.0 || a->ref_logp, PCM_EINVAL, "pcm_policy_loss: a KL term needs the reference log-probabilities");
  PCM_CHECK(a->ld_logp >= a->cols && (!a->old_logp || a->ld_old >= a->cols) && (!a->ref_logp || a->ld_ref >= a->cols) && (a->adv_per_row || a->ld_adv >= a->cols) &&
                (!a->mask || a->ld_mask >= a->cols) && (!a->dlogp || a->ld_dlogp >= a->cols), PCM_EINVAL, "pcm_policy_loss: row stride below the row length");
  const size_t need = pcm_policy_loss_workspace_bytes(a->rows, a->cols);
  PCM_CHECK(need == 0 || (a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= need), PCM_EINVAL,
            "pcm_policy_loss: workspace too small or not 8-byte aligned");
  const Places pc = {a->mask, a->ld_mask, a->lengths, a->lengths_i64, a->cols};
  const PolicyConst con = {log1p(a->clip_high), log1p(-a->clip_low), (float)(1.0 + a->clip_high), (float)(1.0 - a->clip_low), (float)a->kl_coef};
  const long rows = a->rows;
  const int reduce = a->reduce == PCM_POLICY_ROW && rows == 1 ? PCM_POLICY_TOKEN : a->reduce;      // one row: its mean is the mean of all places
  pcm_with_dtype(a->dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    const PolicyRows<Dt> r = {(cp)a->logp, (cp)a->old_logp, (cp)a->ref_logp, a->ld_logp, a->ld_old, a->ld_ref, a->advantages, a->adv_per_row ? 0 : a->ld_adv, pc, con,
                              (typename Dt::raw*)a->dlogp, a->ld_dlogp, rows, (float)a->grad_scale, reduce};
    if (need == 0) {
      PCM_LAUNCH(policy_small_kernel<Dt>, dim3(1), dim3(1024), 0, stream, r, a->kl_coef, a->loss, a->stats);
      return;
    }
    double *counts = (double*)a->workspace, *part = counts + (rows > POLICY_COUNT_PARTS ? rows : POLICY_COUNT_PARTS);
    PolicyCount pn = {-1.0, nullptr, 0, nullptr};
    if (reduce == PCM_POLICY_TOKEN) {
      if (!a->mask && !a->lengths) pn.known = (double)rows * (double)a->cols;
      else if (a->mask || rows > 4096) {          // (up to 4096 lengths each workgroup adds up itself: 16 loads a thread against a launch)
        const long b = a->mask ? al_blocks(rows * ((a->cols + 15) / 16)) : al_blocks(rows);
        pn.nparts = (int)(b < POLICY_COUNT_PARTS ? b : POLICY_COUNT_PARTS);
        pn.part = counts;
        PCM_LAUNCH(policy_count_kernel, dim3(pn.nparts), dim3(256), 0, stream, pc, rows, counts);
      }
    } else if (reduce == PCM_POLICY_ROW && a->mask) {
      pn.per_row = counts;
      if (a->cols <= 4096) PCM_LAUNCH(policy_count_rows_kernel<64>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, pc, rows, counts);
      else PCM_LAUNCH(policy_count_rows_kernel<1024>, dim3((unsigned)rows), dim3(1024), 0, stream, pc, rows, counts);
    }
    const int nb = policy_blocks(rows, a->cols, Dt::VEC);
    PCM_LAUNCH(policy_main_kernel<Dt>, dim3(nb), dim3(256), 0, stream, r, pn, part);
    PCM_LAUNCH(policy_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)part, nb, a->kl_coef, a->loss, a->stats);
  });
  return pcm_post_launch("pcm_policy_loss");
}
