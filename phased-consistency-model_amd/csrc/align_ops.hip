// pcm-build-flags: -Xclang -target-feature -Xclang -packed-fp32-ops
// Alignment of a distilled student: preference losses over paired log ratios, the clipped policy loss with its KL term, and the log-probability
// of a noisy sampler transition, each with its gradient.  Large calls are bound by memory (a few operations per element read; 60 in the policy loss,
// which is why its exponentials are counted), small ones by their launches: about 4 us of host time each.  Times below are of one MI355X, whose
// large copies run at 5.1 TB/s and whose reads alone reach 6.8.
//
// Elements are formed in fp32 (squares and factors of a transition in fp64); every sum over elements, rows or tokens is carried in fp64 and in an order fixed
// by the launch (partial sums in the caller's workspace, added up by index), so results are bitwise the same run to run.  Two kernels add a thread's group of
// elements in fp32 first, where a sum that leaves fp32 takes terms no run comes by: the denoising errors (4 or 8; terms of 1e38 need predictions of 1e19) and
// the policy loss (4; a ratio or exp(d) of 1e38).  Each into fp64 by itself cost the policy loss 0.6 us of 47.5 (2048 x 8192 fp32 with KL, ragged), 1.7 of 40
// (bf16), and the denoising kernel of few elements registers that spilled.
#include "dtype_dev.h"

static inline int al_blocks(long n) { long b = (n + 255) / 256; return (int)(b > PCM_GRID_CAP(2048) ? PCM_GRID_CAP(2048) : (b < 1 ? 1 : b)); }

#define AL_U (16 / Dt::VEC)      /* groups of a thread in flight: 16 elements of every tensor */
// how a launch cuts rows of n elements: teams of 64 (four rows to a workgroup) for short rows, else `chunks` workgroups of 256 per row, so that some
// 4096 workgroups (two rounds of 8 per CU) share the work; at most 64 chunks, whose partial sums one wave adds up with one load per lane.
// Measured on both sides, us of an eager call / of the same call replayed in a graph, where the host's share is gone:
//   teams up to 1024 elements against 512: transition forward, 2048 rows of 1024 fp32 11.6 / 5.7 against 11.6 / 6.1, bf16 11.7 / 3.8 against 11.6 / 4.6;
//   against 2048: 2048 rows of 1500 fp32 11.7 / 11.0 against 11.6 / 7.1, 64 rows of 1500 11.8 / 3.6 against 11.6 / 3.8; 100 pairs of 1500 18.7 / 7.2 against
//   18.8 / 8.3, 1000 pairs 21.9 / 22.2 against 19.6 / 17.5: few rows want the workgroup, many the wave, and the limit looks at the length alone;
//   64 chunks against 16: transition forward, one row of 2^20 fp32 15.5 / 6.8 against 15.6 / 7.9; one pair of 262144 18.7 / 14.2 against 18.8 / 13.3, 8 pairs
//   28.0 / 28.2 against 22.8 / 22.9: of the pairs' loss, one thread adds up a pair's chunks one by one (pair_losses).
struct RowCut { int team, chunks; long len; };
#define ROW_TEAM_MAX 65536L
static RowCut row_cut(long rows, long n, int vec) {
  RowCut c = {256, 1, n};
  if (n <= 1024) { c.team = 64; return c; }
  const long unit = 256L * vec, most = (n + unit - 1) / unit, want = 4096 / rows;
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
  if (TEAM == 1024) { *row = block; *chunk = 0; *tid = threadIdx.x; return true; }
  if (TEAM == 64) { *row = block * 4 + (threadIdx.x >> 6); *chunk = 0; *tid = threadIdx.x & 63; return *row < rows; }
  *row = block / chunks; *chunk = (int)(block - *row * chunks); *tid = threadIdx.x;
  return true;
}

// ---- Log-probability of a transition.  Forward: one pass, 8 bytes read an element (fp32); 64 rows of 262144 in two launches, 26 us.  Gradient: elementwise
// in the forward's cut of rows, so that std and dlogp are read once a workgroup; 64 rows of 262144 fp32 in 31 us, 201 MB at 6.4 TB/s.  Squares and the gradient's
// factor, dlogp / std^2, are fp64: both leave fp32 long before their results do (deviations below 1e-19 or above 1e19).  The memory hides it: 64 rows of
// 262144 fp32 in 27.0 us either way, bf16 in 17.0 against 16.8 with fp32 squares; the gradient 31.9 against 31.8, bf16 16.2 against 16.1.
// x ~ N(mean, std^2) per row:  -1/2 sum ((x - mean) / std)^2 - n log std - n/2 log 2 pi   (/ n) ----
#define LOG_2PI 1.8378770664093454836
__device__ __forceinline__ float transition_value(double acc, double s, long n, int mean_reduce) {
  const double per = -0.5 * acc / (s * s * (double)n) - log(s) - 0.5 * LOG_2PI;
  return (float)(mean_reduce ? per : per * (double)n);
}
template <typename Dt, int TEAM>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void transition_fwd_kernel(const typename Dt::raw* x, const typename Dt::raw* mean, const float* std,
                                                                                      float* logp, double* part, long rows, long n, int chunks, long len, int mean_reduce) {
  __shared__ double red[16];
  long row; int chunk, tid;
  if (!row_cut_place<TEAM>(blockIdx.x, rows, chunks, &row, &chunk, &tid)) return;
  const long i0 = chunk * len, i1 = i0 + len < n ? i0 + len : n;
  const typename Dt::raw *xr = x + row * n, *mr = mean + row * n;
  float a[AL_U][Dt::VEC], b[AL_U][Dt::VEC];
  double acc = 0.0;
  pcm_groups<Dt, TEAM, AL_U>(i0, i1, tid,
    [&](int u, long i, long left) { pcm_ld_group<Dt>(xr + i, left, a[u]); pcm_ld_group<Dt>(mr + i, left, b[u]); },
    [&](int u, long i, long left) {
#pragma unroll
      for (int j = 0; j < Dt::VEC; j++) { const double d = (double)(a[u][j] - b[u][j]); acc += d * d; }
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
  const double f = (double)dlogp[row] / (s * s * (mean_reduce ? (double)n : 1.0));
  float a[AL_U][Dt::VEC], b[AL_U][Dt::VEC];
  pcm_groups<Dt, TEAM, AL_U>(i0, i1, tid,
    [&](int u, long i, long left) { pcm_ld_group<Dt>(xr + i, left, a[u]); pcm_ld_group<Dt>(mr + i, left, b[u]); },
    [&](int u, long i, long left) {
#pragma unroll
      for (int j = 0; j < Dt::VEC; j++) a[u][j] = (float)((double)(a[u][j] - b[u][j]) * f);
      pcm_st_group<Dt>(dr + i, left, a[u]);
    });
}

// ---- preference losses.  rows [0, P) are the preferred side, [P, 2P) the rejected side; rho = log ratio of a row ----
struct PairLoss { double beta, eps; int kind; };
// loss of one pair and its derivative by the preferred row's rho (the rejected row's is its negative)
__device__ __forceinline__ void pair_loss(const PairLoss p, double h, double* loss, double* slope) {
  if (p.kind == PCM_PAIR_SIGMOID) {
    const double s = p.beta * h, e = exp(-fabs(s)), soft = log1p(e);             // -log sig(s) = soft + max(-s, 0)
    *loss = (1.0 - p.eps) * (soft + fmax(-s, 0.0));
    if (p.eps > 0.0) *loss += p.eps * (soft + fmax(s, 0.0));                      // (not 0 times infinity)
    const double far = e / (1.0 + e), near = 1.0 / (1.0 + e);                     // sig(-|s|), sig(|s|): 1 - sig(|s|) has no digits left where s is large
    *slope = p.beta * (p.eps * (s >= 0.0 ? near : far) - (1.0 - p.eps) * (s >= 0.0 ? far : near));
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
// Denoising errors: rho = -w k sum ((t - p)^2 - (t - r)^2);  d rho / d p = 2 w k (t - p).  The difference of the squares is summed as
// (r - p) ((t - p) + (t - r)): its error shrinks with r - p, and predictions that agree give exactly 0, where squares formed apart cancel.
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
    float t[AL_U][Dt::VEC], p[AL_U][Dt::VEC], r[AL_U][Dt::VEC];
    double s = 0.0;
    pcm_groups<Dt, NT, AL_U>(i0, i1, tid,
      [&](int u, long i, long left) {
        pcm_ld_group<Dt, true>(target + o + i, left, t[u]); pcm_ld_group<Dt, true>(pred + o + i, left, p[u]); pcm_ld_group<Dt, true>(ref + o + i, left, r[u]);
      },
      [&](int u, long i, long left) {
        float e = 0.f;
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) e += (r[u][j] - p[u][j]) * ((t[u][j] - p[u][j]) + (t[u][j] - r[u][j]));
        s += (double)e;
      });
    acc[0] = s;
  }
  template <int NT>
  __device__ __forceinline__ void grad(long row, long i0, long i1, int tid, float f) const {
    const long o = row * n;
    float t[AL_U][Dt::VEC], p[AL_U][Dt::VEC];
    pcm_groups<Dt, NT, AL_U>(i0, i1, tid,
      [&](int u, long i, long left) { pcm_ld_group<Dt, true>(target + o + i, left, t[u]); pcm_ld_group<Dt, true>(pred + o + i, left, p[u]); },
      [&](int u, long i, long left) {
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) t[u][j] = (t[u][j] - p[u][j]) * f;
        pcm_st_group<Dt>(dpred + o + i, left, t[u]);
      });
  }
  __device__ __forceinline__ double scale(long row) const { return k * (weight ? (double)weight[row] : 1.0); }
  __device__ __forceinline__ double rho(long row, const double (&s)[SUMS]) const {
#pragma clang fp contract(off)      // (as in TokenRows)
    return -s[0] * scale(row);
  }
  __device__ __forceinline__ double factor(long row, const double (&s)[SUMS]) const { return 2.0 * scale(row); }
  bool wants_grad() const { return dpred != nullptr; }
};
// element (row, c) of rows ld apart, both below 2^32 (one 32 x 32 -> 64 bit multiply-add)
__device__ __forceinline__ long at(long row, long ld, long c) { return (long)((unsigned long)(unsigned)row * (unsigned)ld + (unsigned long)c); }
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
  // bit j of the result: place c + j counts
  template <int VEC>
  static __device__ __forceinline__ unsigned below(long left) { return left <= 0 ? 0u : (left >= VEC ? (1u << VEC) - 1u : (1u << left) - 1u); }
  template <int VEC>
  __device__ __forceinline__ unsigned bits_inside(long row, long c, long len) const {      // all VEC places are inside the row
    unsigned got = (1u << VEC) - 1u;
    if (mask) {
      typedef unsigned mv __attribute__((ext_vector_type(VEC / 4), aligned(1)));
      const mv b = *(const mv*)(mask + at(row, ld_mask, c));
      got = 0u;
#pragma unroll
      for (int w = 0; w < VEC / 4; w++) {
        // the top bit of a byte that is not 0, then the four of them side by side: 8 j + (24 - 7 j) = 24 + j, the other products fall elsewhere
        const unsigned x = ((((b[w] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | b[w]) >> 7) & 0x01010101u;
        got |= (x * 0x01020408u) >> 24 << (4 * w);
      }
    }
    return got & below<VEC>(len - c);
  }
  template <int VEC>
  __device__ __forceinline__ unsigned bits_end(long row, long c, long len) const {         // the row may end before
    unsigned in = below<VEC>(len - c);
    if (mask) {
#pragma unroll
      for (int j = 0; j < VEC; j++)
        if ((in >> j & 1u) && !mask[at(row, ld_mask, c + j)]) in &= ~(1u << j);
    }
    return in;
  }
  template <int VEC>
  __device__ __forceinline__ unsigned bits(long row, long c, long len) const {
    return c + VEC <= cols ? bits_inside<VEC>(row, c, len) : bits_end<VEC>(row, c, len);
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
        in[u] = left >= Dt::VEC ? pc.bits_inside<Dt::VEC>(row, i, len) : pc.bits_end<Dt::VEC>(row, i, len);
        pcm_ld_group<Dt>(lr + i, left, a[u]); pcm_ld_group<Dt>(rr + i, left, b[u]);
      },
      [&](int u, long i, long left) {
        // (each into the fp64 sum: a few of the lowest number, which stands for a logarithm of 0, leave fp32.  512 pairs of 4096 fp32 in 21.8 us against
        // 21.7 with a group's 4 added in fp32 first, of 8192 bf16, 8 to a group, in 23.2 against 22.9)
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) { s += (double)(in[u] >> j & 1u ? a[u][j] - b[u][j] : 0.f); cnt += in[u] >> j & 1u; }
      });
    acc[0] = s; acc[1] = (double)cnt;
  }
  template <int NT>
  __device__ __forceinline__ void grad(long row, long i0, long i1, int tid, float f) const {
    const long len = pc.len(row);
    unsigned in[2];
    pcm_groups<Dt, NT, 2>(i0, i1, tid,
      [&](int u, long i, long left) { in[u] = left >= Dt::VEC ? pc.bits_inside<Dt::VEC>(row, i, len) : pc.bits_end<Dt::VEC>(row, i, len); },
      [&](int u, long i, long left) {
        float g[Dt::VEC];
#pragma unroll
        for (int j = 0; j < Dt::VEC; j++) g[j] = in[u] >> j & 1u ? f : 0.f;
        pcm_st_group<Dt>(dlogp + row * ld_d + i, left, g);
      });
  }
  __device__ __forceinline__ double share(const double (&s)[SUMS]) const { return mean_reduce ? 1.0 / fmax(s[1], 1.0) : 1.0; }
  // Rounded before a pair's other log ratio is subtracted from it: contracted with that subtraction, one row's product would be exact and the other's not,
  // and of equal rows the rounding error would be left -- 1e22 where the sums hold the lowest number of fp32.
  __device__ __forceinline__ double rho(long row, const double (&s)[SUMS]) const {
#pragma clang fp contract(off)
    return s[0] * share(s);
  }
  __device__ __forceinline__ double factor(long row, const double (&s)[SUMS]) const { return share(s); }
  bool wants_grad() const { return dlogp != nullptr; }
};
// Two launches: (1) partial sums of every (row, chunk); (2) the gradient, where each team adds up the partial sums of its pair again instead of
// waiting for a launch that does it once -- at most 2 x 64 numbers out of L2 -- and the first workgroup forms the mean loss.  The gradient has to wait for
// both rows of its pair, so t and p are read twice: 64 pairs of 262144 fp32, (1) 402 MB in 60 us (6.7 TB/s), (2) 268 MB in and 134 out in 64 us
// (6.3 TB/s).  Launching groups of pairs whose rows stay in the 256 MB cache for (2) was slower, 143 us and more: every launch ends with workgroups
// that wait for the last loads.
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
// what the threads first, first + step, ... of the pairs add to the loss; their log ratios are written on the way
template <typename R>
__device__ __forceinline__ double pair_losses(const R& rows_, const double* part, const PairLoss& pl, float* log_ratio, long pairs, int chunks, long first, long step) {
  double acc = 0.0;
  for (long p = first; p < pairs; p += step) {
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
  return acc;
}
template <typename R, int TEAM>
__global__ __launch_bounds__(256) void pair_grad_kernel(R rows_, const double* part, PairLoss pl, double gscale, float* loss, float* log_ratio, long pairs,
                                                        long n, int chunks, long len) {
  __shared__ double red[4];
  if (blockIdx.x == 0) {
    if (!loss) return;
    const double acc = pcm_block_sum<256>(pair_losses(rows_, part, pl, log_ratio, pairs, chunks, threadIdx.x, 256), red);
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
// more pairs than one workgroup forms the loss of beside the gradient: two launches of their own.  2048 pairs x 50: 18.9 us against 24.3 apart, 4096 x 50:
// 23.5 (alone 46) against 24.7 (40), 16384 x 8: 76 against 35
#define PAIR_LOSS_ONE 2048
#define PAIR_LOSS_PARTS 256
template <typename R>
__global__ __launch_bounds__(256) void pair_loss_kernel(R rows_, const double* part, PairLoss pl, float* log_ratio, long pairs, int chunks, double* loss_part) {
  __shared__ double red[4];
  const double acc = pcm_block_sum<256>(pair_losses(rows_, part, pl, log_ratio, pairs, chunks, (long)blockIdx.x * 256 + threadIdx.x, (long)gridDim.x * 256), red);
  if (threadIdx.x == 0) loss_part[blockIdx.x] = acc;
}
__global__ __launch_bounds__(256) void pair_loss_finish_kernel(const double* loss_part, int n, long pairs, float* loss) {
  __shared__ double red[4];
  const double acc = pcm_block_sum<256>((int)threadIdx.x < n ? loss_part[threadIdx.x] : 0.0, red);
  if (threadIdx.x == 0) loss[0] = (float)(acc / (double)pairs);
}
// few elements: one workgroup takes all pairs in one launch -- a row to a wave, or to half of the waves where rows are long.  At the limit (one pair of
// 16384 fp32) 14.2 us among others against 18.8 in two launches, alone 30.7 against 31.3; at twice as much alone 38 against 33.  The host's 4 us a launch
// decide: in a replayed graph, where they are gone, one pair of 4096 takes 5.8 us either way, of 16384 10.0 against 7.4, 16 pairs of 1000 14.4 against 7.2; and 8
// masked pairs of 2048 log-probabilities take 23.4 eager against 20.2
#define PAIR_SMALL_ELEMENTS 32768L
#define PAIR_SMALL_ROWS 128
template <typename R>
__global__ __launch_bounds__(1024) void pair_small_kernel(R rows_, PairLoss pl, double gscale, float* loss, float* log_ratio, int pairs, int n, int want_grad) {
  __shared__ double red[16 * R::SUMS], rho[PAIR_SMALL_ROWS], factor[PAIR_SMALL_ROWS], slope[PAIR_SMALL_ROWS / 2];
  const int rows = 2 * pairs, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const bool by_wave = n <= 1024;
  const int team = by_wave ? wave : wave >> 3, teams = by_wave ? 16 : 2, half = threadIdx.x & 511;
  double s[R::SUMS];
  for (int row = team; row < rows; row += teams) {      // (rows is even: both halves of the workgroup take as many)
    if (by_wave) rows_.template sums<64>(row, 0, n, lane, s);
    else rows_.template sums<512>(row, 0, n, half, s);
#pragma unroll
    for (int a = 0; a < R::SUMS; a++) s[a] = pcm_lane_sum(s[a]);
    if (!by_wave) {
      __syncthreads();
      if (lane == 0)
#pragma unroll
        for (int a = 0; a < R::SUMS; a++) red[wave * R::SUMS + a] = s[a];
      __syncthreads();
#pragma unroll
      for (int a = 0; a < R::SUMS; a++) {
        s[a] = red[team * 8 * R::SUMS + a];
#pragma unroll
        for (int w = 1; w < 8; w++) s[a] += red[(team * 8 + w) * R::SUMS + a];
      }
    }
    if (by_wave ? lane == 0 : half == 0) {
      rho[row] = rows_.rho(row, s); factor[row] = rows_.factor(row, s);
      log_ratio[row] = (float)rho[row];
    }
  }
  __syncthreads();
  double l = 0.0;
  if ((int)threadIdx.x < pairs) pair_loss(pl, rho[threadIdx.x] - rho[pairs + threadIdx.x], &l, &slope[threadIdx.x]);
  l = pcm_block_sum<1024>(l, red);
  if (threadIdx.x == 0) loss[0] = (float)(l / (double)pairs);
  if (!want_grad) return;
  for (int row = team; row < rows; row += teams) {
    const float f = (float)((row < pairs ? slope[row] : -slope[row - pairs]) * factor[row] * gscale / (double)pairs);
    if (by_wave) rows_.template grad<64>(row, 0, n, lane, f);
    else rows_.template grad<512>(row, 0, n, half, f);
  }
}
static bool pair_small(long rows, long n) { return rows <= PAIR_SMALL_ROWS && rows * n <= PAIR_SMALL_ELEMENTS; }
// bytes of the partial sums
static size_t pair_ws_bytes(long rows, long n, int sums) {      // (the 16-bit formats cut into no more chunks than fp32)
  if (pair_small(rows, n)) return 0;
  const RowCut c = row_cut(rows, n, 4);
  return ((size_t)rows * c.chunks * sums + (rows > 2 * PAIR_LOSS_ONE ? PAIR_LOSS_PARTS : 0)) * sizeof(double);
}
template <typename R>
static void pair_launch(const R& r, double* part, const PairLoss& pl, double gscale, float* loss, float* log_ratio, long pairs, long n, void* stream) {
  const long rows = 2 * pairs;
  if (pair_small(rows, n)) {
    PCM_LAUNCH(pair_small_kernel<R>, dim3(1), dim3(1024), 0, stream, r, pl, gscale, loss, log_ratio, (int)pairs, (int)n, r.wants_grad() ? 1 : 0);
    return;
  }
  const RowCut c = row_cut(rows, n, R::Dt::VEC);
  const bool apart = pairs > PAIR_LOSS_ONE;
  const unsigned nb = row_cut_blocks(c, rows), ng = r.wants_grad() ? nb + 1 : (apart ? 0 : 1);      // workgroups of the gradient, and the one of the loss
  float* at_once = apart ? nullptr : loss;
  if (c.team == 64) {
    PCM_LAUNCH((pair_sums_kernel<R, 64>), dim3(nb), dim3(256), 0, stream, r, part, rows, n, c.chunks, c.len);
    if (ng) PCM_LAUNCH((pair_grad_kernel<R, 64>), dim3(ng), dim3(256), 0, stream, r, (const double*)part, pl, gscale, at_once, log_ratio, pairs, n, c.chunks, c.len);
  } else {
    PCM_LAUNCH((pair_sums_kernel<R, 256>), dim3(nb), dim3(256), 0, stream, r, part, rows, n, c.chunks, c.len);
    if (ng) PCM_LAUNCH((pair_grad_kernel<R, 256>), dim3(ng), dim3(256), 0, stream, r, (const double*)part, pl, gscale, at_once, log_ratio, pairs, n, c.chunks, c.len);
  }
  if (apart) {
    double* loss_part = part + rows * c.chunks * R::SUMS;
    const long want = (pairs + 255) / 256;
    const int nl = (int)(want < PCM_GRID_CAP(PAIR_LOSS_PARTS) ? want : PCM_GRID_CAP(PAIR_LOSS_PARTS));
    PCM_LAUNCH(pair_loss_kernel<R>, dim3(nl), dim3(256), 0, stream, r, (const double*)part, pl, log_ratio, pairs, c.chunks, loss_part);
    PCM_LAUNCH(pair_loss_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)loss_part, nl, pairs, loss);
  }
}

// ---- clipped policy loss with a KL term ----
// e^x to about two steps: 2^t with t = x log2 e, the product's rounding error e carried along as the factor 1 + e ln 2 (v_exp_f32 alone would be off by
// |x| half steps).  Half the instructions of expf; results below 2^-126 come out as 0: a ratio or an exp(d) that small adds less than the last digit of
// anything it stands beside.
__device__ __forceinline__ float exp_of(float x) {
  const float hi = 1.44269502162933349609375f, lo = 1.92596299112661746887e-8f;      // log2 e in two fp32 numbers
  const float t = x * hi, e = fmaf(x, lo, fmaf(x, hi, -t)), r = PCM_EXP2F(t);
  return fabsf(x) < 100.0f ? r * fmaf(e, 0.693147182464599609375f, 1.0f) : r;        // (beyond, r is 0 or infinite, or x is no number)
}
// the KL estimate exp(d) - d - 1 and its rise exp(d) - 1.  Below 1/2 the estimate is the power series d^2 (1/2! + d/3! + ... + d^7/9!) -- the difference itself
// would leave nothing of a small d -- whose first term left out is 2 / (10! 2^8) of the sum at the most, and the rise is d more.  Above, the rise is
// exp(d) - 1 itself: made from the estimate it would lose its digits to d, and all of them where the reference is far below the policy.  The estimate is
// then the difference in fp32, which costs no second exponential: the four half steps of exp(d) are 44 of the estimate at d = 1/2, 23 at -1/2, 15 at 1 and
// under 5 from 4 on.  (d = inf: the estimate is infinite, not inf - inf.)
__device__ __forceinline__ void kl_term(float d, float* kl, float* rise) {
  if (fabsf(d) < 0.5f) {
    float s = fmaf(d, 1.0f / 362880.0f, 1.0f / 40320.0f);
    s = fmaf(d, s, 1.0f / 5040.0f); s = fmaf(d, s, 1.0f / 720.0f); s = fmaf(d, s, 1.0f / 120.0f); s = fmaf(d, s, 1.0f / 24.0f);
    s = fmaf(d, s, 1.0f / 6.0f); s = fmaf(d, s, 0.5f);
    *kl = d * d * s;
    *rise = d + *kl;
  } else {
    *rise = exp_of(d) - 1.0f;
    *kl = *rise - fminf(d, 3.4028234663852886e38f);
  }
}
// log(1 + hi) and log(1 - lo) in fp64 and rounded to fp32, 1 + hi, 1 - lo, KL coefficient
struct PolicyConst { double log_over, log_under; float log_over_f, log_under_f, over, under, kl; };
// what a place needs of its advantage a: a bound holds r = e^x where a's sign times x is beyond `border`, and the objective is then `held`
struct PolicySide {
  float a, border, held;
  bool neg, zero;
  __device__ __forceinline__ PolicySide() {}
  __device__ __forceinline__ PolicySide(const PolicyConst& c, float adv) {
    a = adv; neg = adv < 0.f; zero = adv == 0.f;
    border = zero ? __uint_as_float(0x7f800000u) : (neg ? -c.log_under_f : c.log_over_f);
    held = -adv * (neg ? c.under : c.over);
  }
};
// one place: the clipped objective, the KL estimate, the derivative of objective + kl * KL by logp.  The side of the border that logp - old_logp is on is that
// of the exact difference: the rounded one decides unless it falls on the rounded border itself, and then fp64, where the difference of two fp32
// numbers this close is exact, does.
template <bool KL>
__device__ __forceinline__ void policy_place(const PolicyConst& c, const PolicySide& s, float lp, float old, float ref, float* obj, float* kl, float* slope,
                                             bool* held) {
  const float x = lp - old, y = s.neg ? -x : x;
  bool beyond = y > s.border;
  if (y == s.border) {
    const double e = (double)lp - (double)old;
    beyond = !s.zero && (s.neg ? e < c.log_under : e > c.log_over);
  }
  // an advantage of zero adds nothing, also where exp leaves fp32 or either policy rules the place out; a NaN stays one
  const float ar = s.zero ? (x == x ? 0.f : x) : s.a * exp_of(x);
  *held = beyond;
  *obj = beyond ? s.held : -ar;
  *slope = beyond ? 0.f : -ar;
  if constexpr (KL) {
    float rise;
    kl_term(ref - lp, kl, &rise);
    *slope -= c.kl * (c.kl != 0.f ? rise : 0.f);      // (coefficient 0: the KL is only watched, no 0 times infinity enters the gradient)
  }
}
#define POLICY_GROUP 4      /* places of a thread's group in every format (8 need 98 registers: half the waves, 59 us against 50 at 2048 x 8192) */
template <typename Dt_>
struct PolicyRows {
  typedef Dt_ Dt;
  typedef typename Dt::raw raw;
  const raw *logp, *old, *ref;      // old: logp itself where there is none (r = 1)
  long ld_logp, ld_old, ld_ref;
  const float* adv;
  long ld_adv;                      // 0: one per row
  Places pc;
  PolicyConst con;
  raw* dlogp;                       // NULL: no gradient
  long ld_d;
  int rows, gpr;                    // groups of a row
  double gscale;
};
// what a launch adds up: objective, KL (both weighted), places held by the clip, places
enum { POLICY_OBJ, POLICY_KL, POLICY_HELD, POLICY_COUNT, POLICY_SUMS };
struct PolicySums {
  double obj, kl;
  int held, count;
  __device__ __forceinline__ PolicySums() : obj(0.0), kl(0.0), held(0), count(0) {}
  __device__ __forceinline__ void to(double (&s)[POLICY_SUMS]) const { s[POLICY_OBJ] = obj; s[POLICY_KL] = kl; s[POLICY_HELD] = (double)held; s[POLICY_COUNT] = (double)count; }
};
// what a row's places share: length, weight in the loss, weight in the gradient, advantage (where it is one per row)
struct PolicyRow { int len; double w; float wg; PolicySide side; };
template <typename Dt>
__device__ __forceinline__ PolicyRow policy_row(const PolicyRows<Dt>& a, int row, int len, double w) {
  PolicyRow r;
  r.len = len; r.w = w; r.wg = (float)(w * a.gscale);
  if (!a.ld_adv) r.side = PolicySide(a.con, a.adv[row]);
  return r;
}
// The group of places c .. of a row.  A row's last group is moved back so that it ends with the row: every access is a whole one and no load stands in a branch
// of its own, which would make the wave wait for one load before it issues the next; the places it shares with the group before are left out.  NARROW:
// rows shorter than a group, read place by place (the last one in place of those outside).  A group in which nothing counts reads nothing.
template <bool KL, bool NARROW, typename Dt>
__device__ __forceinline__ void policy_group(const PolicyRows<Dt>& a, int row, int c, const PolicyRow& r, PolicySums& s) {
  constexpr int V = POLICY_GROUP;
  const int cols = (int)a.pc.cols, c0 = NARROW ? 0 : (c + V <= cols ? c : cols - V), skip = c - c0;
  const unsigned in = (NARROW ? a.pc.template bits_end<V>(row, c0, r.len) : a.pc.template bits_inside<V>(row, c0, r.len)) >> skip << skip;
  float out[V];
#pragma unroll
  for (int j = 0; j < V; j++) out[j] = 0.f;
  if (in) {
    float lp[V], old[V], ref[V], adv[V];
    const typename Dt::raw *pl = a.logp + at(row, a.ld_logp, c0), *po = a.old + at(row, a.ld_old, c0), *pr = KL ? a.ref + at(row, a.ld_ref, c0) : nullptr;
    if constexpr (NARROW) {
#pragma unroll
      for (int j = 0; j < V; j++) {
        const int k = j < cols ? j : cols - 1;
        lp[j] = Dt::ld(pl[k]); old[j] = Dt::ld(po[k]);
        if (KL) ref[j] = Dt::ld(pr[k]);
      }
    } else {
      pcm_ld_group<Dt, true>(pl, lp);
      pcm_ld_group<Dt, true>(po, old);
      if (KL) pcm_ld_group<Dt, true>(pr, ref);
    }
    PolicySide side = r.side;
    if (a.ld_adv) {
      const float* pa = a.adv + at(row, a.ld_adv, c0);
      if constexpr (NARROW) {
#pragma unroll
        for (int j = 0; j < V; j++) adv[j] = pa[j < cols ? j : cols - 1];
      } else {
        pcm_ld_group<DtF32, true>(pa, adv);
      }
    }
    float so = 0.f, sk = 0.f;
#pragma unroll
    for (int j = 0; j < V; j++) {
      float obj, kl = 0.f, slope;
      bool held;
      if (a.ld_adv) side = PolicySide(a.con, adv[j]);
      policy_place<KL>(a.con, side, lp[j], old[j], KL ? ref[j] : 0.f, &obj, &kl, &slope, &held);
      const bool counts = in >> j & 1u;
      so += counts ? obj : 0.f;
      if (KL) sk += counts ? kl : 0.f;
      s.held += counts && held ? 1 : 0;
      out[j] = counts ? slope * r.wg : 0.f;
    }
    s.obj += r.w * (double)so;
    if (KL) s.kl += r.w * (double)sk;
    s.count += __builtin_popcount(in);
  }
  if (a.dlogp) {
    typename Dt::raw* pd = a.dlogp + at(row, a.ld_d, c0);
    if (!NARROW && skip == 0) pcm_st_group<Dt>(pd, V, out);
    else
#pragma unroll
      for (int j = 0; j < V; j++)
        if (j >= skip && c0 + j < cols) pd[j] = Dt::st(out[j]);
  }
}
// Groups numbered row by row; the thread takes g, g + NT, ... below end.  weight(row): the row's weight in the loss, asked for when the row changes
template <bool KL, bool NARROW, int NT, typename Dt, typename W>
__device__ __forceinline__ void policy_groups(const PolicyRows<Dt>& a, long g, long end, W&& weight, PolicySums& s) {
  if (g >= end) return;
  const int drow = NT / a.gpr, dcol = NT - drow * a.gpr;
  int row = (int)(g / a.gpr), col = (int)(g - (long)row * a.gpr), last = -1;
  PolicyRow r;
  for (; g < end; g += NT) {
    if (row != last) { last = row; r = policy_row(a, row, (int)a.pc.len(row), weight(row)); }
    policy_group<KL, NARROW>(a, row, col * POLICY_GROUP, r, s);
    col += dcol; row += drow;
    if (col >= a.gpr) { col -= a.gpr; row++; }
  }
}
// how many places count, where the launch has to find out, as partial sums over groups of 16 places
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
// weights of rows, 1 / (places * rows): a wave to a row, or a workgroup where there are few long ones
template <int TEAM>
__global__ __launch_bounds__(TEAM == 64 ? 256 : TEAM) void policy_weights_kernel(Places pc, long rows, double* weight) {
  __shared__ int red[16];
  const long row = TEAM == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= rows) return;
  const int tid = TEAM == 64 ? threadIdx.x & 63 : threadIdx.x;
  const long len = pc.len(row);
  int n = 0;
  if (pc.mask) {
    for (long c = tid * 16L; c < len; c += TEAM * 16L) n += __builtin_popcount(pc.bits<16>(row, c, len));
    n = pcm_block_sum<TEAM>(n, red);
  } else n = (int)len;
  if (tid == 0) weight[row] = 1.0 / (fmax((double)n, 1.0) * (double)rows);
}
// sum of the lengths over a workgroup's threads, the loads of a thread independent of one another
template <typename L>
__device__ __forceinline__ long sum_lengths(const L* lengths, long rows, long cols, int nt) {
  long t = 0;
  for (long r = threadIdx.x; r < rows; r += 8L * nt) {
    long v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = r + (long)u * nt < rows ? (long)lengths[r + (long)u * nt] : 0;
#pragma unroll
    for (int u = 0; u < 8; u++) t += v[u] < 0 ? 0 : (v[u] > cols ? cols : v[u]);
  }
  return t;
}
// where the weights come from: one for all places -- 1 / places, the number of places being known (>= 0), the sum of `part`, or that of the lengths; or one
// for each row
struct PolicyWeight { double places; const double* part; int nparts; const double* per_row; };
template <int NT>
__device__ __forceinline__ double policy_weight(const Places& pc, int rows, const PolicyWeight& pw, double* red) {
  double n = pw.places;
  if (pw.part) {
    n = 0.0;
    for (int i = threadIdx.x; i < pw.nparts; i += NT) n += pw.part[i];
    n = pcm_block_sum<NT>(n, red);
  } else if (n < 0.0) {
    n = (double)(pc.i64 ? sum_lengths((const int64_t*)pc.lengths, rows, pc.cols, NT) : sum_lengths((const int32_t*)pc.lengths, rows, pc.cols, NT));
    n = pcm_block_sum<NT>(n, red);
  }
  return 1.0 / fmax(n, 1.0);
}
template <bool KL, bool NARROW, int NT, typename Dt>
__device__ __forceinline__ void policy_part(const PolicyRows<Dt>& a, const PolicyWeight& pw, long g, long end, double* red, double (&sum)[POLICY_SUMS]) {
  PolicySums s;
  const double w = pw.per_row ? 0.0 : policy_weight<NT>(a.pc, a.rows, pw, red);
  policy_groups<KL, NARROW, NT>(a, g, end, [&](int row) { return pw.per_row ? pw.per_row[row] : w; }, s);
  s.to(sum);
  pcm_block_sums<NT>(sum, red);
}
__device__ __forceinline__ void policy_result(const double (&s)[POLICY_SUMS], double kl, float* loss, float* stats) {
  loss[0] = (float)(kl != 0.0 ? s[POLICY_OBJ] + kl * s[POLICY_KL] : s[POLICY_OBJ]);
  stats[0] = (float)s[POLICY_OBJ]; stats[1] = (float)s[POLICY_KL]; stats[2] = (float)(s[POLICY_HELD] / fmax(s[POLICY_COUNT], 1.0)); stats[3] = (float)s[POLICY_COUNT];
}
__device__ __forceinline__ void policy_store(const double (&s)[POLICY_SUMS], double* part) {
  if (threadIdx.x == 0)
#pragma unroll
    for (int k = 0; k < POLICY_SUMS; k++) part[(long)blockIdx.x * POLICY_SUMS + k] = s[k];
}
// (256, 8): 8 waves to a SIMD, so that all 2048 workgroups are resident at once; a workgroup takes consecutive groups (a strided grid reads 15 % slower).
// 2048 x 8192 fp32 with old and reference log-probabilities: 268 MB in 50 us; with ragged rows, 194 MB, 43 us (without its arithmetic 13 % less).
template <bool KL, bool NARROW, typename Dt>
__global__ __launch_bounds__(256, 8) void policy_main_kernel(PolicyRows<Dt> a, PolicyWeight pw, double* part) {
  __shared__ double red[4 * POLICY_SUMS];
  const long total = (long)a.rows * a.gpr, per = (total + gridDim.x - 1) / gridDim.x, g0 = blockIdx.x * per;
  double s[POLICY_SUMS];
  policy_part<KL, NARROW, 256>(a, pw, g0 + threadIdx.x, g0 + per < total ? g0 + per : total, red, s);
  policy_store(s, part);
}
// the mean of row means, a row to a workgroup at a time: it counts the row's places first, and no launch has to do that before
template <bool KL, typename Dt>
__global__ __launch_bounds__(256, 8) void policy_row_kernel(PolicyRows<Dt> a, double* part) {
  __shared__ double red[4 * POLICY_SUMS];
  PolicySums t;
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int len = (int)a.pc.len(row);
    int n = len;
    if (a.pc.mask) {
      n = 0;
      for (int c = threadIdx.x * 16; c < len; c += 256 * 16) n += __builtin_popcount(a.pc.template bits<16>(row, c, len));
      n = pcm_block_sum<256>(n, (int*)red);
    }
    const PolicyRow r = policy_row(a, row, len, 1.0 / (fmax((double)n, 1.0) * (double)a.rows));
    for (int g = threadIdx.x; g < a.gpr; g += 256) policy_group<KL, false>(a, row, g * POLICY_GROUP, r, t);
  }
  double s[POLICY_SUMS];
  t.to(s);
  pcm_block_sums<256>(s, red);
  policy_store(s, part);
}
__global__ __launch_bounds__(256) void policy_finish_kernel(const double* part, int nparts, double kl, float* loss, float* stats) {
  __shared__ double red[4 * POLICY_SUMS];
  double s[POLICY_SUMS] = {0.0, 0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < nparts; i += 256)
#pragma unroll
    for (int k = 0; k < POLICY_SUMS; k++) s[k] += part[i * POLICY_SUMS + k];
  pcm_block_sums<256>(s, red);
  if (threadIdx.x == 0) policy_result(s, kl, loss, stats);
}
// few places: one workgroup counts, forms loss and gradient, and adds up, in one launch.  At the limit (64 x 256 bf16, masked) 17.2 us among others against
// 23.9 in three launches, alone 39 against 36; at twice as much 22.4 against 24.1 and 47 against 36.  In a replayed graph, without the host's share, 8 x 4 takes 6.9
// against 9.5, 64 x 128 9.5 against 10.2, 64 x 256 15.0 against 10.3
#define POLICY_SMALL_PLACES 16384
#define POLICY_SMALL_ROWS 2048
template <bool KL, bool NARROW, typename Dt>
__global__ __launch_bounds__(1024) void policy_small_kernel(PolicyRows<Dt> a, int reduce, double kl, float* loss, float* stats) {
  __shared__ double red[16 * POLICY_SUMS];
  __shared__ double weight[POLICY_SMALL_ROWS];
  PolicyWeight pw = {1.0, nullptr, 0, nullptr};
  if (reduce == PCM_POLICY_TOKEN) {
    if (a.pc.mask) pw.places = pcm_block_sum<1024>((double)count_groups(a.pc, a.rows, threadIdx.x, 1024), red);
    else pw.places = a.pc.lengths ? -1.0 : (double)a.rows * (double)a.pc.cols;
  } else if (reduce == PCM_POLICY_ROW) {
    for (int row = threadIdx.x >> 6; row < a.rows; row += 16) {
      const int len = (int)a.pc.len(row), lane = threadIdx.x & 63;
      int n = len;
      if (a.pc.mask) {
        n = 0;
        for (int c = lane * 16; c < len; c += 64 * 16) n += __builtin_popcount(a.pc.template bits<16>(row, c, len));
        n = pcm_lane_sum(n);
      }
      if (lane == 0) weight[row] = 1.0 / (fmax((double)n, 1.0) * (double)a.rows);
    }
    __syncthreads();
    pw.per_row = weight;
  }
  double s[POLICY_SUMS];
  policy_part<KL, NARROW, 1024>(a, pw, threadIdx.x, (long)a.rows * a.gpr, red, s);
  if (threadIdx.x == 0) policy_result(s, kl, loss, stats);
}

// ---- entry points ----
#define AL_MAX_LD 4294967296L
#define AL_MAX_ROWS 16777216L
// a launch has fewer than 2^32 threads: long rows take a workgroup of 256 each (several only where rows are few), and the pairs' loss one more
static bool rows_ok(long rows, long n) { return rows > 0 && rows <= AL_MAX_ROWS && (n <= 1024 || rows <= AL_MAX_ROWS - 2); }
// the forward pass takes a row to a workgroup of 1024 where rows are too few for one chunk each but short enough: one launch instead of two.  16 rows of
// 16384: 4.2 us against 3.1 + 2.5 and 4 us less host time; one row of 65536 among others 12 us against 16, of 131072 alone 28 against 26
static RowCut transition_cut(long rows, long n, int vec) {
  RowCut c = row_cut(rows, n, vec);
  if (c.chunks > 1 && n <= ROW_TEAM_MAX) { c.team = 1024; c.chunks = 1; c.len = n; }
  return c;
}
extern "C" size_t pcm_transition_logprob_workspace_bytes(long rows, long n) {
  if (rows <= 0 || n <= 0) return 0;
  const RowCut c = transition_cut(rows, n, 4);      // (the 16-bit formats cut into no more chunks than fp32)
  return c.chunks > 1 ? (size_t)rows * c.chunks * sizeof(double) : 0;
}
extern "C" int pcm_transition_logprob(const void* x, const void* mean, const float* std, int dtype, int mean_reduce, float* logp, long rows, long n,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  PCM_CHECK(x && mean && std && logp && pcm_dt_ok(dtype) && n > 0 && rows_ok(rows, n), PCM_EINVAL, "pcm_transition_logprob: null/empty, too many rows or unknown format");
  const size_t need = pcm_transition_logprob_workspace_bytes(rows, n);
  PCM_CHECK(need == 0 || (workspace && ((uintptr_t)workspace % 8) == 0 && workspace_bytes >= need), PCM_EINVAL,
            "pcm_transition_logprob: workspace too small or not 8-byte aligned");
  pcm_with_dtype(dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    const RowCut c = transition_cut(rows, n, Dt::VEC);
    const dim3 grid(c.team == 1024 ? (unsigned)rows : row_cut_blocks(c, rows));
    double* part = (double*)workspace;
    if (c.team == 64) PCM_LAUNCH((transition_fwd_kernel<Dt, 64>), grid, dim3(256), 0, stream, (cp)x, (cp)mean, std, logp, part, rows, n, c.chunks, c.len, mean_reduce);
    else if (c.team == 256) PCM_LAUNCH((transition_fwd_kernel<Dt, 256>), grid, dim3(256), 0, stream, (cp)x, (cp)mean, std, logp, part, rows, n, c.chunks, c.len, mean_reduce);
    else PCM_LAUNCH((transition_fwd_kernel<Dt, 1024>), grid, dim3(1024), 0, stream, (cp)x, (cp)mean, std, logp, part, rows, n, c.chunks, c.len, mean_reduce);
    if (c.chunks > 1)
      PCM_LAUNCH(transition_finish_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, (const double*)workspace, std, logp, rows, n, c.chunks, mean_reduce);
  });
  return pcm_post_launch("pcm_transition_logprob");
}
extern "C" int pcm_transition_logprob_bwd(const void* x, const void* mean, const float* std, const float* dlogp, int dtype, int mean_reduce, void* dmean,
                                          long rows, long n, void* stream) {
  PCM_CHECK(x && mean && std && dlogp && dmean && pcm_dt_ok(dtype) && n > 0 && rows_ok(rows, n), PCM_EINVAL,
            "pcm_transition_logprob_bwd: null/empty, too many rows or unknown format");
  pcm_with_dtype(dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    const RowCut c = row_cut(rows, n, Dt::VEC);
    const dim3 grid(row_cut_blocks(c, rows));
    typename Dt::raw* d = (typename Dt::raw*)dmean;
    if (c.team == 64) PCM_LAUNCH((transition_bwd_kernel<Dt, 64>), grid, dim3(256), 0, stream, (cp)x, (cp)mean, std, dlogp, d, rows, n, c.chunks, c.len, mean_reduce);
    else PCM_LAUNCH((transition_bwd_kernel<Dt, 256>), grid, dim3(256), 0, stream, (cp)x, (cp)mean, std, dlogp, d, rows, n, c.chunks, c.len, mean_reduce);
  });
  return pcm_post_launch("pcm_transition_logprob_bwd");
}

static int pair_args_ok(const char* who, int dtype, long pairs, long n, double beta, int kind, double eps) {
  PCM_CHECK(pcm_dt_ok(dtype), PCM_EINVAL, "%s: unknown element format %d", who, dtype);
  PCM_CHECK(pairs > 0 && pairs <= AL_MAX_ROWS && rows_ok(2 * pairs, n), PCM_EINVAL, "%s: number of pairs %ld", who, pairs);
  PCM_CHECK(beta > 0.0 && beta < 1e30, PCM_EINVAL, "%s: beta must be positive and finite", who);
  PCM_CHECK(kind == PCM_PAIR_SIGMOID || kind == PCM_PAIR_HINGE || kind == PCM_PAIR_SQUARE, PCM_EINVAL, "%s: unknown kind %d", who, kind);
  PCM_CHECK(eps >= 0.0 && eps < 0.5 && (eps == 0.0 || kind == PCM_PAIR_SIGMOID), PCM_EINVAL, "%s: label smoothing must be in [0, 0.5) and needs the sigmoid kind", who);
  return PCM_OK;
}
extern "C" size_t pcm_denoise_preference_loss_workspace_bytes(long pairs, long n) { return pairs > 0 && n > 0 ? pair_ws_bytes(2 * pairs, n, DenoiseRows<DtF32>::SUMS) : 0; }
extern "C" int pcm_denoise_preference_loss(const pcm_denoise_preference_args* a, void* stream) {
  PCM_CHECK(a && a->pred && a->ref && a->target && a->loss && a->log_ratio && a->n > 0, PCM_EINVAL, "pcm_denoise_preference_loss: null/empty");
  const int rc = pair_args_ok("pcm_denoise_preference_loss", a->dtype, a->pairs, a->n, a->beta, a->kind, a->label_smoothing);
  if (rc != PCM_OK) return rc;
  const size_t need = pcm_denoise_preference_loss_workspace_bytes(a->pairs, a->n);
  PCM_CHECK(need == 0 || (a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= need), PCM_EINVAL,
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
extern "C" size_t pcm_preference_loss_workspace_bytes(long pairs, long cols) { return pairs > 0 && cols > 0 ? pair_ws_bytes(2 * pairs, cols, TokenRows<DtF32>::SUMS) : 0; }
extern "C" int pcm_preference_loss(const pcm_preference_args* a, void* stream) {
  PCM_CHECK(a && a->logp && a->ref_logp && a->loss && a->log_ratio && a->cols > 0, PCM_EINVAL, "pcm_preference_loss: null/empty");
  const int rc = pair_args_ok("pcm_preference_loss", a->dtype, a->pairs, a->cols, a->beta, a->kind, a->label_smoothing);
  if (rc != PCM_OK) return rc;
  PCM_CHECK(a->ld_logp >= a->cols && a->ld_ref >= a->cols && (!a->mask || a->ld_mask >= a->cols) && (!a->dlogp || a->ld_dlogp >= a->cols), PCM_EINVAL,
            "pcm_preference_loss: row stride below the row length");
  PCM_CHECK(a->cols < AL_MAX_LD && a->ld_logp < AL_MAX_LD && a->ld_ref < AL_MAX_LD && a->ld_mask < AL_MAX_LD && a->ld_dlogp < AL_MAX_LD, PCM_EINVAL,
            "pcm_preference_loss: row stride of 2^32 elements or more");
  const size_t need = pcm_preference_loss_workspace_bytes(a->pairs, a->cols);
  PCM_CHECK(need == 0 || (a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= need), PCM_EINVAL,
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
// a workgroup to a row: rows long enough to keep it busy, and enough of them for the chip or none too long for one.  Masked fp32 with KL, us eager / replayed,
// by row against a launch for the weights and one over all groups: 2048 x 256 21.4 / 13.2 against 24.1 / 10.6, 2048 x 500 21.2 / 14.3 against 23.8 / 14.4, 512 x 520
// 21.4 / 9.3 against 24.2 / 11.4, 40 x 4096 21.4 / 11.5 against 24.1 / 10.4, 40 x 5000 21.4 / 14.1 against 24.1 / 10.7, 300 x 8192 24.2 / 24.9 against 25.1 / 21.2,
// 512 x 8192 26.2 / 26.5 against 25.5 / 25.9, 2048 x 8192 52.4 / 52.6 against 58.3 / 58.2
static bool policy_by_row(int reduce, long rows, long cols) { return reduce == PCM_POLICY_ROW && cols >= 512 && (rows >= 512 || cols <= 4096); }
#define POLICY_COUNT_PARTS 512
// partial counts, or weights of rows
static long policy_counts(long rows, int reduce) { return reduce == PCM_POLICY_ROW && rows > POLICY_COUNT_PARTS ? rows : POLICY_COUNT_PARTS; }
extern "C" size_t pcm_policy_loss_workspace_bytes(long rows, long cols, int reduce) {
  if (rows <= 0 || cols <= 0 || policy_small(rows, cols)) return 0;
  return (size_t)(policy_counts(rows, reduce) + POLICY_SUMS * 2048) * sizeof(double);
}
#define POLICY_LAUNCH(kernel, grid, block, ...)                                                                              \
  do {                                                                                                                       \
    if (a->cols < POLICY_GROUP) {                                                                                            \
      if (kl) PCM_LAUNCH((kernel<true, true, Dt>), grid, block, 0, stream, __VA_ARGS__);                                     \
      else PCM_LAUNCH((kernel<false, true, Dt>), grid, block, 0, stream, __VA_ARGS__);                                       \
    } else if (kl) PCM_LAUNCH((kernel<true, false, Dt>), grid, block, 0, stream, __VA_ARGS__);                               \
    else PCM_LAUNCH((kernel<false, false, Dt>), grid, block, 0, stream, __VA_ARGS__);                                        \
  } while (0)
extern "C" int pcm_policy_loss(const pcm_policy_args* a, void* stream) {
  PCM_CHECK(a && a->logp && a->advantages && a->loss && a->stats && a->rows > 0 && a->rows <= AL_MAX_ROWS && a->cols > 0, PCM_EINVAL, "pcm_policy_loss: null/empty or too many rows");
  PCM_CHECK(pcm_dt_ok(a->dtype), PCM_EINVAL, "pcm_policy_loss: unknown element format %d", a->dtype);
  PCM_CHECK(a->reduce == PCM_POLICY_TOKEN || a->reduce == PCM_POLICY_ROW || a->reduce == PCM_POLICY_SUM, PCM_EINVAL, "pcm_policy_loss: unknown reduce %d", a->reduce);
  PCM_CHECK(a->clip_low >= 0.0 && a->clip_low < 1.0 && a->clip_high >= 0.0, PCM_EINVAL, "pcm_policy_loss: clip_low must be in [0, 1), clip_high >= 0");
  PCM_CHECK(a->kl_coef == 0.0 || a->ref_logp, PCM_EINVAL, "pcm_policy_loss: a KL term needs the reference log-probabilities");
  PCM_CHECK(a->ld_logp >= a->cols && (!a->old_logp || a->ld_old >= a->cols) && (!a->ref_logp || a->ld_ref >= a->cols) && (a->adv_per_row || a->ld_adv >= a->cols) &&
                (!a->mask || a->ld_mask >= a->cols) && (!a->dlogp || a->ld_dlogp >= a->cols), PCM_EINVAL, "pcm_policy_loss: row stride below the row length");
  PCM_CHECK(a->cols < 2147483648L - 65536 && a->ld_logp < AL_MAX_LD && a->ld_old < AL_MAX_LD && a->ld_ref < AL_MAX_LD && a->ld_adv < AL_MAX_LD && a->ld_mask < AL_MAX_LD &&
                a->ld_dlogp < AL_MAX_LD, PCM_EINVAL, "pcm_policy_loss: row stride of 2^32 elements or more");
  const size_t need = pcm_policy_loss_workspace_bytes(a->rows, a->cols, a->reduce);
  PCM_CHECK(need == 0 || (a->workspace && ((uintptr_t)a->workspace % 8) == 0 && a->workspace_bytes >= need), PCM_EINVAL,
            "pcm_policy_loss: workspace too small or not 8-byte aligned");
  const Places pc = {a->mask, a->ld_mask, a->lengths, a->lengths_i64, a->cols};
  const PolicyConst con = {log1p(a->clip_high), log1p(-a->clip_low), (float)log1p(a->clip_high), (float)log1p(-a->clip_low), (float)(1.0 + a->clip_high), (float)(1.0 - a->clip_low), (float)a->kl_coef};
  const long rows = a->rows;
  const int reduce = a->reduce == PCM_POLICY_ROW && rows == 1 ? PCM_POLICY_TOKEN : a->reduce;      // one row: its mean is the mean of all places
  const bool kl = a->ref_logp != nullptr, by_row = policy_by_row(reduce, rows, a->cols);
  const int gpr = (int)((a->cols + POLICY_GROUP - 1) / POLICY_GROUP);
  pcm_with_dtype(a->dtype, [&](auto dt) {
    typedef decltype(dt) Dt;
    typedef const typename Dt::raw* cp;
    const PolicyRows<Dt> r = {(cp)a->logp, (cp)(a->old_logp ? a->old_logp : a->logp), (cp)a->ref_logp, a->ld_logp, a->old_logp ? a->ld_old : a->ld_logp, a->ld_ref,
                              a->advantages, a->adv_per_row ? 0 : a->ld_adv, pc, con, (typename Dt::raw*)a->dlogp, a->ld_dlogp, (int)rows, gpr, a->grad_scale};
    if (need == 0) {
      POLICY_LAUNCH(policy_small_kernel, dim3(1), dim3(1024), r, reduce, a->kl_coef, a->loss, a->stats);
      return;
    }
    double *counts = (double*)a->workspace, *part = counts + policy_counts(rows, a->reduce);
    int nb = al_blocks(rows * gpr);
    if (by_row) {
      nb = (int)(rows < PCM_GRID_CAP(2048) ? rows : PCM_GRID_CAP(2048));
      if (kl) PCM_LAUNCH((policy_row_kernel<true, Dt>), dim3(nb), dim3(256), 0, stream, r, part);
      else PCM_LAUNCH((policy_row_kernel<false, Dt>), dim3(nb), dim3(256), 0, stream, r, part);
    } else {
      PolicyWeight pw = {1.0, nullptr, 0, nullptr};
      if (reduce == PCM_POLICY_TOKEN) {
        pw.places = a->mask || a->lengths ? -1.0 : (double)rows * (double)a->cols;
        if (a->mask || (a->lengths && rows > 4096)) {      // (each workgroup adds up 4096 lengths itself in 20.1 us against 23.1 with a launch, 16384 in 26.3 against 23.1)
          const long b = a->mask ? al_blocks(rows * ((a->cols + 15) / 16)) : al_blocks(rows);
          pw.nparts = (int)(b < POLICY_COUNT_PARTS ? b : POLICY_COUNT_PARTS);
          pw.part = counts;
          PCM_LAUNCH(policy_count_kernel, dim3(pw.nparts), dim3(256), 0, stream, pc, rows, counts);
        }
      } else if (reduce == PCM_POLICY_ROW) {
        pw.per_row = counts;
        // (us replayed, a wave to a row against a workgroup: 2048 x 511 15.2 against 22.6, 300 x 4096 15.1 against 15.0, 500 x 8192 26.2 against 24.2, 8 x 32768 16.6
        // against 10.3)
        if (a->cols <= 4096) PCM_LAUNCH(policy_weights_kernel<64>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, pc, rows, counts);
        else PCM_LAUNCH(policy_weights_kernel<1024>, dim3((unsigned)rows), dim3(1024), 0, stream, pc, rows, counts);
      }
      POLICY_LAUNCH(policy_main_kernel, dim3(nb), dim3(256), r, pw, part);
    }
    PCM_LAUNCH(policy_finish_kernel, dim3(1), dim3(256), 0, stream, (const double*)part, nb, a->kl_coef, a->loss, a->stats);
  });
  return pcm_post_launch("pcm_policy_loss");
}
