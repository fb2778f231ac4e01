// Distillation from a teacher's top logits, value and gradient (include/proxgrad_hip_rows.h: pg_distill_value_and_gradient).
//
// Per row, with z = x / T, e_v = exp(z_v - max z), S = sum e, q = e / S, the listed classes and their p:
//   L = sum_k p_k (log p_k - log q_k) + p_r (log p_r - log Q_r),     Q_r = sum of q outside the list
//   dL/dx_v = ((sum p + p_r) q_v - phat_v - [v not listed] p_r q_v / Q_r) / T
// so outside the list the gradient is ONE multiple of e_v, and only the listed classes (and the label) need more: every
// vector is written with the unlisted coefficient, then a few threads overwrite the listed entries.  Q_r is summed over
// the unlisted classes themselves (1 - sum of the listed q loses everything where the student agrees with the teacher),
// which a bitmap of the row in LDS makes possible; the bitmap also finds classes listed twice.
#include "pg_rows.h"

namespace pgrows {
namespace {

constexpr double LOG2E = 1.4426950408889634;
constexpr double LN2 = 0.6931471805599453;
constexpr int BIT0 = 8;         // bits in front of a chunk's first aligned vector (the head of a misaligned row: at most 7)
constexpr int STAT = 6;         // doubles per (row, part)
constexpr int MAX_PARTS = 64;   // one lane each when a row's parts are joined
constexpr int MAX_TOP = 1024;

struct DArgs {
  const void* x;
  void* g;
  const void *t, *idx, *lse, *w, *lab;
  int64_t ldx, ldg, ldt, ldi, row0, nrows;  // rows of this launch
  int V, K, tdt, ibits, lsedt, wdt, labbits;
  double invT, lam, lab_lam;
  int parts, pv;  // parts of a row, 16-byte vectors per part
  double *stat, *xk;
  double *partials, *acc, *out;
  unsigned* counter;
  void* value;
  int first, last;  // of the launches of this call
};

// ---- one row's scalars, from the statistics over the whole row ----------------------------------------------------
template <typename C>
struct RowScal {
  C M, cB, cR, c1;  // reference score; coefficients of e at listed / unlisted classes, of exp(x - M) for labels at T != 1
  C ql, qy;         // what a unit of teacher mass / the label takes off
  C ls, ls1;        // log sum exp((x - M) / T) and log sum exp(x - M)
  double pr, log_qr;
  bool empty;
};
template <typename C, bool TAIL, bool TWO>
__device__ __forceinline__ RowScal<C> row_scalars(const DArgs& a, double w, bool has_label, C M, C s_rest, C s_list, C s1, C n_listed,
                                                  double mass) {
  RowScal<C> r;
  const C S = TAIL ? s_rest + s_list : s_rest;
  r.empty = S == C(0);  // every score -inf (the largest score always contributes 1)
  r.M = M;
  r.ls = lg2(S) * (C)LN2;
  r.ql = (C)(a.lam * w * a.invT);
  r.qy = has_label ? (C)(a.lab_lam * w) : C(0);
  C rest = C(0);
  r.pr = 0.0;
  r.log_qr = 0.0;
  if constexpr (TAIL) {
    if ((int64_t)n_listed < a.V) {  // the list may hold every class: then nothing is outside it
      const double left = 1.0 - mass;
      r.pr = left > 0.0 ? left : (left == left ? 0.0 : left);
      const C qr = s_rest / S;
      r.log_qr = (double)(lg2(qr) * (C)LN2);
      rest = (r.pr > 0.0 && qr > C(0)) ? (C)r.pr / qr : C(0);
    }
  }
  const C total = (C)(mass + r.pr);
  r.cB = r.ql * total / S;
  r.cR = TAIL ? r.ql * (total - rest) / S : r.cB;
  r.c1 = C(0);
  r.ls1 = r.ls;
  if constexpr (TWO) {
    r.c1 = r.qy / s1;
    r.ls1 = lg2(s1) * (C)LN2;
  } else {  // labels at T = 1 share e
    r.cB += r.qy / S;
    r.cR += r.qy / S;
  }
  if (r.empty) {
    r.cB = r.cR = r.c1 = r.ql = r.qy = C(0);
    r.M = Lim<C>::lowest;
  }
  return r;
}

// probability of a listed entry: log p and p
template <typename C>
__device__ __forceinline__ void entry_p(const DArgs& a, int64_t row, int k, double norm, C& lp, C& p) {
  const double t = ld_real(a.t, a.tdt, row * a.ldt + k) * a.invT;
  lp = (C)(t == -INFINITY ? t : t - norm);  // (a list of -inf only has norm -inf)
  p = ex2(lp * (C)LOG2E);
}

// ---- a row's place in memory: head elements up to the first 16-byte boundary, whole vectors, tail -----------------
template <typename T>
struct Place {
  int h, nmain, hV;
  __device__ __forceinline__ Place(const T* xr, int V) {
    constexpr int N = Elem<T>::N;
    const int off = (int)((reinterpret_cast<uintptr_t>(xr) & 15u) / sizeof(T));
    h = off ? N - off : 0;
    h = h < V ? h : V;
    nmain = (V - h) / N;
    hV = h + nmain * N;
  }
};

template <typename T>
__device__ __forceinline__ unsigned listed_bits(const unsigned* bm, int vbit) {  // of the vector whose first bit is vbit (a multiple of N)
  constexpr int N = Elem<T>::N;
  return (bm[vbit >> 5] >> (vbit & 31)) & ((1u << N) - 1u);
}

// running maximum and sums of one thread
template <typename C, bool TAIL, bool TWO>
struct Run {
  C m = Lim<C>::lowest, s = C(0), sl = C(0), s1 = C(0), n = C(0);
  C c;  // log2(e) / T
  __device__ __forceinline__ void raise(C to) {
    const C d = m - to;
    const C f = ex2(d * c);
    s *= f;
    if constexpr (TAIL) sl *= f;
    if constexpr (TWO) s1 *= ex2(d * (C)LOG2E);
    m = to;
  }
  __device__ __forceinline__ void listed(C x) {  // a listed class (TAIL only)
    if (x > m) raise(x);
    sl += ex2((x - m) * c);
    n += C(1);
  }
  template <int N>
  __device__ __forceinline__ void add(const C (&f)[N], unsigned bits) {
    C vm = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) vm = fmx(vm, f[i]);
    if (vm > m) raise(vm);
    C e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = ex2((f[i] - m) * c);
    if constexpr (TAIL) {
      if (bits) {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = (bits >> i) & 1u ? C(0) : e[i];
      }
    }
#pragma unroll
    for (int o = 1; o < N; o *= 2)
#pragma unroll
      for (int i = 0; i < N; i += 2 * o) e[i] += e[i + o];
    s += e[0];
    if constexpr (TWO) {
      C t = C(0);
#pragma unroll
      for (int i = 0; i < N; ++i) t += ex2((f[i] - m) * (C)LOG2E);
      s1 += t;
    }
  }
  __device__ __forceinline__ void add1(C x, bool in_list) {
    if (x > m) raise(x);
    if (!(TAIL && in_list)) s += ex2((x - m) * c);
    if constexpr (TWO) s1 += ex2((x - m) * (C)LOG2E);
  }
};

// ---- the general form: a row in parts, two reads ------------------------------------------------------------------
// Any length, any number of rows.  First launch: the statistics of each part (and the listed scores, which an in-place
// gradient overwrites); second launch: every part joins its row's statistics and writes its piece of the gradient.
constexpr int PT = 256;

template <typename T, bool TAIL, bool TWO>
__global__ __launch_bounds__(PT) void distill_part_stats(DArgs a) {
  using C = typename Elem<T>::C;
  constexpr int N = Elem<T>::N;
  extern __shared__ unsigned bm[];
  __shared__ C sm[PT / 64][5];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = blockIdx.x % a.parts;
  const int64_t r = blockIdx.x / a.parts, row = a.row0 + r;
  if (a.w != nullptr && ld_real(a.w, a.wdt, row) == 0.0) return;
  const T* xr = (const T*)a.x + row * a.ldx;
  const Place<T> pl(xr, a.V);
  const int v0 = min(part * a.pv, pl.nmain), v1 = min(v0 + a.pv, pl.nmain);
  const bool lastp = part == a.parts - 1;
  const int e0 = part == 0 ? 0 : pl.h + v0 * N, e1 = lastp ? a.V : pl.h + v1 * N;
  const int bbase = pl.h + v0 * N - BIT0;  // element of bit 0
  const int words = (a.pv * N + BIT0 + N + 31) / 32;
  if constexpr (TAIL) {
    for (int i = tid; i < words; i += PT) bm[i] = 0;
    __syncthreads();
  }
  Run<C, TAIL, TWO> run;
  run.c = (C)(a.invT * LOG2E);
  bool bad = false;
  for (int k = tid; k < a.K; k += PT) {
    const int64_t id = ld_int(a.idx, a.ibits, row * a.ldi + k);
    bad |= id < -1 || id >= a.V;
    if (id >= e0 && id < e1) {
      const C x = up<T>(xr[id]);
      a.xk[r * (a.K + 1) + k] = (double)x;
      if constexpr (TAIL) {
        const int b = (int)id - bbase;
        const unsigned old = atomicOr(&bm[b >> 5], 1u << (b & 31));
        if (!((old >> (b & 31)) & 1u)) run.listed(x);
      }
    }
  }
  if (tid == 0 && a.lab != nullptr) {
    const int64_t y = ld_int(a.lab, a.labbits, row);
    bad |= y < -1 || y >= a.V;
    if (y >= e0 && y < e1) a.xk[r * (a.K + 1) + a.K] = (double)up<T>(xr[y]);
  }
  if constexpr (TAIL) __syncthreads();
  const T* xm = xr + pl.h;
  for (int v = v0 + tid; v < v1; v += PT) {
    C f[N];
    unpack<T>(ld16(xm + (int64_t)v * N), f);
    run.template add<N>(f, TAIL ? listed_bits<T>(bm, (v - v0) * N + BIT0) : 0u);
  }
  // (thread i: the i-th element of the head; thread PT - 1 - i: of the tail)
  const int ee = part == 0 && tid < pl.h ? tid : (lastp && pl.hV + (PT - 1 - tid) < a.V ? pl.hV + (PT - 1 - tid) : -1);
  if (ee >= 0) {
    const int b = ee - bbase;
    run.add1(up<T>(xr[ee]), TAIL && ((bm[b >> 5] >> (b & 31)) & 1u));
  }
  if (bad) run.s = (C)NAN;
  const C M = wave_max(run.m);
  const C f = ex2((run.m - M) * run.c);
  const C s = wave_sum(run.s * f), sl = TAIL ? wave_sum(run.sl * f) : C(0), n = TAIL ? wave_sum(run.n) : C(0);
  const C s1 = TWO ? wave_sum(run.s1 * ex2((run.m - M) * (C)LOG2E)) : C(0);
  if (lane == 0) sm[wave][0] = M, sm[wave][1] = s, sm[wave][2] = sl, sm[wave][3] = s1, sm[wave][4] = n;
  __syncthreads();
  if (tid == 0) {
    C m = sm[0][0];
    for (int i = 1; i < PT / 64; ++i) m = fmx(m, sm[i][0]);
    C o[4] = {};
    for (int i = 0; i < PT / 64; ++i) {
      const C g = ex2((sm[i][0] - m) * run.c);
      o[0] += sm[i][1] * g;
      o[1] += sm[i][2] * g;
      if constexpr (TWO) o[2] += sm[i][3] * ex2((sm[i][0] - m) * (C)LOG2E);
      o[3] += sm[i][4];
    }
    double* st = a.stat + (r * a.parts + part) * STAT;
    st[0] = (double)m;
    for (int i = 0; i < 4; ++i) st[1 + i] = (double)o[i];
  }
}

template <typename T, bool TAIL, bool TWO>
__global__ __launch_bounds__(PT) void distill_part_grad(DArgs a) {
  using C = typename Elem<T>::C;
  constexpr int N = Elem<T>::N;
  extern __shared__ unsigned bm[];
  __shared__ double smd[PT / 64][2];
  __shared__ int dup;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = blockIdx.x % a.parts;
  const int64_t r = blockIdx.x / a.parts, row = a.row0 + r;
  const T* xr = (const T*)a.x + row * a.ldx;
  T* gr = (T*)a.g + row * a.ldg;
  const Place<T> pl(xr, a.V);
  const int v0 = min(part * a.pv, pl.nmain), v1 = min(v0 + a.pv, pl.nmain);
  const bool lastp = part == a.parts - 1;
  const int e0 = part == 0 ? 0 : pl.h + v0 * N, e1 = lastp ? a.V : pl.h + v1 * N;
  const int bbase = pl.h + v0 * N - BIT0;
  const int ee = part == 0 && tid < pl.h ? tid : (lastp && pl.hV + (PT - 1 - tid) < a.V ? pl.hV + (PT - 1 - tid) : -1);
  const double w = a.w != nullptr ? ld_real(a.w, a.wdt, row) : 1.0;
  double v_row = 0.0;
  if (w == 0.0) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int v = v0 + tid; v < v1; v += PT) st16(gr + pl.h + (int64_t)v * N, zero);
    if (ee >= 0) gr[ee] = (T)0.f;
  } else {
    const int words = (a.pv * N + BIT0 + N + 31) / 32;
    for (int i = tid; i < words; i += PT) bm[i] = 0;
    if (tid == 0) dup = 0;
    __syncthreads();
    const int64_t y = a.lab != nullptr ? ld_int(a.lab, a.labbits, row) : -1;
    // the teacher's side: log normaliser and listed mass
    double tm = -INFINITY, ts = 0.0;
    for (int k = tid; k < a.K; k += PT) {
      const int64_t id = ld_int(a.idx, a.ibits, row * a.ldi + k);
      if (id < 0 || id >= a.V) continue;
      if (id >= e0 && id < e1) {
        const int b = (int)id - bbase;
        if ((atomicOr(&bm[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1u) dup = 1;
      }
      const double t = ld_real(a.t, a.tdt, row * a.ldt + k) * a.invT;
      if constexpr (TAIL) {
        ts += exp(t - ld_real(a.lse, a.lsedt, row));
      } else if (t > tm || t != t) {
        ts = t != t ? t : ts * exp(tm - t) + 1.0;
        if (t > tm) tm = t;
      } else if (t > -INFINITY) {
        ts += exp(t - tm);
      }
    }
    const double wm = wave_max(tm);
    const double wsum = wave_sum(TAIL || tm == -INFINITY ? ts : ts * exp(tm - wm));
    if (lane == 0) smd[wave][0] = wm, smd[wave][1] = wsum;
    __syncthreads();
    tm = smd[0][0];
    for (int i = 1; i < PT / 64; ++i) tm = fmax(tm, smd[i][0]);
    ts = 0.0;
    for (int i = 0; i < PT / 64; ++i) ts += TAIL || smd[i][0] == -INFINITY ? smd[i][1] : smd[i][1] * exp(smd[i][0] - tm);
    const double norm = TAIL ? ld_real(a.lse, a.lsedt, row) : tm + log(ts);
    const double mass = TAIL ? ts : (ts == 0.0 ? 0.0 : ts / ts);  // a list without mass: no teacher
    // the row's parts joined, one lane each
    const double* st = a.stat + r * a.parts * STAT;
    const bool in = lane < a.parts;
    const C pm = in ? (C)st[lane * STAT] : Lim<C>::lowest;
    const C M = wave_max(pm);
    const C c = (C)(a.invT * LOG2E);
    const C f = ex2((pm - M) * c);
    const C s = wave_sum(in ? (C)st[lane * STAT + 1] * f : C(0));
    const C sl = TAIL ? wave_sum(in ? (C)st[lane * STAT + 2] * f : C(0)) : C(0);
    const C s1 = TWO ? wave_sum(in ? (C)st[lane * STAT + 3] * ex2((pm - M) * (C)LOG2E) : C(0)) : C(0);
    const C nl = TAIL ? wave_sum(in ? (C)st[lane * STAT + 4] : C(0)) : C(0);
    const RowScal<C> rs = row_scalars<C, TAIL, TWO>(a, w, y >= 0, M, s, sl, s1, nl, mass);
    for (int v = v0 + tid; v < v1; v += PT) {
      C x[N], o[N];
      unpack<T>(ld16(xr + pl.h + (int64_t)v * N), x);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        o[i] = ex2((x[i] - rs.M) * c) * rs.cR;
        if constexpr (TWO) o[i] += ex2((x[i] - rs.M) * (C)LOG2E) * rs.c1;
      }
      st16(gr + pl.h + (int64_t)v * N, pack<T>(o));
    }
    auto entry = [&](C x, C coef) { return ex2((x - rs.M) * c) * coef + (TWO ? ex2((x - rs.M) * (C)LOG2E) * rs.c1 : C(0)); };
    if (ee >= 0) gr[ee] = (T)entry(up<T>(xr[ee]), rs.cR);
    __syncthreads();  // the vectors are written: the listed entries go over them
    const double* xk = a.xk + r * (a.K + 1);
    for (int k = tid; k < a.K; k += PT) {
      const int64_t id = ld_int(a.idx, a.ibits, row * a.ldi + k);
      if (id < 0 || id >= a.V) continue;
      C lp, p;
      entry_p<C>(a, row, k, norm, lp, p);
      const C x = (C)xk[k];
      if (part == 0 && !rs.empty && p != C(0)) v_row += a.lam * w * (double)(p * (lp - ((x - rs.M) * (C)a.invT - rs.ls)));
      if (id >= e0 && id < e1) {
        C ph = p;
        bool owner = true;
        if (dup) {  // a class listed twice: its first entry writes the sum
          for (int q = 0; q < a.K; ++q) {
            if (q == k || ld_int(a.idx, a.ibits, row * a.ldi + q) != id) continue;
            owner &= q > k;
            C lq, pq;
            entry_p<C>(a, row, q, norm, lq, pq);
            ph += pq;
          }
        }
        if (owner) gr[id] = (T)(entry(x, rs.cB) - rs.ql * ph - (id == y ? rs.qy : C(0)));
      }
    }
    if (tid == PT - 1) {
      if (y >= e0 && y < e1) {
        const int b = (int)y - bbase;
        if (!((bm[b >> 5] >> (b & 31)) & 1u)) gr[y] = (T)(entry((C)xk[a.K], rs.cR) - rs.qy);
      }
      if (part == 0 && !rs.empty) {
        if (TAIL && rs.pr != 0.0) v_row += a.lam * w * rs.pr * (log(rs.pr) - rs.log_qr);
        if (y >= 0 && y < a.V) v_row += a.lab_lam * w * (double)(rs.ls1 - ((C)xk[a.K] - rs.M));
        if (rs.ls != rs.ls) v_row = NAN;  // a NaN score, or an index or label out of range
      }
    }
  }
  double v[1] = {v_row}, one[1] = {1.0}, fin[1];
  if (grid_reduce_finalize<1, 0, PT / 64>(v, a.partials, a.counter, a.acc + 1, one, fin) && threadIdx.x == 0) {
    const double total = a.first ? fin[0] : *a.acc + fin[0];
    *a.acc = total;
    if (a.last) {
      *a.out = total;
      if (a.value != nullptr) *(C*)a.value = (C)total;
    }
  }
}

template <typename T, bool TAIL, bool TWO>
pg_status run_parts(pg_ctx* c, DArgs a, int64_t rows) {
  constexpr int N = Elem<T>::N;
  const int64_t vecs = (a.V + N - 1) / N;
  // a part: at least 1024 vectors (16 KiB), at most what the bitmap holds; enough parts for two workgroups per CU
  const int64_t most = (32 * 1024 * 8) / N;
  int64_t parts = (2 * c->num_cu + rows - 1) / rows;
  parts = std::min<int64_t>(parts, (vecs + 1023) / 1024);
  parts = std::max<int64_t>(parts, (vecs + most - 1) / most);
  parts = std::max<int64_t>(1, std::min<int64_t>(parts, MAX_PARTS));
  a.parts = (int)parts;
  a.pv = (int)((vecs + parts - 1) / parts);
  const size_t lds = ((size_t)a.pv * N + BIT0 + N + 31) / 32 * 4 + 4;
  if (lds > 64 * 1024) {
    pg_set_error("pg_distill: rows of more than %lld classes are not supported for this type", (long long)(64 * 1024 * 8 / N * N) * MAX_PARTS);
    return PG_ERR_UNSUPPORTED;
  }
  const int64_t ws = (int64_t)PG_RED_MAX_BLOCKS * (PG_RED_MAX_NS - 1) - 8;  // doubles behind the reduction's own partials
  int64_t batch = std::min<int64_t>(ws / (parts * STAT + a.K + 1), PG_RED_MAX_BLOCKS / parts);
  a.acc = c->red_partials + PG_RED_MAX_BLOCKS;
  a.stat = a.acc + 8;
  for (int64_t r0 = 0; r0 < rows; r0 += batch) {
    const int64_t nb = std::min<int64_t>(batch, rows - r0);
    a.row0 = r0;
    a.nrows = nb;
    a.xk = a.stat + nb * parts * STAT;
    a.first = r0 == 0;
    a.last = r0 + nb == rows;
    distill_part_stats<T, TAIL, TWO><<<(unsigned)(nb * parts), PT, lds, c->stream>>>(a);
    PG_LAUNCH_CHECK();
    distill_part_grad<T, TAIL, TWO><<<(unsigned)(nb * parts), PT, lds, c->stream>>>(a);
    PG_LAUNCH_CHECK();
  }
  return PG_OK;
}

template <typename T>
pg_status run_t(pg_ctx* c, const DArgs& a, int64_t rows, bool tail, bool two) {
  if (tail) return two ? run_parts<T, true, true>(c, a, rows) : run_parts<T, true, false>(c, a, rows);
  return two ? run_parts<T, false, true>(c, a, rows) : run_parts<T, false, false>(c, a, rows);
}

__global__ void store_zero(double* out, void* value, int f64) {
  *out = 0.0;
  if (value != nullptr) {
    if (f64) *(double*)value = 0.0;
    else *(float*)value = 0.f;
  }
}

}  // namespace
}  // namespace pgrows

extern "C" {

int32_t pg_rows_abi_version(void) { return PG_ROWS_ABI_VERSION; }

pg_status pg_distill_value_and_gradient(pg_ctx* c, const pg_distill* d, int32_t dtype, const void* scores, int64_t ld, void* grad,
                                        int64_t grad_ld, void* value, double* f_out) {
  using namespace pgrows;
  PG_REQUIRE(c != nullptr && d != nullptr, "null argument");
  PG_REQUIRE(dtype_ok(dtype), "bad dtype");
  PG_REQUIRE(d->rows >= 0 && d->classes >= 0 && d->top >= 0, "negative size");
  PG_REQUIRE(d->classes < (1ll << 30), "classes must be below 2^30");
  PG_REQUIRE(d->top <= MAX_TOP, "top must be at most 1024");
  PG_REQUIRE(d->temperature > 0.0 && std::isfinite(d->temperature), "temperature must be positive and finite");
  PG_REQUIRE(d->lam >= 0.0 && d->label_lam >= 0.0 && std::isfinite(d->lam) && std::isfinite(d->label_lam), "lam and label_lam must be nonnegative and finite");
  const bool any = d->rows > 0 && d->classes > 0;
  if (any) {
    PG_REQUIRE(scores != nullptr && grad != nullptr, "null rows");
    PG_REQUIRE((ld >= d->classes && grad_ld >= d->classes) || d->rows == 1, "rows overlap: ld below the number of classes");
    PG_REQUIRE(scores != grad || ld == grad_ld || d->rows == 1, "a gradient in the scores' own buffer needs the scores' ld");
    PG_REQUIRE(((uintptr_t)scores | (uintptr_t)grad) % dtype_size(dtype) == 0, "scores or gradient not aligned to their element");
    if (d->top > 0) {
      PG_REQUIRE(d->teacher != nullptr && d->index != nullptr, "null teacher");
      PG_REQUIRE(dtype_ok(d->teacher_dtype), "bad teacher_dtype");
      PG_REQUIRE(d->index_bits == 32 || d->index_bits == 64, "index_bits must be 32 or 64");
    }
    PG_REQUIRE(d->teacher_lse == nullptr || d->lse_dtype == PG_F32 || d->lse_dtype == PG_F64, "bad lse_dtype");
    PG_REQUIRE(d->weights == nullptr || d->weights_dtype == PG_F32 || d->weights_dtype == PG_F64, "bad weights_dtype");
    PG_REQUIRE(d->labels == nullptr || d->label_bits == 32 || d->label_bits == 64, "label_bits must be 32 or 64");
  }
  DeviceScope dev(c->device);
  PG_TRY(dev.st);
  PG_TRY(refuse_foreign_capture(c));
  double* out = c->dscal + PG_S_MISC;
  if (!any) {
    store_zero<<<1, 1, 0, c->stream>>>(out, value, dtype == PG_F64);
    PG_LAUNCH_CHECK();
  } else {
    DArgs a{};
    a.x = scores, a.g = grad, a.t = d->teacher, a.idx = d->index, a.lse = d->teacher_lse, a.w = d->weights, a.lab = d->labels;
    a.ldx = ld, a.ldg = grad_ld, a.ldt = d->teacher_ld, a.ldi = d->index_ld;
    a.V = (int)d->classes, a.K = (int)d->top;
    a.tdt = d->teacher_dtype, a.ibits = d->index_bits, a.lsedt = d->lse_dtype, a.wdt = d->weights_dtype, a.labbits = d->label_bits;
    a.invT = 1.0 / d->temperature, a.lam = d->lam, a.lab_lam = d->label_lam;
    a.partials = c->red_partials, a.counter = c->red_counter, a.out = out, a.value = value;
    const bool tail = d->teacher_lse != nullptr && d->top > 0, two = d->labels != nullptr && d->temperature != 1.0;
    if (dtype == PG_F32) PG_TRY(run_t<float>(c, a, d->rows, tail, two));
    else if (dtype == PG_F64) PG_TRY(run_t<double>(c, a, d->rows, tail, two));
    else if (dtype == PG_BF16) PG_TRY(run_t<__bf16>(c, a, d->rows, tail, two));
    else PG_TRY(run_t<_Float16>(c, a, d->rows, tail, two));
  }
  if (f_out == nullptr) return PG_OK;
  PG_TRY(pg_read_scalars(c, PG_S_MISC, 1));
  *f_out = c->hscal[PG_S_MISC];
  return PG_OK;
}

}  // extern "C"
