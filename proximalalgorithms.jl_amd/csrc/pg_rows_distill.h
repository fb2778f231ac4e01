// Kernels of the distillation loss (pg_rows_distill.hip has the entry point; one translation unit per element type).
//
// Per row, with z = x / T, e_v = exp(z_v - max z), S = sum e, q = e / S, the listed classes and their p:
//   L = sum_k p_k (log p_k - log q_k) + p_r (log p_r - log Q_r),     Q_r = sum of q outside the list
//   dL/dx_v = ((sum p + p_r) q_v - phat_v - [v not listed] p_r q_v / Q_r) / T
// so outside the list the gradient is ONE multiple of e_v, and only the listed classes (and the label) need more: every
// vector is written with the unlisted coefficient, then a few threads overwrite the listed entries.  Q_r is summed over
// the unlisted classes themselves (1 - sum of the listed q loses everything where the student agrees with the teacher),
// which a bitmap of the row in LDS makes possible; the bitmap also finds classes listed twice.
//
// Bound by memory: 8192 x 131072 bf16 838 us (5.13 TB/s read and written, a copy of that size 4.7), 4096 x 32768 bf16 103 us (5.2; a copy 5.4);
// with the outside class, 2048 x 131000 bf16, 250 us (4.3): 31 us a row and CU, 25 of them memory, the vector unit 19 (half of
// that two exponentials a score at a quarter of the rate) -- the difference is the reduction between the passes.
#pragma once
#include <algorithm>

#include "pg_rows.h"

namespace pgrows {

struct DArgs;
pg_status distill_f32(pg_ctx* c, const DArgs& a, int64_t rows);
pg_status distill_f64(pg_ctx* c, const DArgs& a, int64_t rows);
pg_status distill_bf16(pg_ctx* c, const DArgs& a, int64_t rows);
pg_status distill_f16(pg_ctx* c, const DArgs& a, int64_t rows);

constexpr double LOG2E = 1.4426950408889634;
constexpr double LN2 = 0.6931471805599453;
constexpr int BIT0 = 8;         // bits in front of a chunk's first aligned vector (the head of a misaligned row: at most 7)
constexpr int STAT = 8;         // doubles per (row, part)
constexpr int MAX_PARTS = 64;   // one lane each when a row's parts are joined
constexpr int MAX_TOP = 1024;
constexpr int PART_BITS = 32 * 1024 * 8;                          // classes of a part: its bitmap takes 32 KiB of LDS
constexpr int64_t MAX_CLASSES = (int64_t)MAX_PARTS * PART_BITS;  // 2^24

struct DArgs {
  const void* x;
  void* g;
  const void *t, *idx, *lse, *w, *lab;
  int64_t ldx, ldg, ldt, ldi, row0, nrows;  // rows of this launch
  int V, K, tdt, ibits, lsedt, wdt, labbits;
  double invT, lam, lab_lam;
  int squares;  // T = 2: 1, T = 4: 2, else 0
  int parts, pv;  // parts of a row, 16-byte vectors per part
  double *stat, *xk;
  double *partials, *acc, *out;
  unsigned* counter;
  void* value;
  int first, last;  // of the launches of this call
};

namespace {

// ---- one row's scalars, from the statistics over the whole row ----------------------------------------------------
template <typename C>
struct Sums {  // of exp((x - m) / T) and exp(x - m)
  C m, s, s1;
  static __device__ __forceinline__ Sums none() { return {Lim<C>::lowest, C(0), C(0)}; }
};
template <typename C>
struct RowScal {
  C M, Mu;           // reference scores: of the row, of the unlisted classes (the same where the list is no class of its own)
  C cB, cR, c1, c1u; // coefficients: of exp((x - M) / T) at listed classes, of exp((x - Mu) / T) at the others, of exp(x - M), exp(x - Mu) for labels at T != 1
  C ql, qy;          // what a unit of teacher mass / the label takes off
  C S, S1, Su;       // sums of exp((x - M) / T), exp(x - M), and over the unlisted of exp((x - Mu) / T)
  double pr;
  bool empty;
};
// what only the value needs: log sum exp((x - M) / T), log sum exp(x - M), log of the student's mass outside the list
template <typename C>
struct RowLogs {
  C ls, ls1;
  double log_qr;
  template <typename Args>
  __device__ __forceinline__ RowLogs(const Args& a, const RowScal<C>& r, bool two)
      : ls(lg2(r.S) * (C)LN2), ls1(two ? lg2(r.S1) * (C)LN2 : ls), log_qr((double)(lg2(r.Su) * (C)LN2 + (r.Mu - r.M) * (C)a.invT - ls)) {}
};
// u: the unlisted classes, or without an outside class all; l: the listed ones.  Each has its own reference: what the outside class gets is
// divided among its classes by their softmax, however far below the listed ones they lie.
template <typename C, typename Args>
__device__ __forceinline__ RowScal<C> row_scalars(const Args& a, bool tail, bool two, double w, bool has_label, const Sums<C>& u, const Sums<C>& l, C n_listed,
                                                  double mass) {
  RowScal<C> r;
  r.M = r.Mu = u.m;
  C S = u.s, S1 = u.s1, wu = C(1), w1 = C(1);
  if (tail) {
    const C c = (C)(a.invT * LOG2E);
    r.M = fmx(u.m, l.m);
    wu = ex2((u.m - r.M) * c);
    S = u.s * wu + l.s * ex2((l.m - r.M) * c);
    if (two) {
      w1 = ex2((u.m - r.M) * (C)LOG2E);
      S1 = u.s1 * w1 + l.s1 * ex2((l.m - r.M) * (C)LOG2E);
    }
  }
  r.empty = S == C(0);  // every score -inf (the largest score always contributes 1)
  r.S = S, r.S1 = S1, r.Su = u.s;
  r.ql = (C)(a.lam * w * a.invT);
  r.qy = has_label ? (C)(a.lab_lam * w) : C(0);
  C rest = C(0);
  r.pr = 0.0;
  if (tail) {
    if ((int64_t)n_listed < a.V) {  // the list may hold every class: then nothing is outside it
      const double left = 1.0 - mass;
      r.pr = left > 0.0 ? left : (left == left ? 0.0 : left);
      rest = (r.pr > 0.0 && u.s > C(0)) ? (C)r.pr / u.s : C(0);
    }
  }
  const C total = (C)(mass + r.pr), inv = C(1) / S;
  r.cB = r.ql * total * inv;
  r.cR = tail ? r.ql * (total * wu * inv - rest) : r.cB;
  r.c1 = r.c1u = C(0);
  if (two) {
    r.c1 = r.qy / S1;
    r.c1u = r.c1 * w1;
  } else {  // labels at T = 1 share e
    r.cB += r.qy * inv;
    r.cR += r.qy * wu * inv;
  }
  if (r.empty) {
    r.cB = r.cR = r.c1 = r.c1u = r.ql = r.qy = C(0);
    r.M = r.Mu = Lim<C>::lowest;
  }
  return r;
}
// the gradient's entry at a listed class (less its teacher's mass and label), and at any other
template <bool two, typename C>
__device__ __forceinline__ C entry_listed(const RowScal<C>& r, C x, C c) {
  return ex2((x - r.M) * c) * r.cB + (two ? ex2((x - r.M) * (C)LOG2E) * r.c1 : C(0));
}
template <bool two, typename C>
__device__ __forceinline__ C entry_other(const RowScal<C>& r, C x, C c) {
  return ex2((x - r.Mu) * c) * r.cR + (two ? ex2((x - r.Mu) * (C)LOG2E) * r.c1u : C(0));
}

// probability of a listed entry: log p and p
template <typename C>
__device__ __forceinline__ void entry_p(const DArgs& a, int64_t row, int k, double norm, C& lp, C& p) {
  const double t = ld_real(a.t, a.tdt, row * a.ldt + k) * a.invT;
  lp = (C)(t == -INFINITY ? t : t - norm);  // (a list of -inf only has norm -inf)
  p = ex2(lp * (C)LOG2E);
}

// ---- a row's place in memory: head elements up to the first boundary of ALIGN bytes, whole 16-byte vectors, tail -----------------
template <typename T, int ALIGN = 16>
struct Place {
  int h, nmain, hV;
  __device__ __forceinline__ Place(const T* xr, int V) {
    constexpr int N = Elem<T>::N;
    const int off = (int)((reinterpret_cast<uintptr_t>(xr) & (ALIGN - 1u)) / sizeof(T));
    h = off ? ALIGN / (int)sizeof(T) - off : 0;
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

// what(i, exp(x_i - m)) for each i, beside e = exp((x - m) / T): e squared once for T = 2, twice for T = 4 (`squares`; a rounding each,
// against a whole exponential), else an exponential of its own
template <typename C, int N, typename F>
__device__ __forceinline__ void power(int squares, const C (&x)[N], const C (&e)[N], C m, F what) {
  if (squares == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) what(i, e[i] * e[i]);
  } else if (squares == 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) what(i, (e[i] * e[i]) * (e[i] * e[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) what(i, ex2((x[i] - m) * (C)LOG2E));
  }
}
// f[i] = -inf where bit i is set: two operations each (written in C they become five, or a test, a comparison and a choice)
template <int I = 0, int N>
__device__ __forceinline__ void leave_out(float (&f)[N], unsigned bits) {
  if constexpr (I < N) {
    int m;
    asm("v_bfe_i32 %0, %2, %3, 1\n\tv_bfi_b32 %1, %0, %4, %1" : "=&v"(m), "+v"(f[I]) : "v"(bits), "n"(I), "s"(0xff800000u));
    leave_out<I + 1>(f, bits);
  }
}
template <int N>
__device__ __forceinline__ void leave_out(double (&f)[N], unsigned bits) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (bits >> i) & 1u ? -(double)INFINITY : f[i];
}

// Sums of one thread, relative to a reference score m that is one of the row's (or the type's lowest value while there is
// none): any score will do that is not far below the largest, so m is raised rarely, by a branch.  Far:
// an exponent of 20, whose rounding is 20 * 2^-24 of its exponential, like those of the terms that count least.
template <typename C, bool TWO>
struct Run : Sums<C> {
  using Sums<C>::m;
  using Sums<C>::s;
  using Sums<C>::s1;
  C lim = Lim<C>::lowest;
  C c, head;  // log2(e) / T; an exponent of 20 in scores
  int squares;
  __device__ __forceinline__ Run(double invT, int sq) : Sums<C>(Sums<C>::none()), c(uniform((C)(invT * LOG2E))), head(uniform((C)(20.0 / fmax(invT, 1.0)))), squares(sq) {}
  __device__ __forceinline__ void raise(C to) {
    const C d = m - to;
    s *= ex2(d * c);
    if constexpr (TWO) s1 *= ex2(d * (C)LOG2E);
    m = to;
    lim = to + head;
    opaque(m);  // keep the branch
  }
  template <int N>
  __device__ __forceinline__ void add(C (&f)[N], unsigned bits) {  // bits: elements to leave out
    if (bits) leave_out(f, bits);
    C vm = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i) vm = fmx(vm, f[i]);
    if (vm > lim) raise(vm);
    C e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = ex2((f[i] - m) * c);
    if constexpr (TWO) {
      C t[2] = {C(0), C(0)};
      power(squares, f, e, m, [&](int i, C v) { t[i & 1] += v; });
      s1 += t[0] + t[1];
    }
#pragma unroll
    for (int o = 1; o < N; o *= 2)
#pragma unroll
      for (int i = 0; i < N; i += 2 * o) e[i] += e[i + o];
    s += e[0];
  }
  __device__ __forceinline__ void add1(C x) {
    if (x > lim) raise(x);
    s += ex2((x - m) * c);
    if constexpr (TWO) s1 += ex2((x - m) * (C)LOG2E);
  }
  // over the wave's lanes
  __device__ __forceinline__ Sums<C> joined() const {
    Sums<C> o = Sums<C>::none();
    o.m = wave_max(m);
    o.s = wave_sum(s * ex2((m - o.m) * c));
    if constexpr (TWO) o.s1 = wave_sum(s1 * ex2((m - o.m) * (C)LOG2E));
    return o;
  }
};
// of two sets of scores
template <bool TWO, typename C>
__device__ __forceinline__ void join(Sums<C>& to, const Sums<C>& o, C c) {
  const C m = fmx(to.m, o.m), d = to.m - m, e = o.m - m;
  to.s = to.s * ex2(d * c) + o.s * ex2(e * c);
  if constexpr (TWO) to.s1 = to.s1 * ex2(d * (C)LOG2E) + o.s1 * ex2(e * (C)LOG2E);
  to.m = m;
}

// ---- the general form: a row in parts, two reads ------------------------------------------------------------------
// Any length, and few rows: a part per workgroup.  First launch: the statistics of each part (and the listed scores, which an
// in-place gradient overwrites); second launch: every part joins its row's statistics and writes its piece of the
// gradient; the second read comes from a cache where the rows are few.  What a workgroup needs is asked for at its start.
constexpr int PT = 256;  // threads
constexpr int PV = 4;    // vectors of a thread at a time

template <typename T>
struct Part {
  Place<T> pl;
  int part, v0, v1, e0, e1, bbase, ee, words;
  int64_t r, row;
  __device__ __forceinline__ Part(const DArgs& a)
      : pl((const T*)a.x + (a.row0 + blockIdx.x / a.parts) * a.ldx, a.V), part(blockIdx.x % a.parts), r(blockIdx.x / a.parts), row(a.row0 + r) {
    constexpr int N = Elem<T>::N;
    const int tid = threadIdx.x;
    v0 = min(part * a.pv, pl.nmain), v1 = min(v0 + a.pv, pl.nmain);
    const bool last = part == a.parts - 1;
    e0 = part == 0 ? 0 : pl.h + v0 * N, e1 = last ? a.V : pl.h + v1 * N;  // its classes
    bbase = pl.h + v0 * N - BIT0;                                         // class of bit 0
    // thread i: the i-th element of the row's head; thread PT - 1 - i: of its tail
    ee = part == 0 && tid < pl.h ? tid : (last && pl.hV + (PT - 1 - tid) < a.V ? pl.hV + (PT - 1 - tid) : -1);
    words = (a.pv * N + BIT0 + N + 31) / 32;
  }
  __device__ __forceinline__ bool has(int64_t e) const { return e >= e0 && e < e1; }
};

template <typename T, bool TAIL, bool TWO>
__global__ __launch_bounds__(PT) void distill_part_stats(DArgs a) {
  using C = typename Elem<T>::C;
  constexpr int N = Elem<T>::N;
  extern __shared__ unsigned bm[];
  __shared__ Sums<C> sm[PT / 64][2];
  __shared__ C sn[PT / 64];
  __shared__ int dup;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Part<T> q(a);
  if (a.w != nullptr && ld_real_u(a.w, a.wdt, q.row) == 0.0) return;
  const T* xr = (const T*)a.x + q.row * a.ldx;
  const T* xm = xr + q.pl.h;
  u32x4 d[PV];
  auto load = [&](int v) {
#pragma unroll
    for (int j = 0; j < PV; ++j) d[j] = v + j * PT < q.v1 ? ld16(at16(xm, v + j * PT)) : minus_inf16<T>();
  };
  load(q.v0 + tid);
  const T edge = q.ee >= 0 ? xr[q.ee] : (T)0.f;
  if constexpr (TAIL) {
    for (int i = tid; i < q.words; i += PT) bm[i] = 0;
    if (tid == 0) dup = 0;
    __syncthreads();
  }
  Run<C, TWO> run(a.invT, a.squares), list(a.invT, a.squares);
  C n = C(0);  // listed classes
  bool bad = false;
  for (int k = tid; k < a.K; k += PT) {
    const int64_t id = ld_int(a.idx, a.ibits, q.row * a.ldi + k);
    bad |= id < -1 || id >= a.V;
    if (q.has(id)) {
      const C x = up<T>(xr[id]);
      a.xk[q.r * (a.K + 1) + k] = (double)x;
      if constexpr (TAIL) {
        const int b = (int)id - q.bbase;
        const unsigned old = atomicOr(&bm[b >> 5], 1u << (b & 31));
        if (!((old >> (b & 31)) & 1u)) list.add1(x), n += C(1);
        else dup = 1;
      }
    }
  }
  if (tid == 0 && a.lab != nullptr) {
    const int64_t y = ld_int_u(a.lab, a.labbits, q.row);
    bad |= y < -1 || y >= a.V;
    if (q.has(y)) a.xk[q.r * (a.K + 1) + a.K] = (double)up<T>(xr[y]);
  }
  if constexpr (TAIL) {
    __syncthreads();
    if (dup) {  // a class listed twice: its first entry counts, whichever came to the bitmap first, so that the sums keep their order
      list = Run<C, TWO>(a.invT, a.squares), n = C(0);
      for (int k = tid; k < a.K; k += PT) {
        const int64_t id = ld_int(a.idx, a.ibits, q.row * a.ldi + k);
        if (!q.has(id)) continue;
        bool first = true;
        for (int o = 0; o < k; ++o) first &= ld_int(a.idx, a.ibits, q.row * a.ldi + o) != id;
        if (first) list.add1(up<T>(xr[id])), n += C(1);
      }
    }
  }
  for (int v = q.v0 + tid; v - tid < q.v1; v += PV * PT) {
    if (v != q.v0 + tid) load(v);
#pragma unroll
    for (int j = 0; j < PV; ++j) {
      C f[N];
      unpack<T>(d[j], f);
      run.template add<N>(f, TAIL ? listed_bits<T>(bm, min(v + j * PT - q.v0, q.v1 - q.v0) * N + BIT0) : 0u);
    }
  }
  if (q.ee >= 0) {
    const int b = q.ee - q.bbase;
    if (!(TAIL && ((bm[b >> 5] >> (b & 31)) & 1u))) run.add1(up<T>(edge));
  }
  if (bad) run.s = (C)NAN;
  const Sums<C> u = run.joined();
  Sums<C> l = Sums<C>::none();
  if constexpr (TAIL) l = list.joined(), n = wave_sum(n);
  if (lane == 0) sm[wave][0] = u, sm[wave][1] = l, sn[wave] = n;
  __syncthreads();
  if (tid == 0) {
    Sums<C> all = sm[0][0], listed = sm[0][1];
    n = sn[0];
    for (int i = 1; i < PT / 64; ++i) {
      join<TWO>(all, sm[i][0], run.c);
      if constexpr (TAIL) join<TWO>(listed, sm[i][1], run.c), n += sn[i];
    }
    double* st = a.stat + (q.r * a.parts + q.part) * STAT;
    st[0] = (double)all.m, st[1] = (double)all.s, st[2] = (double)all.s1;
    st[3] = (double)listed.m, st[4] = (double)listed.s, st[5] = (double)listed.s1, st[6] = (double)n;
  }
}

template <typename T, bool TAIL, bool TWO>
__global__ __launch_bounds__(PT) void distill_part_grad(DArgs a) {
  using C = typename Elem<T>::C;
  constexpr int N = Elem<T>::N;
  extern __shared__ unsigned bm[];
  __shared__ C smt[PT / 64][2];
  __shared__ double smd[PT / 64];
  __shared__ int dup;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Part<T> q(a);
  const T* xr = (const T*)a.x + q.row * a.ldx;
  const T* xm = xr + q.pl.h;
  T* gr = (T*)a.g + q.row * a.ldg;
  T* gm = gr + q.pl.h;
  const double w = a.w != nullptr ? ld_real_u(a.w, a.wdt, q.row) : 1.0;
  double v_row = 0.0;
  if (w == 0.0) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int v = q.v0 + tid; v < q.v1; v += PT) st16(at16(gm, v), zero);
    if (q.ee >= 0) gr[q.ee] = (T)0.f;
  } else {
    u32x4 d[PV];
    auto load = [&](int v) {
#pragma unroll
      for (int j = 0; j < PV; ++j) d[j] = v + j * PT < q.v1 ? ld16(at16(xm, v + j * PT)) : minus_inf16<T>();
    };
    // the row's parts, one lane each
    const double* st = a.stat + q.r * a.parts * STAT;
    const int mine = min(lane, a.parts - 1) * STAT;
    Sums<C> pu = Sums<C>::none(), pl = pu;
    C pn = C(0);
    pu.m = (C)st[mine], pu.s = (C)st[mine + 1];
    if constexpr (TWO) pu.s1 = (C)st[mine + 2];
    if constexpr (TAIL) pl.m = (C)st[mine + 3], pl.s = (C)st[mine + 4], pn = (C)st[mine + 6];
    if constexpr (TAIL && TWO) pl.s1 = (C)st[mine + 5];
    load(q.v0 + tid);
    const T edge = q.ee >= 0 ? xr[q.ee] : (T)0.f;
    for (int i = tid; i < q.words; i += PT) bm[i] = 0;
    if (tid == 0) dup = 0;
    __syncthreads();
    const int64_t y = a.lab != nullptr ? ld_int_u(a.lab, a.labbits, q.row) : -1;
    const double lse = TAIL ? ld_real_u(a.lse, a.lsedt, q.row) : 0.0;
    // the teacher's side: log normaliser and listed mass
    C tm = Lim<C>::lowest, ts = C(0);
    double tmass = 0.0;
    for (int k = tid; k < a.K; k += PT) {
      const int64_t id = ld_int(a.idx, a.ibits, q.row * a.ldi + k);
      if (id < 0 || id >= a.V) continue;
      if (q.has(id)) {
        const int b = (int)id - q.bbase;
        if ((atomicOr(&bm[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1u) dup = 1;
      }
      const double t = ld_real(a.t, a.tdt, q.row * a.ldt + k) * a.invT;
      if constexpr (TAIL) {
        tmass += exp_series(t - lse);
      } else {
        const C tc = (C)t;
        if (tc > tm) {
          ts *= ex2((tm - tc) * (C)LOG2E);
          tm = tc;
        }
        ts += ex2((tc - tm) * (C)LOG2E);
      }
    }
    if constexpr (TAIL) {
      tmass = wave_sum(tmass);
      if (lane == 0) smd[wave] = tmass;
    } else {
      const C wm = wave_max(tm);
      ts = wave_sum(ts * ex2((tm - wm) * (C)LOG2E));
      if (lane == 0) smt[wave][0] = wm, smt[wave][1] = ts;
    }
    __syncthreads();
    double norm, mass;
    if constexpr (TAIL) {
      norm = lse;
      mass = smd[0];
      for (int i = 1; i < PT / 64; ++i) mass += smd[i];
    } else {
      tm = smt[0][0];
      for (int i = 1; i < PT / 64; ++i) tm = fmx(tm, smt[i][0]);
      ts = C(0);
      for (int i = 0; i < PT / 64; ++i) ts += smt[i][1] * ex2((smt[i][0] - tm) * (C)LOG2E);
      norm = (double)tm + (double)(lg2(ts) * (C)LN2);
      mass = ts == C(0) ? 0.0 : (double)(ts / ts);  // a list without mass: no teacher
    }
    const bool in = lane < a.parts;
    const C c = (C)(a.invT * LOG2E);
    auto over_parts = [&](const Sums<C>& p) {
      Sums<C> o = Sums<C>::none();
      o.m = wave_max(p.m);
      o.s = wave_sum(in ? p.s * ex2((p.m - o.m) * c) : C(0));
      if constexpr (TWO) o.s1 = wave_sum(in ? p.s1 * ex2((p.m - o.m) * (C)LOG2E) : C(0));
      return o;
    };
    const Sums<C> u = over_parts(pu);
    Sums<C> l = Sums<C>::none();
    C nl = C(0);
    if constexpr (TAIL) l = over_parts(pl), nl = wave_sum(in ? pn : C(0));
    const RowScal<C> rs = row_scalars<C>(a, TAIL, TWO, w, y >= 0, u, l, nl, mass);
    const RowLogs<C> lg(a, rs, TWO);
    for (int v = q.v0 + tid; v - tid < q.v1; v += PV * PT) {
      if (v != q.v0 + tid) load(v);
#pragma unroll
      for (int j = 0; j < PV; ++j) {
        if (v + j * PT >= q.v1) continue;
        C x[N], o[N];
        unpack<T>(d[j], x);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = entry_other<TWO>(rs, x[i], c);
        st16(at16(gm, v + j * PT), pack<T>(o));
      }
    }
    if (q.ee >= 0) gr[q.ee] = (T)entry_other<TWO>(rs, up<T>(edge), c);
    __syncthreads();  // the vectors are written: the listed entries go over them
    const double* xk = a.xk + q.r * (a.K + 1);
    for (int k = tid; k < a.K; k += PT) {
      const int64_t id = ld_int(a.idx, a.ibits, q.row * a.ldi + k);
      if (id < 0 || id >= a.V) continue;
      C lp, p;
      entry_p<C>(a, q.row, k, norm, lp, p);
      const C x = (C)xk[k];
      if (q.part == 0 && !rs.empty && p != C(0) && a.lam != 0.0) v_row += a.lam * w * ((double)p * ((double)lp - ((double)(x - rs.M) * a.invT - (double)lg.ls)));
      if (q.has(id)) {
        C ph = p;
        bool owner = true;
        if (dup) {  // a class listed twice: its first entry writes the sum
          for (int o = 0; o < a.K; ++o) {
            if (o == k || ld_int(a.idx, a.ibits, q.row * a.ldi + o) != id) continue;
            owner &= o > k;
            C lo, po;
            entry_p<C>(a, q.row, o, norm, lo, po);
            ph += po;
          }
        }
        if (owner) gr[id] = (T)(entry_listed<TWO>(rs, x, c) - rs.ql * ph - (id == y ? rs.qy : C(0)));
      }
    }
    if (tid == PT - 1) {
      if (q.has(y)) {
        const int b = (int)y - q.bbase;
        if (!((bm[b >> 5] >> (b & 31)) & 1u)) gr[y] = (T)(entry_other<TWO>(rs, (C)xk[a.K], c) - rs.qy);
      }
      if (q.part == 0 && !rs.empty) {
        if (TAIL && rs.pr != 0.0 && a.lam != 0.0) v_row += a.lam * w * rs.pr * ((double)(lg2((C)rs.pr) * (C)LN2) - lg.log_qr);
        if (y >= 0 && y < a.V && a.lab_lam != 0.0) v_row += a.lab_lam * w * (double)(lg.ls1 - ((C)xk[a.K] - rs.M));
      }
      if (rs.S != rs.S) v_row = NAN;  // a NaN score, or an index or label out of range
    }
  }
  if (q.part != 0) return;  // the first part of each row carries its value
  double total;
  if (sum_workgroups<PT / 64>(v_row, (unsigned)a.nrows, (unsigned)q.r, a.partials, a.counter, total)) {
    if (!a.first) total += *a.acc;
    *a.acc = total;
    if (a.last) store_value<C>(total, a.out, a.value);
  }
}

template <typename T, bool TAIL, bool TWO>
pg_status run_parts(pg_ctx* c, DArgs a, int64_t rows) {
  constexpr int N = Elem<T>::N;
  const int64_t vecs = (a.V + N - 1) / N;
  // two workgroups per CU if the rows are few, but no part below 2 vectors a thread, and none that its bitmap does not hold
  const int64_t most = PART_BITS / N;
  int64_t parts = (2 * c->num_cu + rows - 1) / rows;
  parts = std::min<int64_t>(parts, (vecs + 2 * PT - 1) / (2 * PT));
  parts = std::max<int64_t>(parts, (vecs + most - 1) / most);
  parts = std::max<int64_t>(1, std::min<int64_t>(parts, MAX_PARTS));
  a.parts = (int)parts;
  a.pv = (int)((vecs + parts - 1) / parts);
  const size_t lds = ((size_t)a.pv * N + BIT0 + N + 31) / 32 * 4 + 4;
  const int64_t ws = (int64_t)PG_RED_MAX_BLOCKS * (PG_RED_MAX_NS - 1) - 8;  // doubles behind the reduction's own partials
  const int64_t batch = std::min<int64_t>(ws / (parts * STAT + a.K + 1), PG_RED_MAX_BLOCKS);
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

// ---- the row in registers: one read, one write ---------------------------------------------------------------------
// NT threads hold a row as NV 16-byte vectors each (NT = 64: a wave per row, four rows per workgroup; else a workgroup per row).
// Pass 1 takes running maximum and sums as the vectors arrive, one reduction joins them, pass 2 writes the gradient from the
// registers and, as a vector leaves, loads the same vector of the group's NEXT row in its place, so that the memory pipes
// stay busy through the reduction.  Loads return in order, so nothing may be asked for between those loads and pass 1 that
// is needed before it: the next row's list is asked for a pass ahead and waits in LDS, and no register may spill there.
// Vectors start at a 128-byte line of the scores, and of the gradient where its rows lie alike, or each wave's access ends in two half
// lines (2048 x 131000 bf16: both on a line 235 us, one of them 246, both 8 bytes off 257; 65536 x 1003 f32, a wave to a row,
// 105 against 114 with vectors from 16 bytes).  64 bytes for a wave's rows of two-byte types: head and tail take a thread each.
template <typename T, int NT, int NV>
struct RowsGeom {
  using C = typename Elem<T>::C;
  static constexpr int N = Elem<T>::N;
  static constexpr int WG = NT < 256 ? 256 : NT;
  static constexpr int GPW = WG / NT, NW = NT / 64;
  static constexpr int capacity = NT * NV * N;  // classes a group's registers hold
  static constexpr int ALIGN = NT == 64 && sizeof(T) == 2 ? 64 : 128;
  static constexpr int FRONT = NT == 64 ? 32 : 64;  // bits in front of the first vector's: at least its head
  static __host__ __device__ int words(int V) { return ((V + FRONT + N + 31) / 32 + 1) & ~1; }
  // two bitmaps and two lists (this row's, the next's) of scores and classes, one of logits and of probabilities
  static __host__ __device__ int group_bytes(int V, int K) { return words(V) * 8 + (K * (4 * (int)sizeof(C) + 8) + 7) / 8 * 8; }
};

template <typename T, int NT, int NV, bool tail, bool two>
__global__ __launch_bounds__((NT < 256 ? 256 : NT), sizeof(T) == 8 ? 2 : (NT == 64 && NV <= 2 && !tail && !two ? 8 : 4)) void distill_rows(DArgs) {
  // (Waves to a SIMD.  Float64 in 128 registers spills some eighty of them: two, and no workgroup of 1024 threads.  Short rows wait for
  // their lists and each other's lines rather than for bandwidth: eight, 65536 x 500 f16 91 us, 104 with the six that 80 registers
  // allow; the other modes spill then and are no faster, 65536 x 500 f32 with an outside class 94 against 91.)

  // The arguments stay in memory and are read where they are used: hoisted out of the row loop they fill the scalar registers and
  // spill into vector ones
  const PG_CONST_AS DArgs* ap = (const PG_CONST_AS DArgs*)__builtin_amdgcn_kernarg_segment_ptr();
#define a (*ap)
  using G = RowsGeom<T, NT, NV>;
  using P = Place<T, G::ALIGN>;
  using C = typename G::C;
  constexpr int N = G::N, NW = G::NW, GPW = G::GPW;
  constexpr int AGAIN = 1 << 30;  // marks a list entry whose class an earlier one holds
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ Sums<C> sm[NW][2];  // [wave][unlisted, listed]; without an outside class the latter has the teacher's maximum and sum
  __shared__ C smn[NW];
  __shared__ double smt[NW];
  __shared__ C sxy[GPW][2];
  __shared__ int flags[GPW][3][2];  // [row mod 3][a class is listed twice, the label is listed]
  const int tid = threadIdx.x % NT, lane = threadIdx.x & 63;
  const int wave_in_wg = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int grp = NT == 64 ? wave_in_wg : 0, wave = NT == 64 ? 0 : wave_in_wg;
  const int nwords = G::words(a.V), K = a.K;
  unsigned* bm0 = (unsigned*)(lds + G::group_bytes(a.V, K) * grp);  // [2][nwords]
  C* lx0 = (C*)(bm0 + 2 * nwords);                                  // [2][K]
  C* lt = lx0 + 2 * K;                                              // [K] logits
  C* lp = lt + K;                                                   // [K] probabilities
  int* li0 = (int*)(lp + K);                                        // [2][K]
  for (int i = tid; i < 2 * nwords; i += NT) bm0[i] = 0;
  if (tid < 6) flags[grp][tid >> 1][tid & 1] = 0;
  group_sync<NT>();

  const int64_t stride = (int64_t)gridDim.x * GPW;
  const C c = uniform((C)(a.invT * LOG2E));

  // the next row that has a weight (the others' gradients are zeros)
  auto advance = [&](int64_t row, double& w) {
    w = 1.0;
    for (; row < a.nrows; row += stride) {
      if (a.w == nullptr || (w = ld_real_u(a.w, a.wdt, row)) != 0.0) break;
      T* gr = (T*)a.g + row * a.ldg;
      const P pl(gr, a.V);
      const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma clang loop unroll(disable)
      for (int v = tid; v < pl.nmain; v += NT) st16(at16(gr + pl.h, v), zero);
      if (tid < pl.h) gr[tid] = (T)0.f;
      if (pl.hV + tid < a.V) gr[pl.hV + tid] = (T)0.f;
    }
    return row;
  };
  // a row's list entry tid (class, logit) and label, not looked at yet
  auto ask_list = [&](int64_t row, RawInt& id, RawReal<C>& t, int64_t& y) {
    y = -1;
    if (row < a.nrows) {
      if (tid < K) {
        id.load(a.idx, a.ibits, row * a.ldi + tid);
        t.load(a.t, a.tdt, row * a.ldt + tid);
      }
      if (a.lab != nullptr) y = ld_int_u(a.lab, a.labbits, row);
    }
  };
  // class or label: -1 absent, -2 out of range
  auto checked = [&](int64_t i) { return i < -1 || i >= a.V ? -2 : (int)i; };
  // ... and the scores there (before anything overwrites them: the gradient may go into the scores' buffer)
  auto ask_scores = [&](int64_t row, int id, int y, T& x, T& xy) {
    x = xy = (T)0.f;
    if (row < a.nrows) {
      const T* xr = (const T*)a.x + row * a.ldx;
      if (id >= 0) x = xr[id];
      if (y >= 0 && tid == NT - 1) xy = xr[y];
    }
  };
  // the list into LDS: classes and their bits, scores, logits
  auto put_list = [&](int64_t row, int id, RawReal<C> t, int y, T x, T xy, int par, int slot) {
    if (row >= a.nrows) return;
    const T* xr = (const T*)a.x + row * a.ldx;
    const P pl(xr, a.V);
    unsigned* bm = bm0 + par * nwords;
    auto put = [&](int k, int id, C t, T x) {
      int mark = 0;
      if (id >= 0) {
        const int b = id - pl.h + G::FRONT;
        const unsigned bit = 1u << (b & 31);
        if (atomicOr(&bm[b >> 5], bit) & bit) {
          mark = AGAIN;
          flags[grp][slot][0] = 1;
        }
        if (id == y) flags[grp][slot][1] = 1;
      }
      li0[par * K + k] = id < 0 ? id : id | mark;
      lx0[par * K + k] = up<T>(x);
      lt[k] = t;
    };
    if (tid < K) put(tid, id, t.get(a.tdt), x);
#pragma clang loop unroll(disable)
    for (int k = tid + NT; k < K; k += NT) {
      const int i = checked(ld_int(a.idx, a.ibits, row * a.ldi + k));
      put(k, i, (C)ld_real(a.t, a.tdt, row * a.ldt + k), i >= 0 ? xr[i] : (T)0.f);
    }
    if (tid == NT - 1) sxy[grp][par] = up<T>(xy);
  };
  // of the entries of one class the first holds it, whichever came to the bitmap first: the sums keep their order
  auto order_list = [&](int par, int slot) {
    if (flags[grp][slot][0] == 0) return;
    int* li = li0 + par * K;
#pragma clang loop unroll(disable)
    for (int k = tid; k < K; k += NT) {
      if (li[k] < 0) continue;
      const int id = li[k] & ~AGAIN;
      bool again = false;
#pragma clang loop unroll(disable)
      for (int q = 0; q < k; ++q) again |= (li[q] & ~AGAIN) == id;
      li[k] = again ? id | AGAIN : id;
    }
  };
  // head elements: threads 0 ..; tail elements: threads NT - 1 .. down
  auto edge_of = [&](const P& pl) { return tid < pl.h ? tid : (pl.hV + (NT - 1 - tid) < a.V ? pl.hV + (NT - 1 - tid) : -1); };

  u32x4 d[NV];
  T edge = (T)0.f;
  double w;
  int y, par = 0, slot = 0;
  int64_t row = advance((int64_t)blockIdx.x * GPW + grp, w);
  {
    RawInt rid;
    RawReal<C> t;
    T x, xy;
    int64_t ry;
    ask_list(row, rid, t, ry);
    const int id = row < a.nrows && tid < K ? checked(rid.get(a.ibits)) : -1;
    y = checked(ry);
    ask_scores(row, id, y, x, xy);
    if (row < a.nrows) {
      const T* xr = (const T*)a.x + row * a.ldx;
      const P pl(xr, a.V);
      const int ee = edge_of(pl);
      if (ee >= 0) edge = xr[ee];
      const __amdgpu_buffer_rsrc_t rx = row_rsrc(xr + pl.h, pl.nmain * 16);
      const int off = tid * 16;
#pragma unroll
      for (int j = 0; j < NV; ++j) d[j] = ldb16(rx, off + j * NT * 16);
    }
    put_list(row, id, t, y, x, xy, 0, 0);
    group_sync<NT>();
    order_list(0, 0);
  }
  double v_acc = 0.0;
  while (row < a.nrows) {
    asm volatile("" : "+s"(ap));
    const T* xr = (const T*)a.x + row * a.ldx;
    T* gr = (T*)a.g + row * a.ldg;
    const P pl(xr, a.V);
    const int ee = edge_of(pl);
    const int bbase = pl.h - G::FRONT;
    unsigned* bm = bm0 + par * nwords;
    const C* lx = lx0 + par * K;
    const int* li = li0 + par * K;
    double w_next;
    RawInt id_raw;
    RawReal<C> t_next;
    int64_t y_raw;
    const int64_t nrow = advance(row + stride, w_next);
    ask_list(nrow, id_raw, t_next, y_raw);

    // pass 1
    Run<C, two> run(a.invT, a.squares);
    // the list, while the row is on its way: the teacher's mass, or maximum and sum, and the scores that the sums below leave out
    Run<C, two> listed(a.invT, a.squares);
    C tm = Lim<C>::lowest, ts = C(0), nl = C(0);
    double tmass = 0.0;
    bool bad = y == -2;
    const double lse = tail ? ld_real_u(a.lse, a.lsedt, row) : 0.0;
#pragma clang loop unroll(disable)
    for (int k = tid; k < K; k += NT) {
      const int id = li[k];
      bad |= id == -2;
      if (id < 0) continue;
      if constexpr (tail) {
        if (!(id & AGAIN)) listed.add1(lx[k]), nl += C(1);
        tmass += exp_series((double)lt[k] * a.invT - lse);
      } else {
        const C t = (C)((double)lt[k] * a.invT);
        if (t > tm) {
          ts *= ex2((tm - t) * (C)LOG2E);
          tm = t;
        }
        ts += ex2((t - tm) * (C)LOG2E);
      }
    }
    int t0 = tid;
    opaque(t0);
    auto bits_of = [&](int j) { return tail ? listed_bits<T>(bm, min(j * NT + t0, pl.nmain) * N + G::FRONT) : 0u; };
    unsigned bits_next = bits_of(0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * NT < pl.nmain) {
        const unsigned bits = bits_next;
        if (j + 1 < NV) bits_next = bits_of(j + 1);  // on its way from LDS while this vector is added
        if ((j + 1) * NT > pl.nmain) {
          if (j * NT + t0 >= pl.nmain) d[j] = minus_inf16<T>();
          opaque(d[j]);  // keep the branch: every vector but one is whole
        }
        C f[N];
        unpack<T>(d[j], f);
        run.add(f, bits);
      }
    }
    if (ee >= 0) {
      const int b = ee - bbase;
      if (!(tail && ((bm[b >> 5] >> (b & 31)) & 1u))) run.add1(up<T>(edge));
    }
    if (bad) run.s = (C)NAN;
    // joined over the group
    Sums<C> u = run.joined(), l = Sums<C>::none();
    if (wave * 64 < K) {  // a wave that holds entries
      if constexpr (tail) {
        l = listed.joined();
        nl = wave_sum(nl);
        tmass = wave_sum(tmass);
      } else {
        l.m = wave_max(tm);
        l.s = wave_sum(ts * ex2((tm - l.m) * (C)LOG2E));
      }
    }
    if constexpr (NW > 1) {
      if (lane == 0) {
        sm[wave][0] = u, sm[wave][1] = l;
        if constexpr (tail) smn[wave] = nl, smt[wave] = tmass;
      }
      __syncthreads();
      const Sums<C> p = sm[(lane & 15) % NW][0];
      const bool in = (lane & 15) < NW;
      u.m = row16_max(p.m);
      u.s = row16_sum(in ? p.s * ex2((p.m - u.m) * c) : C(0));
      if constexpr (two) u.s1 = row16_sum(in ? p.s1 * ex2((p.m - u.m) * (C)LOG2E) : C(0));
      l = sm[0][1];
      if constexpr (tail) nl = smn[0], tmass = smt[0];
#pragma clang loop unroll(disable)
      for (int i = 1; i < NW && i * 64 < K; ++i) {
        join<tail && two>(l, sm[i][1], tail ? c : (C)LOG2E);
        if constexpr (tail) nl += smn[i], tmass += smt[i];
      }
    } else {
      group_sync<NT>();
    }
    tm = l.m, ts = l.s;
    const double norm = tail ? lse : uniform((double)tm + (double)(lg2(ts) * (C)LN2));
    const double mass = tail ? tmass : (ts == C(0) ? 0.0 : (double)(ts / ts));
    RowScal<C> rs = row_scalars<C>(a, tail, two, w, y >= 0, u, l, nl, mass);
    rs.M = uniform(rs.M), rs.cB = uniform(rs.cB), rs.cR = uniform(rs.cR), rs.c1 = uniform(rs.c1), rs.ql = uniform(rs.ql), rs.qy = uniform(rs.qy);
    if constexpr (tail) {
      rs.Mu = uniform(rs.Mu), rs.c1u = uniform(rs.c1u);
    } else {
      rs.Mu = rs.M, rs.c1u = rs.c1;
    }
    rs.S = uniform(rs.S), rs.S1 = uniform(rs.S1), rs.Su = uniform(rs.Su), rs.pr = uniform(rs.pr);
    rs.empty = __builtin_amdgcn_readfirstlane(rs.empty);
    const int slot_next = slot == 2 ? 0 : slot + 1;
    if (tid < 2) flags[grp][slot_next == 2 ? 0 : slot_next + 1][tid] = 0;  // the row before this one is through with them
    T x_next, xy_next;
    const int id_next = nrow < a.nrows && tid < K ? checked(id_raw.get(a.ibits)) : -1, y_next = checked(y_raw);
    ask_scores(nrow, id_next, y_next, x_next, xy_next);
    // pass 2
    asm volatile("" : "+s"(ap));
    const bool more = nrow < a.nrows;
    const T* xn = (const T*)a.x + (more ? nrow : row) * a.ldx;
    const P pn(xn, a.V);
    const int en = edge_of(pn), next_main = more ? pn.nmain : 0;
    const __amdgpu_buffer_rsrc_t rg = row_rsrc(gr + pl.h, pl.nmain * 16), rn = row_rsrc(xn + pn.h, next_main * 16);
    T edge_next = (T)0.f;
    if (more && en >= 0) edge_next = xn[en];
    int off = tid * 16;
    opaque(off);  // NV sums that stay out of the row loop's registers
    // For the two-byte types the coefficient goes into the exponent, |cR| exp2((x - Mu) c) = exp2((x - Mu) c + log2 |cR|): an operation
    // a score less.  The logarithm, 100 at most in earnest, is off by 2^-18: 3e-6 of an entry that is then rounded by up to
    // 2^-12 (Float16) of it.
    const C fold = uniform(lg2((C)fabs(rs.cR)));
    const unsigned sign = rs.cR < C(0) ? 0x80008000u : 0u;  // (without an outside class cR is not negative)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      // (stores and loads without a branch: what lies behind a row's end is dropped by the bounds check, and the compiler can
      // count what is in flight -- with branches here it waits for the whole row before the first vector)
      u32x4 out;
      opaque(d[j]);  // or the compiler keeps the unpacked vectors of pass 1, twice the registers
      if (j * NT < pl.nmain) {
        C x[N], o[N];
        unpack<T>(d[j], x);
        if constexpr (sizeof(T) == 2 && !two) {
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] = ex2(fma(x[i] - rs.Mu, c, fold));
          out = pack<T>(o);
          if constexpr (tail) out ^= u32x4{sign, sign, sign, sign};
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) o[i] = ex2((x[i] - rs.Mu) * c);
          if constexpr (two) {
            power(a.squares, x, o, rs.Mu, [&](int i, C v) { o[i] = o[i] * rs.cR + v * rs.c1u; });
          } else {
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] *= rs.cR;
          }
          out = pack<T>(o);
        }
      }
      stb16(rg, off + j * NT * 16, out);
      d[j] = ldb16(rn, off + j * NT * 16);
    }
    if (ee >= 0) gr[ee] = (T)entry_other<two>(rs, up<T>(edge), c);
    asm volatile("" : "+s"(ap));
    const RowLogs<C> lg(a, rs, two);
    // the list's probabilities and its part of the value; its bits go
#pragma clang loop unroll(disable)
    for (int k = tid; k < K; k += NT) {
      const int id = li[k];
      C p = C(0);
      if (id >= 0) {
        const double t = (double)lt[k] * a.invT;
        const C l = t == -INFINITY ? (C)t : (C)(t - norm);  // (a list of -inf only has no norm)
        p = ex2(l * (C)LOG2E);
        if (p != C(0) && !rs.empty && a.lam != 0.0) v_acc += a.lam * w * ((double)p * ((double)l - ((double)(lx[k] - rs.M) * a.invT - (double)lg.ls)));
        bm[((id & ~AGAIN) - bbase) >> 5] = 0;
      }
      lp[k] = p;
    }
    put_list(nrow, id_next, t_next, y_next, x_next, xy_next, par ^ 1, slot_next);
    group_sync<NT>();  // the vectors are written: the listed entries go over them
    const bool dup = flags[grp][slot][0] != 0;
#pragma clang loop unroll(disable)
    for (int k = tid; k < K; k += NT) {
      const int id = li[k];
      if (id < 0 || (id & AGAIN)) continue;
      C ph = lp[k];
      if (dup) {  // a class listed twice: the entry that holds it writes the sum
#pragma clang loop unroll(disable)
        for (int q = 0; q < K; ++q)
          if (li[q] == (id | AGAIN)) ph += lp[q];
      }
      gr[id] = (T)(entry_listed<two>(rs, lx[k], c) - rs.ql * ph - (id == y ? rs.qy : C(0)));
    }
    if (tid == NT - 1) {
      if (y >= 0) {
        const C xy = sxy[grp][par];
        if (!flags[grp][slot][1]) gr[y] = (T)(entry_other<two>(rs, xy, c) - rs.qy);
        if (!rs.empty && a.lab_lam != 0.0) v_acc += a.lab_lam * w * (double)(lg.ls1 - (xy - rs.M));
      }
      if (tail && rs.pr != 0.0 && !rs.empty && a.lam != 0.0) v_acc += a.lam * w * rs.pr * ((double)(lg2((C)rs.pr) * (C)LN2) - lg.log_qr);
      if (rs.S != rs.S) v_acc = NAN;  // a NaN score, or an index or label out of range
    }
    order_list(par ^ 1, slot_next);
    edge = edge_next;
    y = y_next;
    w = w_next;
    row = nrow;
    par ^= 1;
    slot = slot_next;
  }
  double total;
  if (sum_workgroups<G::WG / 64>(v_acc, gridDim.x, blockIdx.x, ap->partials, ap->counter, total)) {
    store_value<C>(total, ap->out, ap->value);
  }
}
#undef a

template <typename T, bool tail, bool two, int NT, int NV>
pg_status run_rows(pg_ctx* c, DArgs a, int64_t rows) {
  using G = RowsGeom<T, NT, NV>;
  const size_t lds = (size_t)G::group_bytes(a.V, a.K) * G::GPW;
  a.acc = c->red_partials + PG_RED_MAX_BLOCKS;
  a.nrows = rows;
  void (*kernel)(DArgs) = distill_rows<T, NT, NV, tail, two>;
  static const int by_registers = [&] {
    int n = 0;
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, G::WG, 0) == hipSuccess ? std::max(n, 1) : 1;
  }();
  const int per_cu = std::min(by_registers, std::max(1, (int)(160 * 1024 / (lds + 1024))));
  const int64_t want = (rows + G::GPW - 1) / G::GPW;
  const int64_t grid = std::min<int64_t>(std::min<int64_t>(want, PG_RED_MAX_BLOCKS), (int64_t)per_cu * c->num_cu);
  kernel<<<(unsigned)grid, G::WG, lds, c->stream>>>(a);
  PG_LAUNCH_CHECK();
  return PG_OK;
}

template <typename T, bool tail, bool two>
pg_status run_mode(pg_ctx* c, const DArgs& a, int64_t rows) {
  const int64_t V = a.V;
  // Few long rows: a workgroup each leaves most of the device idle and takes 11 us for 64 KiB, 19 us for 256 KiB however few they
  // are; in parts 9 us.  At 64 rows of 64 / 256 KiB 10.7 / 16.1 us against 12.7 / 22.2, at 128 rows 11.9 / 24.7 against
  // 13.1 / 23.7, and below 64 KiB a row one launch is the faster at any number (bf16; Float32 of the same bytes alike).
  if (rows <= c->num_cu / 4 && V >= 4096 * Elem<T>::N) return run_parts<T, tail, two>(c, a, rows);
  if (a.K > 0 && !RawReal<typename Elem<T>::C>::takes(a.tdt)) return run_parts<T, tail, two>(c, a, rows);
#define PG_ROWS_TRY(NT, NV)                                                                                                              \
  if (V <= RowsGeom<T, NT, NV>::capacity && RowsGeom<T, NT, NV>::GPW * RowsGeom<T, NT, NV>::group_bytes(a.V, a.K) <= 62 * 1024) \
  return run_rows<T, tail, two, NT, NV>(c, a, rows)
  PG_ROWS_TRY(64, 1);
  PG_ROWS_TRY(64, 2);
  PG_ROWS_TRY(64, 4);
  PG_ROWS_TRY(64, 8);
  PG_ROWS_TRY(256, 4);
  PG_ROWS_TRY(256, 8);
  PG_ROWS_TRY(256, 16);
  PG_ROWS_TRY(512, 16);
  if constexpr (sizeof(T) < 8) PG_ROWS_TRY(1024, 16);
#undef PG_ROWS_TRY
  return run_parts<T, tail, two>(c, a, rows);
}

template <typename T>
pg_status run_t(pg_ctx* c, const DArgs& a, int64_t rows) {
  const bool tail = a.lse != nullptr && a.K > 0, two = a.lab != nullptr && a.invT != 1.0;
  if (tail) return two ? run_mode<T, true, true>(c, a, rows) : run_mode<T, true, false>(c, a, rows);
  return two ? run_mode<T, false, true>(c, a, rows) : run_mode<T, false, false>(c, a, rows);
}

}  // namespace
}  // namespace pgrows
