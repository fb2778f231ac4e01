// Balance of a router's experts, value, counts and gradient (include/proxgrad_hip_rows.h: pg_balance_value_and_gradient).
//
// f = sum_g a_g sum_e c_ge sum_t p_te = sum_g a_g sum_t d_t with d_t = sum_e c_ge p_te, and d_t is what token t's gradient
// a_g p_tj (c_gj - d_t) needs anyhow: the value falls out of the gradient's pass, and the first pass has only to find the
// counts -- integers, so that atomics give the same result in any order, and no exponentials.  Where a group is one
// tile, a workgroup does both passes and the second one finds the scores in the cache.
//
// L lanes take a token, 64 / L tokens a wave: lane l of them holds, in chunk i, the V experts from (i L + l) V on (16 bytes, so that a
// token's chunk is read in one piece).  The k-th highest score is found by bisection over the scores' bit patterns, mapped to
// unsigned numbers in the scores' order: a step counts the keys from a threshold on, whatever k is, all tokens of the wave
// at once, and starts from the thresholds of the wave's tokens before (the first ones from the normal distribution's).  (With a token per wave the search runs in scalar
// registers, on the one scalar unit the CU has: 80 us for 131072 x 256 against 46 with four tokens in vector ones.)
//
// 131072 x 256 f32 (134 MB read twice, 134 written): 94 us, the counting 46 -- 33 with a single step of the search, 7.5 steps of 48
// operations on average --, the gradients 47, 5.7 TB/s.  Small calls are launches and the search of a wave's first tokens: 16384 x 128
// bf16 8 + 8.5 us, 6 of the 8 with a single step.
#include <algorithm>

#include "pg_rows.h"

namespace pgrows {
namespace {

struct BArgs {
  const void* x;
  void* g;
  int64_t ldx, ldg, ldc;
  const pg_balance_tile* tiles;
  const uint8_t* mask;
  const void* chosen;
  int* counts;
  unsigned* state;  // [0] which of the two accumulators this evaluation uses; from [4]: 2 x [groups][copies][experts + 2]
  int64_t groups, ntiles, tokens, tile_tokens;
  unsigned copies;  // of a group's accumulator, taken in turn by its tiles: atomics to one line wait for each other
  int E, k, cbits;
  double lam_e_k;  // lam * experts / k
  float z;         // where a normal distribution has k / experts above
  double *partials, *out;
  unsigned* counter;
  void* value;
};

// ---- order-preserving unsigned keys; 0: never chosen (-inf, NaN) -----------------------------------------------------
template <typename T>
struct Key {
  using U = unsigned;
  static constexpr U top = 0xFFFFu, stride = 1u << 4;  // 16-bit patterns; first step of the search around a guess
  static __device__ __forceinline__ U of(T v) {
    const float f = (float)v;
    const U b = __builtin_bit_cast(unsigned short, v);
    const U k = b & 0x7FFFu ? (b & 0x8000u ? 0xFFFFu - b : b | 0x8000u) : 0x8000u;  // (the two zeros are equal)
    return f > -INFINITY ? k : 0u;
  }
};
template <>
struct Key<float> {
  using U = unsigned;
  static constexpr U top = 0xFFFFFFFFu, stride = 1u << 20;
  static __device__ __forceinline__ U of(float v) {
    const U b = __builtin_bit_cast(unsigned, v + 0.0f);  // (-0 becomes +0: the two are equal)
    const U k = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
    return v > -INFINITY ? k : 0u;
  }
};
template <>
struct Key<double> {
  using U = unsigned long long;
  static constexpr U top = ~0ull, stride = 1ull << 49;
  static __device__ __forceinline__ U of(double v) {
    const U b = __builtin_bit_cast(unsigned long long, v + 0.0);
    const U k = b ^ ((U)((long long)b >> 63) | 0x8000000000000000ull);
    return v > -INFINITY ? k : 0ull;
  }
};

// threads of a workgroup: four waves, so that few tokens are spread over many CUs (the search keeps a CU's issue slots busy: 256
// tokens of 256 experts took 27 us in two workgroups of 1024 threads each); a group of its own workgroup has sixteen
constexpr int BT = 256, BT_WHOLE = 1024;
constexpr unsigned MAX_COPIES = 16;

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) LooseV {
  T v[Elem<T>::N];
};

// the tokens of a wave's step: L lanes each, NI chunks of V experts
template <typename T, int L, int NI>
struct Geom {
  static constexpr int V = Elem<T>::N, PL = NI * V, TW = 64 / L;
  static __device__ __forceinline__ int expert(int i, int j) { return (i * L + (int)(threadIdx.x % L)) * V + j; }
};
// scores of token `tk` (of the last one, t1 - 1, if it lies behind it); -inf behind the last expert
template <typename T, int L, int NI>
struct Scores {
  using G = Geom<T, L, NI>;
  T x[G::PL];
  uint8_t on;
  __device__ __forceinline__ void load(const BArgs& a, int64_t tk, int64_t t1) {
    tk = min(tk, t1 - 1);
    on = a.mask != nullptr ? a.mask[tk] : (uint8_t)1;
    const T* row = (const T*)a.x + tk * a.ldx;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int e = G::expert(i, 0);
      if (e + G::V <= a.E) {
        const LooseV<T> l = *reinterpret_cast<const LooseV<T>*>(row + e);
#pragma unroll
        for (int j = 0; j < G::V; ++j) x[i * G::V + j] = l.v[j];
      } else {
#pragma unroll
        for (int j = 0; j < G::V; ++j) x[i * G::V + j] = e + j < a.E ? row[e + j] : (T)-INFINITY;
      }
    }
  }
};
template <typename T, int L, int NI>
__device__ __forceinline__ void store_scores(T* row, int E, const T (&x)[Geom<T, L, NI>::PL]) {
  using G = Geom<T, L, NI>;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int e = G::expert(i, 0);
    if (e + G::V <= E) {
      LooseV<T> l;
#pragma unroll
      for (int j = 0; j < G::V; ++j) l.v[j] = x[i * G::V + j];
      // non-temporal: nobody reads a gradient here, and the scores, read twice, keep their place in the caches (131072 x 256: 99 us, 106 without)
      typedef u32x4 __attribute__((aligned(2))) Anywhere;
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4, l), reinterpret_cast<Anywhere*>(row + e));
    } else {
#pragma unroll
      for (int j = 0; j < G::V; ++j)
        if (e + j < E) row[e + j] = x[i * G::V + j];
    }
  }
}

// sums and maxima over the L lanes of a token
template <int CTRL>
__device__ __forceinline__ int dpp_int(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
template <int L>
__device__ __forceinline__ int token_sum(int v) {
  if constexpr (L >= 2) v += dpp_int<0xB1>(v);
  if constexpr (L >= 4) v += dpp_int<0x4E>(v);
  if constexpr (L >= 8) v += dpp_int<0x141>(v);
  if constexpr (L >= 16) v += dpp_int<0x140>(v);
  if constexpr (L >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (L >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}
template <int L, typename C>
__device__ __forceinline__ C token_sum(C v) {
  if constexpr (L == 64) return wave_sum(v);
  if constexpr (L >= 2) v += pg_dpp_mov<0xB1>(v);
  if constexpr (L >= 4) v += pg_dpp_mov<0x4E>(v);
  if constexpr (L >= 8) v += pg_dpp_mov<0x141>(v);
  if constexpr (L >= 16) v += pg_dpp_mov<0x140>(v);
  if constexpr (L == 32) v += pg_shfl_xor(v, 16);
  return v;
}
template <int L, typename C>
__device__ __forceinline__ C token_max(C v) {
  if constexpr (L == 64) return wave_max(v);
  if constexpr (L >= 2) v = fmx(v, pg_dpp_mov<0xB1>(v));
  if constexpr (L >= 4) v = fmx(v, pg_dpp_mov<0x4E>(v));
  if constexpr (L >= 8) v = fmx(v, pg_dpp_mov<0x141>(v));
  if constexpr (L >= 16) v = fmx(v, pg_dpp_mov<0x140>(v));
  if constexpr (L == 32) v = fmx(v, pg_shfl_xor(v, 16));
  return v;
}

// cnt[i] += the token chooses this lane's i-th expert.  guess: in, a threshold to start from (above 1); out, this token's.
// A threshold t with more than k keys from it on becomes lo, any other hi; the search ends for a token when exactly k keys lie
// from hi on, or nothing lies between lo and hi.  A step leads away from the guess, four times as far each time, until there is
// a bound on both sides, and then to the middle.  Tokens that have ended go through the others' steps unharmed: their bounds
// only come closer, or, with nothing between, t stays.
template <typename T, int L, int NI>
__device__ __forceinline__ void choose(const T (&x)[Geom<T, L, NI>::PL], bool live, int k, typename Key<T>::U& guess, int (&cnt)[Geom<T, L, NI>::PL]) {
  using U = typename Key<T>::U;
  using G = Geom<T, L, NI>;
  constexpr int PL = G::PL;
  U key[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) key[i] = Key<T>::of(x[i]);
  U lo = 1, hi = Key<T>::top;  // (no key is 1, none is the top)
  U t = guess, step = Key<T>::stride;
  int n_hi = 0;
  bool up_first = false, first = true;
  if (!live) lo = t = hi;  // nothing is chosen
  do {
    int n = 0;
#pragma unroll
    for (int i = 0; i < PL; ++i) n += key[i] >= t;
    n = token_sum<L>(n);
    const bool more = n > k;
    lo = more ? t : lo;
    hi = more ? hi : t;
    n_hi = more ? n_hi : n;
    if (first) up_first = more, first = false;
    const U half = (hi - lo) >> 1;
    step = more == up_first ? step : Key<T>::top;
    const U by = step < half ? step : half;
    step = step > Key<T>::top / 8 ? step : step << 2;
    t = more ? t + by : t - by;
  } while (__any(n_hi != k && hi - lo > 1));
  const int ties = live ? k - n_hi : 0;  // scores equal to lo that are chosen, if not all of them
  if (live) guess = hi;
#pragma unroll
  for (int i = 0; i < PL; ++i) cnt[i] += key[i] >= hi;
  if (__any(ties > 0)) {  // the lowest indices among the equal ones
    const int lane = threadIdx.x & 63;
    const unsigned long long seg = L == 64 ? ~0ull : ((1ull << (L & 63)) - 1) << (lane & ~(L - 1));
    int before = 0;  // equal scores of the token in front of this lane's chunk
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      int lower = 0, all = 0;
#pragma unroll
      for (int j = 0; j < G::V; ++j) {
        const unsigned long long eq = __builtin_amdgcn_ballot_w64(ties > 0 && key[i * G::V + j] == lo) & seg;
        lower += __builtin_popcountll(eq & ((1ull << lane) - 1));
        all += __builtin_popcountll(eq);
      }
      int mine = before + lower;
#pragma unroll
      for (int j = 0; j < G::V; ++j)
        if (ties > 0 && key[i * G::V + j] == lo) cnt[i * G::V + j] += mine++ < ties;
      before += all;
    }
  }
}

__device__ __forceinline__ pg_balance_tile tile_at(const BArgs& a, int64_t q) {
  if (a.tiles != nullptr) return a.tiles[q];
  pg_balance_tile t;
  t.begin = q * a.tile_tokens, t.end = min(t.begin + a.tile_tokens, a.tokens);
  t.group = 0, t.part = (int)q;
  return t;
}

// a threshold for a wave's first tokens to start from: where a normal distribution of the token's mean and variance has k experts above.
// From there the search takes 6 steps, from a fixed number 10; this takes two steps' time (16384 x 128 bf16 in turn 17.1 us against 18.2).
template <typename T, int L, int NI>
__device__ __forceinline__ typename Key<T>::U first_guess(const T (&x)[Geom<T, L, NI>::PL], float z) {
  float n = 0.f, sum = 0.f, sq = 0.f;
#pragma unroll
  for (int i = 0; i < Geom<T, L, NI>::PL; ++i) {
    const float f = (float)x[i];
    const bool in = f > -INFINITY;
    n += in ? 1.f : 0.f;
    const float v = in ? f : 0.f;
    sum += v;
    sq = fma(v, v, sq);
  }
  n = token_sum<L>(n), sum = token_sum<L>(sum), sq = token_sum<L>(sq);
  const float inv = __builtin_amdgcn_rcpf(n), mean = sum * inv;
  const typename Key<T>::U g = Key<T>::of((T)(mean + z * __builtin_amdgcn_sqrtf(fmaxf(sq * inv - mean * mean, 0.f))));
  return g > 1 ? g : Key<T>::of((T)1.0f);  // (no scores, or infinite ones)
}

// choices of the tokens [t0, t1) into sc[experts] (LDS), sc[E] unmasked tokens, sc[E + 1] choices out of range
template <typename T, int L, int NI, int NT>
__device__ __forceinline__ void count_tile(const BArgs& a, int64_t t0, int64_t t1, unsigned* sc) {
  using G = Geom<T, L, NI>;
  constexpr int STEP = NT / L;  // tokens between a wave's steps
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  unsigned live = 0;
  if (a.chosen != nullptr) {
    for (int64_t t = t0 + threadIdx.x; t < t1; t += NT) {
      if (a.mask != nullptr && !a.mask[t]) continue;
      ++live;
      for (int j = 0; j < a.k; ++j) {
        const int64_t e = ld_int(a.chosen, a.cbits, t * a.ldc + j);
        if (e < -1 || e >= a.E) atomicAdd(&sc[a.E + 1], 1u);
        else if (e >= 0) atomicAdd(&sc[e], 1u);
      }
    }
    if (live) atomicAdd(&sc[a.E], live);
    return;
  }
  int cnt[G::PL] = {};
  int64_t t = t0 + wave * G::TW;
  if (t >= t1) return;
  Scores<T, L, NI> s, next;
  s.load(a, t + lane / L, t1);
  next.load(a, t + STEP + lane / L, t1);
  typename Key<T>::U guess = first_guess<T, L, NI>(s.x, a.z);
#pragma clang loop unroll(disable)
  for (;;) {
    const bool on = s.on && t + lane / L < t1;
    live += on;
    choose<T, L, NI>(s.x, on, a.k, guess, cnt);
    t += STEP, s = next;
    if (t >= t1) break;
    next.load(a, t + STEP + lane / L, t1);  // on its way while this one is looked through
  }
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < G::V; ++j)
      if (cnt[i * G::V + j]) atomicAdd(&sc[G::expert(i, j)], (unsigned)cnt[i * G::V + j]);
  if (lane % L == 0 && live) atomicAdd(&sc[a.E], live);
}

// the first tokens of a wave in a tile
template <typename T, int L, int NI>
__device__ __forceinline__ void first_scores(const BArgs& a, int64_t t0, int64_t t1, Scores<T, L, NI>& b) {
  if (t0 + (int64_t)(threadIdx.x / 64) * (64 / L) < t1) b.load(a, t0 + threadIdx.x / L, t1);
}

// gradients of the tokens [t0, t1) from the counts in sc; b: first_scores; returns this thread's part of the value
template <typename T, int L, int NI, int NT>
__device__ __forceinline__ double grad_tile(const BArgs& a, int64_t t0, int64_t t1, const unsigned* sc, Scores<T, L, NI> b) {
  using C = typename Elem<T>::C;
  using G = Geom<T, L, NI>;
  constexpr int PL = G::PL, STEP = NT / L;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  int64_t t = t0 + wave * G::TW;
  if (t >= t1) return 0.0;
  Scores<T, L, NI> next;
  const double n = (double)sc[a.E];
  const double ag = sc[a.E + 1] ? (double)NAN : (n > 0 ? a.lam_e_k / (n * n) : 0.0);
  C c[PL];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < G::V; ++j) c[i * G::V + j] = G::expert(i, j) < a.E ? (C)sc[G::expert(i, j)] : C(0);
  double sum = 0.0;
#pragma clang loop unroll(disable)
  for (; t < t1; t += STEP, b = next) {
    next.load(a, t + STEP + lane / L, t1);
    const int64_t tk = t + lane / L;
    C x[PL], m = Lim<C>::lowest, s = C(0), d = C(0);
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      x[i] = up<T>(b.x[i]);
      m = fmx(m, x[i]);
    }
    m = token_max<L>(m);
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      x[i] = ex2((x[i] - m) * (C)1.4426950408889634);
      s += x[i];
      d += x[i] * c[i];
    }
    s = token_sum<L>(s);
    d = token_sum<L>(d);
    if (tk < t1) {
      const bool on = b.on != 0 && s != C(0);  // (s = 0: every score -inf)
      const C dd = d / s, f = (C)ag / s;
      T o[PL];
#pragma unroll
      for (int i = 0; i < PL; ++i) o[i] = on ? (T)(f * x[i] * (c[i] - dd)) : (T)0.f;
      if (on) sum += ag * (double)dd;
      store_scores<T, L, NI>((T*)a.g + tk * a.ldg, a.E, o);
    }
  }
  return lane % L == 0 ? sum : 0.0;
}

template <typename T, int L, int NI, int NT>
__device__ __forceinline__ void zero_tile(const BArgs& a, int64_t t0, int64_t t1) {
  T o[Geom<T, L, NI>::PL];
#pragma unroll
  for (int i = 0; i < Geom<T, L, NI>::PL; ++i) o[i] = (T)0.f;
  for (int64_t t = t0 + threadIdx.x / L; t < t1; t += NT / L) store_scores<T, L, NI>((T*)a.g + t * a.ldg, a.E, o);
}

template <typename C, int NT>
__device__ __forceinline__ bool finish(const BArgs& a, double v) {
  double total;
  const bool last = sum_workgroups<NT / 64>(v, gridDim.x, blockIdx.x, a.partials, a.counter, total);
  if (last) {
    store_value<C>(total, a.out, a.value);
  }
  return last;
}

// first pass: counts into this evaluation's accumulator
template <typename T, int L, int NI>
__global__ __launch_bounds__(BT) void balance_count(BArgs a) {
  extern __shared__ unsigned sc[];
  const int W = a.E + 2;
  unsigned* acc = a.state + 4 + (size_t)(a.state[0] & 1u) * a.groups * a.copies * W;
  for (int64_t q = blockIdx.x; q < a.ntiles; q += gridDim.x) {
    const pg_balance_tile tl = tile_at(a, q);
    if (tl.group < 0) continue;  // tokens of no group
    for (int i = threadIdx.x; i < W; i += BT) sc[i] = 0;
    __syncthreads();
    count_tile<T, L, NI, BT>(a, tl.begin, tl.end, sc);
    __syncthreads();
    for (int i = threadIdx.x; i < W; i += BT)
      if (sc[i]) atomicAdd(&acc[((size_t)tl.group * a.copies + (unsigned)max(tl.part, 0) % a.copies) * W + i], sc[i]);
    __syncthreads();
  }
}

// second pass: gradients and value; the group's first tile hands the counts out and clears the other accumulator for the
// next evaluation, the last workgroup to finish turns the two over
template <typename T, int L, int NI>
__global__ __launch_bounds__(BT) void balance_grad(BArgs a) {
  extern __shared__ unsigned sc[];
  const int W = a.E + 2;
  const unsigned turn = a.state[0] & 1u;
  const unsigned* acc = a.state + 4 + (size_t)turn * a.groups * a.copies * W;
  unsigned* other = a.state + 4 + (size_t)(turn ^ 1u) * a.groups * a.copies * W;
  double v = 0.0;
  for (int64_t q = blockIdx.x; q < a.ntiles; q += gridDim.x) {
    const pg_balance_tile tl = tile_at(a, q);
    if (tl.group < 0) {
      zero_tile<T, L, NI, BT>(a, tl.begin, tl.end);
      continue;
    }
    Scores<T, L, NI> b;
    first_scores<T, L, NI>(a, tl.begin, tl.end, b);  // on their way while the counts are added up
    for (int i = threadIdx.x; i < W; i += BT) {
      const unsigned* mine = acc + (size_t)tl.group * a.copies * W + i;
      unsigned n = mine[0];
      if (a.copies > 1) {  // all of them asked for at once
#pragma unroll
        for (unsigned p = 1; p < MAX_COPIES; ++p) {
          const unsigned m = mine[(size_t)min(p, a.copies - 1) * W];
          n += p < a.copies ? m : 0u;
        }
      }
      sc[i] = n;
      if (tl.part <= 0) {
        if (i < a.E) a.counts[(size_t)tl.group * a.E + i] = (int)n;
        for (unsigned p = 0; p < a.copies; ++p) other[((size_t)tl.group * a.copies + p) * W + i] = 0;
      }
    }
    __syncthreads();
    v += grad_tile<T, L, NI, BT>(a, tl.begin, tl.end, sc, b);
    __syncthreads();
  }
  if (finish<typename Elem<T>::C, BT>(a, v)) a.state[0] = turn ^ 1u;
}

// both passes, a workgroup per group
template <typename T, int L, int NI>
__global__ __launch_bounds__(BT_WHOLE) void balance_whole(BArgs a) {
  extern __shared__ unsigned sc[];
  const int W = a.E + 2;
  double v = 0.0;
  for (int64_t q = blockIdx.x; q < a.ntiles; q += gridDim.x) {
    const pg_balance_tile tl = tile_at(a, q);
    if (tl.group < 0) {
      zero_tile<T, L, NI, BT_WHOLE>(a, tl.begin, tl.end);
      continue;
    }
    for (int i = threadIdx.x; i < W; i += BT_WHOLE) sc[i] = 0;
    __syncthreads();
    count_tile<T, L, NI, BT_WHOLE>(a, tl.begin, tl.end, sc);
    __syncthreads();
    for (int i = threadIdx.x; i < a.E; i += BT_WHOLE) a.counts[(size_t)tl.group * a.E + i] = (int)sc[i];
    Scores<T, L, NI> b;
    first_scores<T, L, NI>(a, tl.begin, tl.end, b);
    v += grad_tile<T, L, NI, BT_WHOLE>(a, tl.begin, tl.end, sc, b);
    __syncthreads();
  }
  finish<typename Elem<T>::C, BT_WHOLE>(a, v);
}

template <typename T, int L, int NI, int LG, int NG>
pg_status launch(pg_ctx* c, const BArgs& a, bool whole) {
  const size_t lds = (size_t)(a.E + 2) * 4;
  const unsigned grid = (unsigned)std::min<int64_t>(a.ntiles, std::min(8 * c->num_cu, PG_RED_MAX_BLOCKS));
  if (whole) {
    balance_whole<T, L, NI><<<grid, BT_WHOLE, lds, c->stream>>>(a);
    PG_LAUNCH_CHECK();
    return PG_OK;
  }
  balance_count<T, L, NI><<<grid, BT, lds, c->stream>>>(a);
  PG_LAUNCH_CHECK();
  balance_grad<T, LG, NG><<<grid, BT, lds, c->stream>>>(a);
  PG_LAUNCH_CHECK();
  return PG_OK;
}
// A token's lanes.  Counting: at most 16 where that leaves a lane at most 16 scores, so that a wave's step serves four tokens and more; gradients: as many as hold
// the token in one chunk each (a lane's registers are the number of waves that wait for memory).
template <typename T>
pg_status run(pg_ctx* c, const BArgs& a, bool whole) {
  constexpr int V = Elem<T>::N, M = 16 / V;
  if (a.E <= V) return launch<T, 1, 1, 1, 1>(c, a, whole);
  if (a.E <= 2 * V) return launch<T, 2, 1, 2, 1>(c, a, whole);
  if (a.E <= 4 * V) return launch<T, 4, 1, 4, 1>(c, a, whole);
  if (a.E <= 8 * V) return launch<T, 8, 1, 8, 1>(c, a, whole);
  if (a.E <= 16 * V) return launch<T, 16, 1, 16, 1>(c, a, whole);
  if (a.E <= 32 * V) return launch<T, 16, 2, 32, 1>(c, a, whole);
  if constexpr (M >= 4) {
    if (a.E <= 64 * V) return launch<T, 16, 4, 64, 1>(c, a, whole);
  }
  if (a.E <= 32 * M * V) return launch<T, 32, M, 64, M / 2>(c, a, whole);
  return launch<T, 64, M, 64, M>(c, a, whole);
}

__global__ void balance_zero(double* out, void* value, int f64) {
  if (f64) store_value<double>(0.0, out, value);
  else store_value<float>(0.0, out, value);
}

}  // namespace
}  // namespace pgrows

extern "C" pg_status pg_balance_value_and_gradient(pg_ctx* c, const pg_balance* b, int32_t dtype, const void* scores, int64_t ld, void* grad,
                                                   int64_t grad_ld, void* value, double* f_out) {
  using namespace pgrows;
  PG_REQUIRE(c != nullptr && b != nullptr, "null argument");
  PG_REQUIRE(dtype_ok(dtype), "bad dtype");
  PG_REQUIRE(b->tokens >= 0 && b->groups >= 0 && b->ntiles >= 0, "negative size");
  PG_REQUIRE(b->tokens < (1ll << 31), "tokens must be below 2^31");
  PG_REQUIRE(b->experts >= 1 && b->experts <= 1024, "experts must be between 1 and 1024");
  PG_REQUIRE(b->k >= 1 && b->k <= b->experts, "k must be between 1 and the number of experts");
  PG_REQUIRE(b->lam >= 0.0 && std::isfinite(b->lam), "lam must be nonnegative and finite");
  const bool any = b->tokens > 0 && b->ntiles > 0;
  if (any) {
    PG_REQUIRE(scores != nullptr && grad != nullptr, "null rows");
    PG_REQUIRE(b->tiles != nullptr || (b->groups == 1 && b->tile_tokens > 0 && b->ntiles == (b->tokens + b->tile_tokens - 1) / b->tile_tokens),
               "without tiles: one group, ntiles of tile_tokens tokens");
    PG_REQUIRE((b->counts != nullptr || b->groups == 0) && b->state != nullptr, "null plan");
    PG_REQUIRE(b->whole || (b->copies >= 1 && b->copies <= (int)MAX_COPIES), "copies must be between 1 and 16");
    PG_REQUIRE((ld >= b->experts && grad_ld >= b->experts) || b->tokens == 1, "rows overlap: ld below the number of experts");
    PG_REQUIRE(scores != grad || ld == grad_ld || b->tokens == 1, "a gradient in the scores' own buffer needs the scores' ld");
    PG_REQUIRE(((uintptr_t)scores | (uintptr_t)grad) % dtype_size(dtype) == 0, "scores or gradient not aligned to their element");
    PG_REQUIRE(b->chosen == nullptr || b->chosen_bits == 32 || b->chosen_bits == 64, "chosen_bits must be 32 or 64");
  }
  DeviceScope dev(c->device);
  PG_TRY(dev.st);
  PG_TRY(refuse_foreign_capture(c));
  double* out = f_out != nullptr ? c->dscal + PG_S_MISC : nullptr;
  if (!any) {
    balance_zero<<<1, 1, 0, c->stream>>>(out, value, dtype == PG_F64);
    PG_LAUNCH_CHECK();
  } else {
    BArgs a{};
    a.x = scores, a.g = grad, a.ldx = ld, a.ldg = grad_ld, a.ldc = b->chosen_ld;
    a.tiles = b->tiles, a.mask = (const uint8_t*)b->mask, a.chosen = b->chosen, a.counts = b->counts, a.state = b->state;
    a.groups = b->groups, a.ntiles = b->ntiles, a.tokens = b->tokens, a.tile_tokens = b->tile_tokens, a.E = b->experts, a.k = b->k, a.cbits = b->chosen_bits;
    a.copies = (unsigned)b->copies;
    a.lam_e_k = b->lam * b->experts / b->k;
    // (the normal distribution's quantile by the rational approximation 26.2.23 of Abramowitz and Stegun, good to 5e-4)
    const double share = (double)b->k / b->experts, q = std::sqrt(-2.0 * std::log(std::max(std::min(share, 1.0 - share), 1e-4)));
    const double tail = q - (2.515517 + q * (0.802853 + q * 0.010328)) / (1.0 + q * (1.432788 + q * (0.189269 + q * 0.001308)));
    a.z = (float)(share <= 0.5 ? tail : -tail);
    a.partials = c->red_partials, a.out = out, a.counter = c->row_tickets, a.value = value;
    const bool whole = b->whole != 0;
    if (dtype == PG_F32) PG_TRY(run<float>(c, a, whole));
    else if (dtype == PG_F64) PG_TRY(run<double>(c, a, whole));
    else if (dtype == PG_BF16) PG_TRY(run<__bf16>(c, a, whole));
    else PG_TRY(run<_Float16>(c, a, whole));
  }
  if (f_out == nullptr) return PG_OK;
  PG_TRY(pg_read_scalars(c, PG_S_MISC, 1));
  *f_out = c->hscal[PG_S_MISC];
  return PG_OK;
}
