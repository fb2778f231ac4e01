// Balance of a router's experts, value, counts and gradient (include/proxgrad_hip_rows.h: pg_balance_value_and_gradient).
//
// f = sum_g a_g sum_e c_ge sum_t p_te = sum_g a_g sum_t d_t with d_t = sum_e c_ge p_te, and d_t is what token t's gradient
// a_g p_tj (c_gj - d_t) needs anyhow: the value falls out of the gradient's pass, and the first pass has only to find the
// counts -- integers, so that atomics give the same result in any order, and no exponentials.  Where a group is one
// tile, a workgroup does both passes and the second one finds the scores in the cache.
//
// One wave takes a token, lane l its experts l * PL .. l * PL + PL - 1, so that lane order is index order.  The k-th highest
// score is found by bisection over the scores' bit patterns (mapped to unsigned numbers in the scores' order): a step is PL
// compares whose 64-bit masks are counted in scalar registers, whatever k is, and starts from the previous token's threshold.
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
  unsigned* state;  // [0] which of the two accumulators this evaluation uses; from [4]: 2 x [groups][experts + 2]
  int64_t groups, ntiles;
  int E, k, cbits;
  double lam_e_k;  // lam * experts / k
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

template <typename T, int PL>
struct __attribute__((packed, aligned(sizeof(T)))) LooseN {
  T v[PL];
};
// a lane's experts; those behind the last one are -inf
template <typename T, int PL>
__device__ __forceinline__ void load_lane(const T* row, int lane, int E, T (&x)[PL]) {
  const int e0 = lane * PL;
  if (e0 + PL <= E) {
    const LooseN<T, PL> l = *reinterpret_cast<const LooseN<T, PL>*>(row + e0);
#pragma unroll
    for (int i = 0; i < PL; ++i) x[i] = l.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < PL; ++i) x[i] = e0 + i < E ? row[e0 + i] : (T)-INFINITY;
  }
}
template <typename T, int PL>
__device__ __forceinline__ void store_lane(T* row, int lane, int E, const T (&x)[PL]) {
  const int e0 = lane * PL;
  if (e0 + PL <= E) {
    LooseN<T, PL> l;
#pragma unroll
    for (int i = 0; i < PL; ++i) l.v[i] = x[i];
    *reinterpret_cast<LooseN<T, PL>*>(row + e0) = l;
  } else {
#pragma unroll
    for (int i = 0; i < PL; ++i)
      if (e0 + i < E) row[e0 + i] = x[i];
  }
}

// cnt[i] += the token chooses this lane's expert i.  guess: in, a threshold to start from; out, this token's
template <typename T, int PL>
__device__ __forceinline__ void choose(const T (&x)[PL], int k, typename Key<T>::U& guess, int (&cnt)[PL]) {
  using U = typename Key<T>::U;
  U key[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) key[i] = Key<T>::of(x[i]);
  auto count = [&](U t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < PL; ++i) n += __builtin_popcountll(__ballot(key[i] >= t));
    return n;
  };
  U lo = 1, hi = Key<T>::top;  // count(lo) >= k > count(hi)
  int n_hi = 0;
  if (count(1) <= k) {
#pragma unroll
    for (int i = 0; i < PL; ++i) cnt[i] += key[i] != 0;
    return;
  }
  U t = guess, step = Key<T>::stride;
  bool below = false, above = false;  // a bound found on that side of the guess
  while (true) {
    const int n = count(t);
    if (n == k) {
#pragma unroll
      for (int i = 0; i < PL; ++i) cnt[i] += key[i] >= t;
      guess = t;
      return;
    }
    if (n > k) {
      lo = t;
      below = true;
    } else {
      hi = t;
      n_hi = n;
      above = true;
    }
    if (hi - lo <= 1) break;
    if (below && above) {
      t = lo + (hi - lo) / 2;
    } else if (below) {  // widening upwards
      t = hi - lo > step ? lo + step : lo + (hi - lo) / 2;
      step = step > Key<T>::top / 8 ? step : step * 4;
    } else {
      t = hi - lo > step ? hi - step : lo + (hi - lo) / 2;
      step = step > Key<T>::top / 8 ? step : step * 4;
    }
  }
  // several scores equal to lo, not all of them chosen: the lowest indices
  const int lane = threadIdx.x & 63;
  int left = k - n_hi;
  int before = 0;  // equal scores in the lanes in front of this one
#pragma unroll
  for (int i = 0; i < PL; ++i) before += __builtin_popcountll(__ballot(key[i] == lo) & ((1ull << lane) - 1));
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    if (key[i] >= hi) ++cnt[i];
    else if (key[i] == lo) cnt[i] += before++ < left;
  }
  guess = lo;
}

constexpr int BT = 256;

// choices of the tokens [t0, t1) into sc[experts] (LDS), sc[E] unmasked tokens, sc[E + 1] choices out of range
template <typename T, int PL>
__device__ __forceinline__ void count_tile(const BArgs& a, int64_t t0, int64_t t1, unsigned* sc) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (a.chosen != nullptr) {
    unsigned live = 0;
    for (int64_t t = t0 + threadIdx.x; t < t1; t += BT) {
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
  int cnt[PL] = {};
  typename Key<T>::U guess = Key<T>::of((T)1.0f);
  unsigned live = 0;
  for (int64_t t = t0 + wave; t < t1; t += BT / 64) {
    if (a.mask != nullptr && !a.mask[t]) continue;
    ++live;
    T x[PL];
    load_lane<T, PL>((const T*)a.x + t * a.ldx, lane, a.E, x);
    choose<T, PL>(x, a.k, guess, cnt);
  }
#pragma unroll
  for (int i = 0; i < PL; ++i)
    if (cnt[i]) atomicAdd(&sc[lane * PL + i], (unsigned)cnt[i]);
  if (lane == 0 && live) atomicAdd(&sc[a.E], live);
}

// gradients of the tokens [t0, t1) from the counts in sc; returns this thread's part of the value
template <typename T, int PL>
__device__ __forceinline__ double grad_tile(const BArgs& a, int64_t t0, int64_t t1, const unsigned* sc) {
  using C = typename Elem<T>::C;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const double n = (double)sc[a.E];
  const double ag = sc[a.E + 1] ? (double)NAN : (n > 0 ? a.lam_e_k / (n * n) : 0.0);
  C c[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) c[i] = lane * PL + i < a.E ? (C)sc[lane * PL + i] : C(0);
  double sum = 0.0;
  for (int64_t t = t0 + wave; t < t1; t += BT / 64) {
    T* gr = (T*)a.g + t * a.ldg;
    T o[PL];
    C m = Lim<C>::lowest, x[PL];
    const bool live = a.mask == nullptr || a.mask[t];
    if (live) {
      T xt[PL];
      load_lane<T, PL>((const T*)a.x + t * a.ldx, lane, a.E, xt);
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        x[i] = up<T>(xt[i]);
        m = fmx(m, x[i]);
      }
      m = wave_max(m);
      C s = C(0), d = C(0);
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        x[i] = ex2((x[i] - m) * (C)1.4426950408889634);
        s += x[i];
        d += x[i] * c[i];
      }
      s = wave_sum(s);
      d = wave_sum(d);
      if (s != C(0)) {
        d /= s;
        const C f = (C)ag / s;
#pragma unroll
        for (int i = 0; i < PL; ++i) o[i] = (T)(f * x[i] * (c[i] - d));
        sum += ag * (double)d;
        store_lane<T, PL>(gr, lane, a.E, o);
        continue;
      }
    }
#pragma unroll
    for (int i = 0; i < PL; ++i) o[i] = (T)0.f;
    store_lane<T, PL>(gr, lane, a.E, o);
  }
  return lane == 0 ? sum : 0.0;
}

template <typename T, int PL>
__device__ __forceinline__ void zero_tile(const BArgs& a, int64_t t0, int64_t t1) {
  T o[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) o[i] = (T)0.f;
  for (int64_t t = t0 + threadIdx.x / 64; t < t1; t += BT / 64) store_lane<T, PL>((T*)a.g + t * a.ldg, threadIdx.x & 63, a.E, o);
}

template <typename C>
__device__ __forceinline__ bool finish(const BArgs& a, double v) {
  double total;
  const bool last = sum_workgroups<BT / 64>(v, gridDim.x, blockIdx.x, a.partials, a.counter, total);
  if (last) {
    store_value<C>(total, a.out, a.value);
  }
  return last;
}

// first pass: counts into this evaluation's accumulator
template <typename T, int PL>
__global__ __launch_bounds__(BT) void balance_count(BArgs a) {
  extern __shared__ unsigned sc[];
  const int W = a.E + 2;
  unsigned* acc = a.state + 4 + (size_t)(a.state[0] & 1u) * a.groups * W;
  for (int64_t q = blockIdx.x; q < a.ntiles; q += gridDim.x) {
    const pg_balance_tile tl = a.tiles[q];
    if (tl.group < 0) continue;  // tokens of no group
    for (int i = threadIdx.x; i < W; i += BT) sc[i] = 0;
    __syncthreads();
    count_tile<T, PL>(a, tl.begin, tl.end, sc);
    __syncthreads();
    for (int i = threadIdx.x; i < W; i += BT)
      if (sc[i]) atomicAdd(&acc[(size_t)tl.group * W + i], sc[i]);
    __syncthreads();
  }
}

// second pass: gradients and value; the group's first tile hands the counts out and clears the other accumulator for the
// next evaluation, the last workgroup to finish turns the two over
template <typename T, int PL>
__global__ __launch_bounds__(BT) void balance_grad(BArgs a) {
  extern __shared__ unsigned sc[];
  const int W = a.E + 2;
  const unsigned turn = a.state[0] & 1u;
  const unsigned* acc = a.state + 4 + (size_t)turn * a.groups * W;
  unsigned* other = a.state + 4 + (size_t)(turn ^ 1u) * a.groups * W;
  double v = 0.0;
  for (int64_t q = blockIdx.x; q < a.ntiles; q += gridDim.x) {
    const pg_balance_tile tl = a.tiles[q];
    if (tl.group < 0) {
      zero_tile<T, PL>(a, tl.begin, tl.end);
      continue;
    }
    for (int i = threadIdx.x; i < W; i += BT) {
      const unsigned n = acc[(size_t)tl.group * W + i];
      sc[i] = n;
      if (tl.part <= 0) {
        if (i < a.E) a.counts[(size_t)tl.group * a.E + i] = (int)n;
        other[(size_t)tl.group * W + i] = 0;
      }
    }
    __syncthreads();
    v += grad_tile<T, PL>(a, tl.begin, tl.end, sc);
    __syncthreads();
  }
  if (finish<typename Elem<T>::C>(a, v)) a.state[0] = turn ^ 1u;
}

// both passes, a workgroup per group
template <typename T, int PL>
__global__ __launch_bounds__(BT) void balance_whole(BArgs a) {
  extern __shared__ unsigned sc[];
  const int W = a.E + 2;
  double v = 0.0;
  for (int64_t q = blockIdx.x; q < a.ntiles; q += gridDim.x) {
    const pg_balance_tile tl = a.tiles[q];
    if (tl.group < 0) {
      zero_tile<T, PL>(a, tl.begin, tl.end);
      continue;
    }
    for (int i = threadIdx.x; i < W; i += BT) sc[i] = 0;
    __syncthreads();
    count_tile<T, PL>(a, tl.begin, tl.end, sc);
    __syncthreads();
    for (int i = threadIdx.x; i < a.E; i += BT) a.counts[(size_t)tl.group * a.E + i] = (int)sc[i];
    v += grad_tile<T, PL>(a, tl.begin, tl.end, sc);
    __syncthreads();
  }
  finish<typename Elem<T>::C>(a, v);
}

template <typename T, int PL>
pg_status launch(pg_ctx* c, const BArgs& a, bool whole) {
  const size_t lds = (size_t)(a.E + 2) * 4;
  const unsigned grid = (unsigned)std::min<int64_t>(a.ntiles, std::min(8 * c->num_cu, PG_RED_MAX_BLOCKS));
  if (whole) {
    balance_whole<T, PL><<<grid, BT, lds, c->stream>>>(a);
    PG_LAUNCH_CHECK();
    return PG_OK;
  }
  balance_count<T, PL><<<grid, BT, lds, c->stream>>>(a);
  PG_LAUNCH_CHECK();
  balance_grad<T, PL><<<grid, BT, lds, c->stream>>>(a);
  PG_LAUNCH_CHECK();
  return PG_OK;
}
template <typename T>
pg_status run(pg_ctx* c, const BArgs& a, bool whole) {
  if (a.E <= 64) return launch<T, 1>(c, a, whole);
  if (a.E <= 128) return launch<T, 2>(c, a, whole);
  if (a.E <= 256) return launch<T, 4>(c, a, whole);
  if (a.E <= 512) return launch<T, 8>(c, a, whole);
  return launch<T, 16>(c, a, whole);
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
    PG_REQUIRE(b->tiles != nullptr && (b->counts != nullptr || b->groups == 0) && b->state != nullptr, "null plan");
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
    a.groups = b->groups, a.ntiles = b->ntiles, a.E = b->experts, a.k = b->k, a.cbits = b->chosen_bits;
    a.lam_e_k = b->lam * b->experts / b->k;
    a.partials = c->red_partials, a.out = out, a.counter = c->red_counter, a.value = value;
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
