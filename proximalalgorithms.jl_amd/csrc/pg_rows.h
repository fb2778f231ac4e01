// Pieces shared by the losses on rows of scores (pg_rows_distill.hip, pg_rows_balance.hip): element types, 16-byte vectors of
// them, reductions over a wave and over a workgroup.
#pragma once
#include "pg_internal.h"
#include "proxgrad_hip_rows.h"

namespace pgrows {

// ---- host ----
inline bool dtype_ok(int dt) { return dt == PG_F32 || dt == PG_F64 || dt == PG_BF16 || dt == PG_F16; }
inline int dtype_size(int dt) { return dt == PG_F64 ? 8 : (dt == PG_F32 ? 4 : 2); }

// A context's device for the length of a call (the caller's current device may be another one)
struct DeviceScope {
  int prev = -1;
  bool changed = false;
  pg_status st = PG_OK;
  explicit DeviceScope(int device) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != device) {
      if (hipSetDevice(device) != hipSuccess) {
        pg_set_error("hipSetDevice(%d) failed", device);
        st = PG_ERR_HIP;
      } else {
        changed = true;
      }
    }
  }
  ~DeviceScope() {
    if (changed && prev >= 0) (void)hipSetDevice(prev);
  }
};

// The context's workspaces are ordered by its stream; a graph that somebody else records from that stream could be replayed next to it
inline pg_status refuse_foreign_capture(pg_ctx* c) {
  if (c->capturing) return PG_OK;
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  const hipError_t e = hipStreamIsCapturing(c->stream, &cs);
  if (e != hipSuccess) (void)hipGetLastError();
  if (e != hipSuccess || cs != hipStreamCaptureStatusNone) {
    pg_set_error("the context's stream is being captured by somebody else: record with pg_ctx_capture_begin / pg_ctx_capture_end");
    return PG_ERR_UNSUPPORTED;
  }
  return PG_OK;
}

#ifdef __HIPCC__
// ---- device ----
template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Elem;  // compute type, elements per 16 bytes
template <>
struct Elem<float> {
  using C = float;
  static constexpr int N = 4;
};
template <>
struct Elem<double> {
  using C = double;
  static constexpr int N = 2;
};
template <>
struct Elem<__bf16> {
  using C = float;
  static constexpr int N = 8;
};
template <>
struct Elem<_Float16> {
  using C = float;
  static constexpr int N = 8;
};

template <typename T>
__device__ __forceinline__ typename Elem<T>::C up(T v) {
  return (typename Elem<T>::C)v;
}
// 16 bytes at an address that is a multiple of the element's size only: one dwordx4 access on gfx950 (unaligned access mode)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
  u32x4 v;
};
template <typename T>
__device__ __forceinline__ u32x4 ld16(const T* p) {
  return reinterpret_cast<const Loose<T>*>(p)->v;
}
template <typename T>
__device__ __forceinline__ void st16(T* p, u32x4 v) {
  reinterpret_cast<Loose<T>*>(p)->v = v;
}
// vector v of a row: a wave-uniform base and a 32-bit offset (a row is at most 2^24 elements of at most 8 bytes)
template <typename T>
__device__ __forceinline__ T* at16(T* base, int v) {
  return (T*)((const char*)base + (uint64_t)(unsigned)v * 16u);  // (through char*: an integer would lose the address space)
}
// A row as a buffer resource: base and length in scalar registers, one 32-bit offset per lane; a load behind the end gives 0, a
// store behind it is dropped (the hardware's bounds check), so no vector needs a mask or a 64-bit address of its own.
// Both non-temporal (the last argument): a score is read once and a gradient is not read here at all; on 2 x 512 MiB that is
// 103 us against 124 with neither, 119 with the stores and 127 with the loads alone.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000);
}
__device__ __forceinline__ u32x4 ldb16(__amdgpu_buffer_rsrc_t r, int byte) { return __builtin_amdgcn_raw_buffer_load_b128(r, byte, 0, 2); }
__device__ __forceinline__ void stb16(__amdgpu_buffer_rsrc_t r, int byte, u32x4 v) { __builtin_amdgcn_raw_buffer_store_b128(v, r, byte, 0, 2); }
// 16 bytes of -inf
template <typename T>
__device__ __forceinline__ u32x4 minus_inf16() {
  vec<T, Elem<T>::N> e;
#pragma unroll
  for (int i = 0; i < Elem<T>::N; ++i) e[i] = (T)-INFINITY;
  return __builtin_bit_cast(u32x4, e);
}
// a value the compiler knows nothing about any more
__device__ __forceinline__ void opaque(int& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void opaque(float& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void opaque(double& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void opaque(u32x4& v) { asm volatile("" : "+v"(v)); }
template <typename T>
__device__ __forceinline__ void unpack(u32x4 u, typename Elem<T>::C (&f)[Elem<T>::N]) {
  using VT = vec<T, Elem<T>::N>;
  const VT e = __builtin_bit_cast(VT, u);
#pragma unroll
  for (int i = 0; i < Elem<T>::N; ++i) f[i] = (typename Elem<T>::C)e[i];
}
template <typename T>
__device__ __forceinline__ u32x4 pack(const typename Elem<T>::C (&f)[Elem<T>::N]) {
  vec<T, Elem<T>::N> e;
#pragma unroll
  for (int i = 0; i < Elem<T>::N; ++i) e[i] = (T)f[i];  // the one rounding of a gradient entry
  return __builtin_bit_cast(u32x4, e);
}

__device__ __forceinline__ double ld_real(const void* p, int dt, int64_t i) {
  switch (dt) {
    case PG_F64: return ((const double*)p)[i];
    case PG_F32: return (double)((const float*)p)[i];
    case PG_BF16: return (double)(float)((const __bf16*)p)[i];
    default: return (double)(float)((const _Float16*)p)[i];
  }
}
// the same in two steps: loads whose results nothing looks at yet (a conversion beside them would wait for them, and so would two
// kinds of load into one register), and the conversion.  Two loads each, whatever the type: of the element's halves, or twice the same
template <typename C>
struct RawReal {  // C = float: of 2 or 4 bytes; C = double: of 8
  unsigned a, b;
  __device__ __forceinline__ void load(const void* p, int dt, int64_t i) {
    if constexpr (sizeof(C) == 8) {
      const uint2 v = ((const uint2*)p)[i];
      a = v.x, b = v.y;
    } else {
      const int h = dt == PG_F32 ? 1 : 0;  // halves behind the first
      const unsigned short* q = (const unsigned short*)p + (i << h);
      a = q[0], b = q[h];
    }
  }
  __device__ __forceinline__ C get(int dt) const {
    if constexpr (sizeof(C) == 8) {
      return __builtin_bit_cast(double, make_uint2(a, b));
    } else {
      return dt == PG_F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)a) : __builtin_bit_cast(float, dt == PG_F32 ? a | b << 16 : a << 16);
    }
  }
  static bool takes(int dt) { return (dt == PG_F64) == (sizeof(C) == 8); }
};
struct RawInt {
  unsigned a, b;
  __device__ __forceinline__ void load(const void* p, int bits, int64_t i) {
    const int h = bits == 64 ? 1 : 0;
    const unsigned* q = (const unsigned*)p + (i << h);
    a = q[0], b = q[h];
  }
  __device__ __forceinline__ int64_t get(int bits) const { return bits == 64 ? (int64_t)(((unsigned long long)b << 32) | a) : (int64_t)(int)a; }
};
__device__ __forceinline__ int64_t ld_int(const void* p, int bits, int64_t i) {
  return bits == 64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// the same for what is the same in every lane and never written by the kernel that reads it (one value per row): scalar loads
#define PG_CONST_AS __attribute__((address_space(4)))
__device__ __forceinline__ double ld_real_u(const void* p, int dt, int64_t i) {  // PG_F32 or PG_F64
  return dt == PG_F64 ? ((const PG_CONST_AS double*)p)[i] : (double)((const PG_CONST_AS float*)p)[i];
}
__device__ __forceinline__ int64_t ld_int_u(const void* p, int bits, int64_t i) {
  return bits == 64 ? ((const PG_CONST_AS int64_t*)p)[i] : (int64_t)((const PG_CONST_AS int32_t*)p)[i];
}
__device__ __forceinline__ float uniform(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ double uniform(double v) { return pg_readlane(v, 0); }

// (one instruction; results below 2^-126 are 0: an exponent of 20 below the largest's, 2^-97 of it)
__device__ __forceinline__ float ex2(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ double ex2(double v);  // below
__device__ __forceinline__ float lg2(float v) { return __builtin_amdgcn_logf(v); }
__device__ __forceinline__ double lg2(double v) { return log2(v); }
// exp in Float64 from its series: argument n ln 2 + r, |r| <= ln(2) / 2, sum of r^k / k! up to k = 13 (the next term is below 2^-56
// of the sum), times 2^n.  The library's exp and exp2 inside a loop keep their constants in some forty vector registers around
// the loop, which a kernel that holds a row in registers has not got: the compiler moved them to and fro, and in one of its
// builds lanes lost a coefficient on the way (sums off by 1e-11).  Here they pass through scalar registers where they are used.
__device__ __forceinline__ double scalar_const(double v) {
  asm volatile("" : "+s"(v));
  return v;
}
__device__ __forceinline__ double exp_sum(double r) {
  double p = scalar_const(1.0 / 6227020800.0);
  p = fma(p, r, scalar_const(1.0 / 479001600.0));
  p = fma(p, r, scalar_const(1.0 / 39916800.0));
  p = fma(p, r, scalar_const(1.0 / 3628800.0));
  p = fma(p, r, scalar_const(1.0 / 362880.0));
  p = fma(p, r, scalar_const(1.0 / 40320.0));
  p = fma(p, r, scalar_const(1.0 / 5040.0));
  p = fma(p, r, scalar_const(1.0 / 720.0));
  p = fma(p, r, scalar_const(1.0 / 120.0));
  p = fma(p, r, scalar_const(1.0 / 24.0));
  p = fma(p, r, scalar_const(1.0 / 6.0));
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  return fma(p, r, 1.0);
}
__device__ __forceinline__ double exp_scale(double p, double n) { return ldexp(p, (int)fmax(fmin(n, 2000.0), -2000.0)); }
__device__ __forceinline__ double exp_series(double x) {
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, scalar_const(-0x1.62e42fefa38p-1), x);  // ln 2 in two pieces, the first with zeros at its end
  r = fma(n, scalar_const(-0x1.ef35793c7673p-45), r);
  return x < -745.2 ? 0.0 : (x > 709.8 ? (double)INFINITY : exp_scale(exp_sum(r), n));  // (NaN stays NaN)
}
__device__ __forceinline__ double ex2(double x) {
  const double n = rint(x);
  return x < -1080.0 ? 0.0 : (x > 1030.0 ? (double)INFINITY : exp_scale(exp_sum((x - n) * scalar_const(0x1.62e42fefa39efp-1)), n));
}

template <typename C>
struct Lim;
template <>
struct Lim<float> {
  static constexpr float lowest = -3.402823466e+38f;
};
template <>
struct Lim<double> {
  static constexpr double lowest = -1.7976931348623157e+308;
};

template <typename C>
__device__ __forceinline__ C wave_sum(C v) {
  return pg_wave_allreduce<false, C>(v);
}
__device__ __forceinline__ float fmx(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double fmx(double a, double b) { return fmax(a, b); }
// maximum over the 16 lanes of a DPP row / over the wave, NaN passed over (the sums carry it)
template <typename C>
__device__ __forceinline__ C row16_max(C v) {
  v = fmx(v, pg_dpp_mov<0xB1>(v));
  v = fmx(v, pg_dpp_mov<0x4E>(v));
  v = fmx(v, pg_dpp_mov<0x141>(v));
  return fmx(v, pg_dpp_mov<0x140>(v));
}
template <typename C>
__device__ __forceinline__ C wave_max(C v) {
  v = row16_max(v);
  return fmx(fmx(pg_readlane(v, 0), pg_readlane(v, 16)), fmx(pg_readlane(v, 32), pg_readlane(v, 48)));
}
template <typename C>
__device__ __forceinline__ C row16_sum(C v) {
  return pg_row_allreduce<false, C>(v);
}

// The sum of one Float64 per thread over `n` workgroups of NW waves, of which this is number `me`; every thread of each calls it.
// Each publishes its own sum with a write-through store and takes a ticket; the last one adds them in their order (the same
// result whoever is last) and puts the tickets back.  True, with the total, for thread 0 of the last one.  Tickets of one line
// are handed out one after the other, some 12 ns each, so the workgroups draw from 32 lines and the last of each line from one more.
constexpr int TICKET_LINES = 32, TICKET_PITCH = 32;
template <int NW>
__device__ __forceinline__ bool sum_workgroups(double v, unsigned n, unsigned me, double* partials, unsigned* tickets, double& total) {
  __shared__ double sw[NW];
  __shared__ int is_last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto join = [&](double x) {
    x = wave_sum(x);
    if (lane == 0) sw[wave] = x;
    __syncthreads();
    double t = sw[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) t += sw[i];
    return t;
  };
  const double mine = join(v);
  if (n == 1) {
    total = mine;
    return threadIdx.x == 0;
  }
  if (threadIdx.x == 0) {
    __hip_atomic_store(&partials[me], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const unsigned line = me % TICKET_LINES, members = (n - line + TICKET_LINES - 1) / TICKET_LINES;
    unsigned* t = tickets + (1 + line) * TICKET_PITCH;
    bool last = __hip_atomic_fetch_add(t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == members - 1;
    if (last) {
      __hip_atomic_store(t, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const unsigned lines = n < TICKET_LINES ? n : TICKET_LINES;
      last = __hip_atomic_fetch_add(tickets, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == lines - 1;
      if (last) __hip_atomic_store(tickets, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    is_last = last;
  }
  __syncthreads();
  if (!is_last) return false;
  double acc = 0.0;
  for (unsigned i = threadIdx.x; i < n; i += NW * 64) acc += __hip_atomic_load(&partials[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  total = join(acc);
  return threadIdx.x == 0;
}

// the value where it was asked for: the context's scalar block (host memory) and the caller's device scalar
template <typename C>
__device__ __forceinline__ void store_value(double v, double* out, void* value) {
  if (out != nullptr) *out = v;
  if (value != nullptr) *(C*)value = (C)v;
}

// NT threads of one workgroup work on a row: all of it (a workgroup's barrier) or one wave of it (its LDS accesses are in order)
template <int NT>
__device__ __forceinline__ void group_sync() {
  if constexpr (NT == 64) {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}
#endif  // __HIPCC__

}  // namespace pgrows
