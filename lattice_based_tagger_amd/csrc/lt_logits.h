// lt_logits.h -- what the operators over logits share (lt_top.hip,
// lt_distill.hip, lt_verify.hip): element types, rows, block reductions, and
// the host's checks and launches.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/lattice_logits.h"
#include "lt_error.h"

namespace {

constexpr int MAXK = LT_MAX_TOP;
constexpr float LOWEST = -3.4028234663852886e38f;
constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;

struct Rows {
  const void* data;
  int64_t inner, stride_outer, stride_inner;
  int32_t vocab;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    return inner == 1 ? r * stride_outer : (r / inner) * stride_outer + (r % inner) * stride_inner;
  }
};

struct F32 {
  static constexpr float lowest = -3.4028234663852886e38f;
  using raw = float;
  static __device__ __forceinline__ float get(raw v) { return v; }
  static __device__ __forceinline__ raw put(float v) { return v; }
};
struct F16 {
  static constexpr float lowest = -65504.f;
  using raw = uint16_t;
  static __device__ __forceinline__ float get(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ raw put(float v) { return __builtin_bit_cast(raw, (_Float16)v); }
};
struct BF16 {
  static constexpr float lowest = -3.3895313892515355e38f;
  using raw = uint16_t;
  static __device__ __forceinline__ float get(raw v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
  static __device__ __forceinline__ raw put(float v) { return __builtin_bit_cast(raw, (__bf16)v); }
};

// 16 bytes of a row, at any address its type allows (the loads and stores are
// single ones: global memory takes them unaligned).
struct __attribute__((packed, aligned(2))) Bytes16 {
  uint32_t w[4];
};

typedef uint32_t Words16 __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ uint32_t twice(float v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ uint32_t bits_of(float v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ uint32_t bits_of(uint16_t v) { return v; }
__device__ __forceinline__ uint32_t twice(uint16_t v) { return (uint32_t)v << 16 | v; }

// The E = 16 / sizeof(raw) logits of a vector.
template <class T>
struct Vec {
  static constexpr int E = 16 / sizeof(typename T::raw);
  Bytes16 b;
  __device__ __forceinline__ void load(const typename T::raw* p) { b = *(const Bytes16*)p; }
  __device__ __forceinline__ void store(typename T::raw* p) const { *(Bytes16*)p = b; }
  // The same past the caches: what is read or written for the last time.
  __device__ __forceinline__ void load_last(const typename T::raw* p) {
    const Words16 w = __builtin_nontemporal_load((const Words16*)p);
    for (int i = 0; i < 4; ++i) b.w[i] = w[i];
  }
  __device__ __forceinline__ void store_past(typename T::raw* p) const {
    // (the fences of asm: of this store and a plain one in the branches of an
    // if, the compiler makes one plain store)
    asm volatile("" ::: "memory");
    __builtin_nontemporal_store(Words16{b.w[0], b.w[1], b.w[2], b.w[3]}, (Words16*)p);
    asm volatile("" ::: "memory");
  }
  __device__ __forceinline__ float get(int i) const;
  // Rounded to the type, to the nearest.
  __device__ __forceinline__ void put(const float* f) {
    if constexpr (E == 4) {
      for (int i = 0; i < 4; ++i) b.w[i] = __builtin_bit_cast(uint32_t, f[i]);
    } else {
      for (int i = 0; i < 4; ++i) b.w[i] = (uint32_t)T::put(f[2 * i]) | (uint32_t)T::put(f[2 * i + 1]) << 16;
    }
  }
  // What lies in [begin, end) of the vector that belongs at `at`.
  __device__ __forceinline__ void store_part(typename T::raw* x, int at, int begin, int end) const {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (at + i >= begin && at + i < end) {
        if constexpr (E == 4) x[at + i] = __builtin_bit_cast(float, b.w[i]);
        else x[at + i] = (typename T::raw)(b.w[i >> 1] >> (i & 1) * 16);
      }
  }
  // -inf for the logits whose bits are set.
  __device__ __forceinline__ void mask(uint32_t bits) {
    auto all = [&](int i) { return (uint32_t)((int)(bits << (31 - i)) >> 31); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = E == 4 ? all(i) : (all(2 * i) & 0xffffu) | (all(2 * i + 1) & 0xffff0000u);
      b.w[i] = (b.w[i] & ~m) | (twice(T::put(-INFINITY)) & m);
    }
  }
  // What is computed from the logits ahead of this is not kept for later.
  __device__ __forceinline__ void keep() { asm volatile("" : "+v"(b.w[0]), "+v"(b.w[1]), "+v"(b.w[2]), "+v"(b.w[3])); }
  // The vector at `at` of logits that lie in [begin, end), `fill` around them.
  // One that holds one of their ends is the whole vector beside it, shifted.
  __device__ __forceinline__ void load(const typename T::raw* x, int at, int begin, int end, typename T::raw fill) {
    if (!load_inner(x, at, begin, end, fill)) load_edge(x, at, begin, end, fill);
  }
  // The same; false where the vector holds an end (it is `fill` then).
  __device__ __forceinline__ bool load_inner(const typename T::raw* x, int at, int begin, int end, typename T::raw fill) {
    b.w[0] = b.w[1] = b.w[2] = b.w[3] = twice(fill);
    if (at >= begin && at + E <= end) load(x + at);
    else if (at < end && at + E > begin) return false;
    return true;
  }
  __device__ __forceinline__ void load_edge(const typename T::raw* x, int at, int begin, int end, typename T::raw fill) {
    constexpr int BITS = 8 * sizeof(typename T::raw);
    const uint64_t f = (uint64_t)twice(fill) << 32 | twice(fill);
    uint64_t lo, hi;
    if (end - begin < E) {                 // a row of less than a vector
      lo = hi = f;
#pragma nounroll
      for (int i = max(at, begin); i < min(at + E, end); ++i) {
        const int by = (i - at) * BITS;
        const uint64_t field = (~0ull >> (64 - BITS)) << (by & 63), v = (uint64_t)bits_of(x[i]) << (by & 63);
        if (by < 64) lo = (lo & ~field) | v;
        else hi = (hi & ~field) | v;
      }
    } else {
      const bool head = at < begin;
      load(x + (head ? begin : end - E));
      lo = (uint64_t)b.w[1] << 32 | b.w[0];
      hi = (uint64_t)b.w[3] << 32 | b.w[2];
      int by = (head ? begin - at : at + E - end) * BITS;      // 0 < by < 128
      if (by >= 64) {
        by -= 64;
        if (head) hi = lo, lo = f;
        else lo = hi, hi = f;
      }
      if (by) {
        if (head) {
          hi = hi << by | lo >> (64 - by);
          lo = lo << by | f >> (64 - by);
        } else {
          lo = lo >> by | hi << (64 - by);
          hi = hi >> by | f << (64 - by);
        }
      }
    }
    b.w[0] = (uint32_t)lo;
    b.w[1] = (uint32_t)(lo >> 32);
    b.w[2] = (uint32_t)hi;
    b.w[3] = (uint32_t)(hi >> 32);
  }
};
template <>
__device__ __forceinline__ float Vec<F32>::get(int i) const {
  return __builtin_bit_cast(float, b.w[i]);
}
template <>
__device__ __forceinline__ float Vec<F16>::get(int i) const {
  return F16::get((uint16_t)(b.w[i >> 1] >> (i & 1) * 16));
}
template <>
__device__ __forceinline__ float Vec<BF16>::get(int i) const {
  return __builtin_bit_cast(float, i & 1 ? b.w[i >> 1] & 0xffff0000u : b.w[i >> 1] << 16);
}

// A step's vectors of a thread: U of them, NT vectors apart from `base` on, of
// logits in [begin, end); LAST: past the caches.
template <class T, int NT, int U, bool LAST = false>
__device__ __forceinline__ void load_step(Vec<T> (&v)[U], const typename T::raw* x, int base, int tid, int begin, int end) {
  constexpr int E = Vec<T>::E;
  if (base >= begin && base + NT * U * E <= end) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (LAST) v[u].load_last(x + base + (u * NT + tid) * E);
      else v[u].load(x + base + (u * NT + tid) * E);
    }
    return;
  }
  const typename T::raw fill = T::put(-INFINITY);
  uint32_t edges = 0;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (!v[u].load_inner(x, base + (u * NT + tid) * E, begin, end, fill)) edges |= 1u << u;
  // (one copy of this for all u, and that once: else it takes 40 registers)
#pragma nounroll
  while (edges) {
    const int at = __builtin_ctz(edges);
    edges &= edges - 1;
    Vec<T> e;
    e.load_edge(x, base + (at * NT + tid) * E, begin, end, fill);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u].b.w[i] = u == at ? e.b.w[i] : v[u].b.w[i];
  }
}

// Leaves the IEEE mode (bit 9 of the mode register), ahead of a kernel's maxima over
// logits.  (In lt_verify_sums it costs 7 % at its start.)
__device__ __forceinline__ void numbers_win() { __builtin_amdgcn_s_setreg(1 | 9 << 6, 0); }

// The larger of two, of three; a NaN gives way to a number -- a signalling one only
// behind numbers_win(): in the IEEE mode that a kernel starts in, the instructions
// return it, quieted, and with three operands lose the one beside it.
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
template <class T>
__device__ __forceinline__ float max_of(const Vec<T>& v) {
  if constexpr (Vec<T>::E == 4) return max2(max3(v.get(0), v.get(1), v.get(2)), v.get(3));
  else return max3(max3(max3(v.get(0), v.get(1), v.get(2)), v.get(3), v.get(4)), max2(v.get(5), v.get(6)), v.get(7));
}

// A single logit in a vector's place.
template <class T>
struct One {
  static constexpr int E = 1;
  float f;
  __device__ __forceinline__ void load(const typename T::raw* p) { f = T::get(*p); }
  __device__ __forceinline__ void load(const typename T::raw* x, int at, int, int end, typename T::raw) {
    f = at < end ? T::get(x[at]) : -INFINITY;
  }
  __device__ __forceinline__ void mask(uint32_t bits) { f = bits & 1 ? -INFINITY : f; }
  __device__ __forceinline__ float get(int) const { return f; }
  __device__ __forceinline__ void keep() {}
};
template <class T>
__device__ __forceinline__ float max_of(const One<T>& v) {
  return v.f;
}

// 2^x of the hardware: within an ulp, 0 below the normal numbers.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^t for -1020 < t < 1020: 2^n 2^f, n the whole number next to t, 2^f by the
// polynomial of degree 8 through its values at the Chebyshev points of
// [-1/2, 1/2] (relative error at most 1.1e-12; the series needs degree 10 for
// that).  n is added to the exponent's bits.
__device__ __forceinline__ double exp2_64(double t) {
  constexpr double BIG = 6755399441055744.0;       // 1.5 * 2^52: its last bits are whole numbers
  const double b = t + BIG;
  const double f = t - (b - BIG);
  double r = 1.325497460306718e-06;
  r = fma(r, f, 1.531007807039615e-05);
  r = fma(r, f, 0.00015403457039410448);
  r = fma(r, f, 0.0013333450573018062);
  r = fma(r, f, 0.009618129157656703);
  r = fma(r, f, 0.055504109412010456);
  r = fma(r, f, 0.24022650695821055);
  r = fma(r, f, 0.6931471805459343);
  r = fma(r, f, 0.9999999999999997);
  const uint64_t bits = __builtin_bit_cast(uint64_t, r);
  const uint32_t hi = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, b) << 20);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)bits);
}

// log2 of a sum in 32 bits, good to 2^-23 absolutely (the hardware's logarithm
// of the whole would be good to 2^-23 of its value, up to 30 here).
__device__ __forceinline__ double log2_(float s) {
  return (double)__builtin_amdgcn_frexp_expf(s) + (double)__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(s));
}

__device__ __forceinline__ float any_float(const void* p, int64_t i, int dtype) {
  if (dtype == LT_F32) return ((const float*)p)[i];
  return dtype == LT_F16 ? F16::get(((const uint16_t*)p)[i]) : BF16::get(((const uint16_t*)p)[i]);
}

__device__ __forceinline__ int64_t any_id(const void* p, int64_t i, int bytes) {
  return bytes == 8 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// ---- reductions of a block -------------------------------------------------
struct Max {
  template <class T>
  static __device__ __forceinline__ T of(T a, T b) { return a > b ? a : b; }
  static __device__ __forceinline__ float of(float a, float b) { return max2(a, b); }
};
struct Sum {
  template <class T>
  static __device__ __forceinline__ T of(T a, T b) { return a + b; }
};

// v of another lane by a data-parallel-primitives control word, `other` where
// there is none (in steps of 32 bits).
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp(T v, T other) {
  constexpr int N = sizeof(T) / 4;
  struct Words { int w[N]; };
  Words a = __builtin_bit_cast(Words, v), o = __builtin_bit_cast(Words, other);
#pragma unroll
  for (int i = 0; i < N; ++i) a.w[i] = __builtin_amdgcn_update_dpp(o.w[i], a.w[i], CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(T, a);
}

// Op over the lanes up to each one (0 .. lane), `none` being Op's neutral value.
template <class Op, class T>
__device__ __forceinline__ T wave_scan(T v, T none) {
  v = Op::of(v, dpp<0x111, 0xf>(v, none));      // the row's lane - 1, - 2, - 4, - 8
  v = Op::of(v, dpp<0x112, 0xf>(v, none));
  v = Op::of(v, dpp<0x114, 0xf>(v, none));
  v = Op::of(v, dpp<0x118, 0xf>(v, none));
  v = Op::of(v, dpp<0x142, 0xa>(v, none));      // lane 15 of the row before, into rows 1 and 3
  v = Op::of(v, dpp<0x143, 0xc>(v, none));      // lane 31, into rows 2 and 3
  return v;
}

template <class T>
__device__ __forceinline__ T lane_value(T v, int lane) {
  constexpr int N = sizeof(T) / 4;
  struct Words { int w[N]; };
  Words a = __builtin_bit_cast(Words, v);
#pragma unroll
  for (int i = 0; i < N; ++i) a.w[i] = __builtin_amdgcn_readlane(a.w[i], lane);
  return __builtin_bit_cast(T, a);
}

template <class Op, class T>
__device__ __forceinline__ T wave_reduce(T v, T none) {
  return lane_value(wave_scan<Op>(v, none), 63);
}

template <class Op, class T>
__device__ __forceinline__ T neutral();
template <> __device__ __forceinline__ float neutral<Max, float>() { return -INFINITY; }
template <> __device__ __forceinline__ double neutral<Max, double>() { return -INFINITY; }
template <> __device__ __forceinline__ uint64_t neutral<Max, uint64_t>() { return 0; }
template <> __device__ __forceinline__ float neutral<Sum, float>() { return 0.f; }
template <> __device__ __forceinline__ double neutral<Sum, double>() { return 0.; }

// A barrier of a group of NT threads: of a block, or of one wave of several
// that work on rows of their own.
template <int NT>
__device__ __forceinline__ void sync() {
  if constexpr (NT == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// A thread's number in its group, the group's in its block.
template <int NT>
__device__ __forceinline__ int thread_of() { return NT == 64 ? threadIdx.x & 63 : threadIdx.x; }
template <int NT>
__device__ __forceinline__ int group_of() { return NT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0; }

// Every thread gets the result.  sh: NT / 64 entries, free for reuse on return.
template <int NT, class Op, class T>
__device__ __forceinline__ T block_reduce(T v, T* sh) {
  v = wave_reduce<Op>(v, neutral<Op, T>());
  if constexpr (NT == 64) return v;
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < NT / 64; ++w) v = Op::of(v, sh[w]);
  __syncthreads();
  return v;
}

// A logit as a whole number in the order of the values (NaN as -inf, -0 as 0).
__device__ __forceinline__ uint32_t order_of(float x) {
  x = x != x ? -INFINITY : x + 0.f;
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t o) {
  return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

// The order above the complement of the index: no two keys of a row are alike,
// and of equal logits the first has the larger.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~id; }

// Rows lie at any address; their vectors lie on the memory's grid of 128 bytes.
// A row's logits are numbered from the grid's last point before it: `lead` of
// the numbers are no logits.  (Vectors from the row's own start took 18 to 20 %
// longer where that is off the grid, as in rows of an odd vocabulary.)
template <class T>
__device__ __forceinline__ int lead_of(const typename T::raw* x) { return (int)((uintptr_t)x & 127) / (int)sizeof(typename T::raw); }
constexpr int LEAD = 64;                   // more than any lead

// ---- rows of a few logits ----------------------------------------------------
// A wave takes 64 rows, a thread one of them, from LDS: the logits come in
// together (each row's own addresses, 64 of the rows' logits at a time) and lie
// in words of 4 bytes at an odd pitch, so that the threads' reads of one column
// fall on different banks.
constexpr int FEW = 64;                    // logits of such a row, at most

// Behind a row's logits, up to a multiple of 4, lie -inf: what goes over a row
// takes 4 at a time (a read of LDS that is waited for costs 100 cycles).
__host__ __device__ inline int few_pitch(int vocab) { return ((vocab + 3) & ~3) | 1; }

// f(row of the 64, v, its place among all) for every logit, 64 at a time
template <class F>
__device__ __forceinline__ void each_of_rows(int rows, int vocab, F f) {
  const int lane = threadIdx.x & 63, dr = 64 / vocab, dv = 64 - dr * vocab;
  int r = lane / vocab, v = lane - r * vocab;
  for (int i = lane; i < rows * vocab; i += 64) {
    f(r, v, i);
    r += dr;
    v += dv;
    if (v >= vocab) v -= vocab, ++r;
  }
}

// Rows r0 .. r0 + rows (at most 64) to LDS.
template <class T>
__device__ __forceinline__ void load_few(const Rows& x, int64_t r0, int rows, float* few, int pitch) {
  using raw = typename T::raw;
  const raw* const data = (const raw*)x.data;
  const int vocab = x.vocab, lane = threadIdx.x & 63, n = rows * vocab;
  for (int v = vocab; v & 3; ++v) few[lane * pitch + v] = -INFINITY;
  if (x.inner != 1 || x.stride_outer != vocab) {
    each_of_rows(rows, vocab, [&](int r, int v, int) { few[r * pitch + v] = T::get(data[x.at(r0 + r) + v]); });
    return;
  }
  // contiguous: eight loads under way at a time
  const raw* const from = data + r0 * vocab;
  const int dr = 64 / vocab, dv = 64 - dr * vocab;
  int r = lane / vocab, v = lane - r * vocab;
  for (int i0 = lane; i0 < n; i0 += 64 * 8) {
    raw f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = from[min(i0 + 64 * j, n - 1)];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i0 + 64 * j < n) few[r * pitch + v] = T::get(f[j]);
      r += dr;
      v += dv;
      if (v >= vocab) v -= vocab, ++r;
    }
  }
}

// ---- host ------------------------------------------------------------------
#define BAD(...) return lt::set_error(LT_EINVAL, __VA_ARGS__)

inline int dtype_bytes(int d) { return d == LT_F32 ? 4 : 2; }

inline bool rows_ok(const lt_rows* x, const char* what, lt_status* st) {
  *st = LT_OK;
  if (!x) *st = lt::set_error(LT_EINVAL, "%s: NULL", what);
  else if (x->dtype < LT_F32 || x->dtype > LT_BF16) *st = lt::set_error(LT_EINVAL, "%s: dtype %d", what, x->dtype);
  else if (x->rows < 0 || x->inner < 1) *st = lt::set_error(LT_EINVAL, "%s: rows %lld, inner %lld", what, (long long)x->rows, (long long)x->inner);
  else if (x->vocab < 1 || x->vocab > LT_MAX_VOCAB) *st = lt::set_error(LT_EINVAL, "%s: vocab %lld", what, (long long)x->vocab);
  else if (x->rows > 0 && (!x->data || (uintptr_t)x->data % dtype_bytes(x->dtype)))
    *st = lt::set_error(LT_EINVAL, "%s: data is NULL or not aligned to its type", what);
  return *st == LT_OK;
}

inline bool temperature_ok(double t) { return t >= 1e-6 && t <= 1e6; }

inline Rows rows_of(const lt_rows* x) {
  Rows r;
  r.data = x->data;
  r.inner = x->inner;
  r.stride_outer = x->stride_outer;
  r.stride_inner = x->stride_inner;
  r.vocab = (int32_t)x->vocab;
  return r;
}

// The call's device is current for as long as this lives.
struct OnDevice {
  int was = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&was);
    if (err == hipSuccess && was != device) err = hipSetDevice(device);
    else if (err == hipSuccess) was = -1;
  }
  ~OnDevice() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

// `blocks` blocks, in as many launches as the grid's limit (2^32 threads) takes:
// block 0 of a launch is p.block0.
template <class P>
lt_status launch(void (*kernel)(P), int64_t blocks, int threads, P p, void* stream, const char* what, int lds = 0) {
  const int64_t most = (int64_t)1 << 21;
  for (p.block0 = 0; p.block0 < blocks; p.block0 += most) {
    const int64_t n = blocks - p.block0 < most ? blocks - p.block0 : most;
    void* args[] = {&p};
    const hipError_t e = hipLaunchKernel((const void*)kernel, dim3((uint32_t)n), dim3(threads), args, lds, (hipStream_t)stream);
    if (e != hipSuccess) return lt::set_error(LT_EHIP, "%s: %s", what, hipGetErrorString(e));
  }
  return LT_OK;
}

#define ON_DEVICE(d)                                                                                   \
  OnDevice on(d);                                                                                      \
  if (on.err != hipSuccess) return lt::set_error(LT_EHIP, "device %d: %s", (int)(d), hipGetErrorString(on.err))

}  // namespace
