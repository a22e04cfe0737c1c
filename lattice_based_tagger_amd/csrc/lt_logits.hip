// lt_logits.hip -- operators over a model's logits (include/lattice_logits.h):
// the k best of a row with its log-sum-exp, the distillation loss against a
// teacher's top logits with its gradient, and the verification of drafted
// tokens.  One block a row (a sequence, for the verification).
#include <dlfcn.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/lattice_logits.h"
#include "lt_error.h"

namespace {

constexpr int NT = 256;                   // threads of a block
constexpr int NW = NT / 64;               // its waves
constexpr int MAXK = LT_MAX_TOP;
constexpr float LOWEST = -3.4028234663852886e38f;

struct Rows {
  const void* data;
  int64_t inner, stride_outer, stride_inner;
  int32_t vocab;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    return inner == 1 ? r * stride_outer : (r / inner) * stride_outer + (r % inner) * stride_inner;
  }
};

struct F32 {
  using raw = float;
  static __device__ __forceinline__ float get(raw v) { return v; }
  static __device__ __forceinline__ raw put(float v) { return v; }
};
struct F16 {
  using raw = uint16_t;
  static __device__ __forceinline__ float get(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ raw put(float v) { return __builtin_bit_cast(raw, (_Float16)v); }
};
struct BF16 {
  using raw = uint16_t;
  static __device__ __forceinline__ float get(raw v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
  // to the nearest, ties to even; a NaN stays one
  static __device__ __forceinline__ raw put(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    if (v != v) return (raw)((b >> 16) | 0x40);
    return (raw)((b + 0x7fff + ((b >> 16) & 1)) >> 16);
  }
};

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
};
struct Sum {
  template <class T>
  static __device__ __forceinline__ T of(T a, T b) { return a + b; }
};

// Every thread gets the result.  sh: NW entries, free for reuse on return.
template <class Op, class T>
__device__ __forceinline__ T block_reduce(T v, T* sh) {
  for (int o = 32; o; o >>= 1) v = Op::of(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < NW; ++w) v = Op::of(v, sh[w]);
  __syncthreads();
  return v;
}

// sum of exp2((x - m) c) over what a thread has seen; m is LOWEST at first, so
// that a -inf logit adds 0 and a row of the type's lowest value adds 1 each.
struct Running {
  float m = LOWEST, s = 0.f;
  __device__ __forceinline__ void add(float x, float c) {
    if (x > m) {
      s *= exp2f((m - x) * c);
      m = x;
    }
    s += exp2f((x - m) * c);
  }
};

// The order of the logits as whole numbers (NaN as -inf, -0 as 0), above the
// complement of the index: no two keys of a row are alike.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) {
  x = x != x ? -INFINITY : x + 0.f;
  uint32_t b = __builtin_bit_cast(uint32_t, x);
  b ^= (b >> 31) ? 0xffffffffu : 0x80000000u;
  return ((uint64_t)b << 32) | (uint32_t)~id;
}

// ---- the k best ------------------------------------------------------------
struct TopParams {
  Rows x;
  int64_t rows;
  int32_t k;
  float c;                // log2(e) / temperature
  void* values;
  int64_t* ids;
  float* lse;
};

template <class T>
__global__ __launch_bounds__(NT) void lt_top_k(TopParams p) {
  using raw = typename T::raw;
  __shared__ uint64_t sh64[NW];
  __shared__ float shf[NW];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const raw* x = (const raw*)p.x.data + p.x.at(r);
    Running run;
    for (int64_t v = threadIdx.x; v < p.x.vocab; v += NT) run.add(T::get(x[v]), p.c);
    const float m = block_reduce<Max>(run.m, shf);
    const float s = block_reduce<Sum>(run.s * exp2f((run.m - m) * p.c), shf);
    if (threadIdx.x == 0)
      p.lse[r] = m == INFINITY ? m : (float)((double)m * (p.c * 0.6931471805599453) + log((double)s));
    uint64_t below = ~0ull;
    for (int j = 0; j < p.k; ++j) {
      uint64_t best = 0;
      for (int64_t v = threadIdx.x; v < p.x.vocab; v += NT) {
        const uint64_t key = order_key(T::get(x[v]), (uint32_t)v);
        if (key < below && key > best) best = key;
      }
      below = block_reduce<Max>(best, sh64);
      if (threadIdx.x == 0) {
        const uint32_t id = ~(uint32_t)below;
        p.ids[r * p.k + j] = id;
        ((raw*)p.values)[r * p.k + j] = x[id];
      }
    }
  }
}

// ---- distillation ----------------------------------------------------------
struct Teacher {
  const void* ids;
  const void* top;
  const float* top_lse;
  int32_t entries, ids_bytes, top_dtype;
};

struct DistillParams {
  Rows z;
  Teacher t;
  int64_t rows;
  double inv_t;           // 1 / temperature
  float c;                // log2(e) / temperature
  float* loss;
  float* stats;
  const float* weight;
  int64_t weight_stride;
  Rows grad;
};

// A teacher's row in LDS: id[j] (-1: no entry) and p[j].
struct TeacherRow {
  int32_t id[MAXK];
  double p[MAXK];
  double sh[NW];
};

// Fills it; returns sum p (0: a row without entries) and p_rest, in 64 bits:
// p_rest is what is left of 1.
__device__ __forceinline__ void teacher_row(const Teacher& t, int64_t r, int32_t vocab, double inv_t, TeacherRow& o,
                                            double& psum, double& prest) {
  double m = -INFINITY;
  for (int j = threadIdx.x; j < t.entries; j += NT) {
    const int64_t id = any_id(t.ids, r * t.entries + j, t.ids_bytes);
    const bool there = id >= 0 && id < vocab;
    const double v = there ? any_float(t.top, r * t.entries + j, t.top_dtype) * inv_t : -INFINITY;
    o.id[j] = there ? (int32_t)id : -1;
    o.p[j] = v;
    m = v > m || v != v ? v : m;
  }
  double ref = t.top_lse ? (double)t.top_lse[r] : block_reduce<Max>(m, o.sh);
  if (!t.top_lse && ref == -INFINITY) ref = 0;
  double s = 0;
  for (int j = threadIdx.x; j < t.entries; j += NT) {
    const double e = o.id[j] < 0 ? 0.0 : exp(o.p[j] - ref);
    o.p[j] = e;
    s += e;
  }
  psum = block_reduce<Sum>(s, o.sh);
  prest = 0;
  if (t.top_lse) {
    prest = psum < 1 ? 1 - psum : 0;
  } else if (psum > 0) {
    for (int j = threadIdx.x; j < t.entries; j += NT) o.p[j] /= psum;
    psum = 1;
  }
  __syncthreads();
}

constexpr int WINDOW = 1 << 18;           // logits whose membership bits are held at a time

template <class T>
__global__ __launch_bounds__(NT) void lt_distill_fwd(DistillParams p) {
  using raw = typename T::raw;
  __shared__ TeacherRow t;
  __shared__ uint32_t bits[WINDOW / 32];
  __shared__ float shf[NW];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const raw* z = (const raw*)p.z.data + p.z.at(r);
    double psum, prest;
    teacher_row(p.t, r, p.z.vocab, p.inv_t, t, psum, prest);
    Running all, rest;
    for (int64_t w0 = 0; w0 < p.z.vocab; w0 += WINDOW) {
      const int n = (int)min((int64_t)WINDOW, p.z.vocab - w0);
      for (int i = threadIdx.x; i < (n + 31) / 32; i += NT) bits[i] = 0;
      __syncthreads();
      for (int j = threadIdx.x; j < p.t.entries; j += NT) {
        const int64_t v = t.id[j] - w0;
        if (t.id[j] >= 0 && v >= 0 && v < n) atomicOr(&bits[v >> 5], 1u << (v & 31));
      }
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += NT) {
        const float x = T::get(z[w0 + i]);
        all.add(x, p.c);
        if (!(bits[i >> 5] >> (i & 31) & 1)) rest.add(x, p.c);
      }
      __syncthreads();
    }
    const float m = block_reduce<Max>(all.m, shf);
    const float s = block_reduce<Sum>(all.s * exp2f((all.m - m) * p.c), shf);
    const float sr = block_reduce<Sum>(rest.s * exp2f((rest.m - m) * p.c), shf);
    const double logs = log((double)s);
    double loss = 0;
    for (int j = threadIdx.x; j < p.t.entries; j += NT) {
      const double pj = t.p[j];
      if (t.id[j] >= 0 && pj != 0) loss += pj * (log(pj) - ((double)T::get(z[t.id[j]]) - m) * p.inv_t + logs);
    }
    loss = block_reduce<Sum>(loss, t.sh);
    if (threadIdx.x == 0) {
      const double qrest = (double)sr / s;
      if (!(qrest > 0)) prest = 0;
      if (prest > 0) loss += prest * (log(prest) - log(qrest));
      p.loss[r] = (float)loss;
      const double whole = psum + prest;
      float* st = p.stats + r * LT_DISTILL_STATS;
      st[0] = m;
      st[1] = s > 0 ? (float)(whole * p.inv_t / s) : 0.f;
      st[2] = s > 0 ? (float)((whole - (prest > 0 ? prest / qrest : 0)) * p.inv_t / s) : 0.f;
    }
  }
}

template <class T>
__global__ __launch_bounds__(NT) void lt_distill_bwd(DistillParams p) {
  using raw = typename T::raw;
  __shared__ TeacherRow t;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const raw* z = (const raw*)p.z.data + p.z.at(r);
    raw* g = (raw*)p.grad.data + p.grad.at(r);
    double psum, prest;
    teacher_row(p.t, r, p.z.vocab, p.inv_t, t, psum, prest);
    const float* st = p.stats + r * LT_DISTILL_STATS;
    const float m = st[0], w = p.weight[r * p.weight_stride];
    const float in = st[1] * w, out = st[2] * w;
    for (int64_t v = threadIdx.x; v < p.z.vocab; v += NT) g[v] = T::put(exp2f((T::get(z[v]) - m) * p.c) * out);
    __syncthreads();
    for (int j = threadIdx.x; j < p.t.entries; j += NT) {
      const int id = t.id[j];
      if (id < 0) continue;
      double pj = 0;                       // of every entry with this id
      for (int i = 0; i < p.t.entries; ++i)
        if (t.id[i] == id) pj += t.p[i];
      g[id] = T::put(exp2f((T::get(z[id]) - m) * p.c) * in - (float)(pj * p.inv_t) * w);
    }
    __syncthreads();
  }
}

// ---- verification ----------------------------------------------------------
struct VerifyParams {
  Rows target, draft;     // draft.data NULL: certain tokens
  const void* ids;
  const float* accept_u;
  const float* sample_u;
  const int32_t* lengths;
  int64_t batch;
  int32_t drafts, ids_bytes;
  double inv_t;
  int64_t* tokens;
  int64_t* accepted;
};

struct Soft {              // softmax of a row: exp((x - m) / T) / s
  float m;
  double s;
  __device__ __forceinline__ double of(float x, double inv_t) const {
    return s > 0 ? exp(((double)x - m) * inv_t) / s : 0.0;
  }
};

template <class T>
__device__ __forceinline__ Soft soft_row(const typename T::raw* x, int vocab, double inv_t, float* shf, double* shd) {
  float m = LOWEST;
  for (int v = threadIdx.x; v < vocab; v += NT) m = fmaxf(m, T::get(x[v]));
  m = block_reduce<Max>(m, shf);
  double s = 0;
  for (int v = threadIdx.x; v < vocab; v += NT) s += exp(((double)T::get(x[v]) - m) * inv_t);
  return Soft{m, block_reduce<Sum>(s, shd)};
}

template <class T>
__global__ __launch_bounds__(NT) void lt_verify(VerifyParams p) {
  using raw = typename T::raw;
  __shared__ float shf[NW];
  __shared__ double shd[NW];
  __shared__ int sh_last;
  const int V = p.target.vocab;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int64_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
    int n = p.lengths ? p.lengths[b] : p.drafts;
    n = max(0, min(n, p.drafts));
    const raw *x = nullptr, *y = nullptr;
    Soft px{}, qx{};
    int a = 0;
    int64_t id = -1;
    for (;; ++a) {
      x = (const raw*)p.target.data + p.target.at(b * (p.drafts + 1) + a);
      px = soft_row<T>(x, V, p.inv_t, shf, shd);
      if (a == n) break;
      id = any_id(p.ids, b * p.drafts + a, p.ids_bytes);
      const bool there = id >= 0 && id < V;
      double q = 1;
      if (p.draft.data) {
        y = (const raw*)p.draft.data + p.draft.at(b * p.drafts + a);
        qx = soft_row<T>(y, V, p.inv_t, shf, shd);
        q = there ? qx.of(T::get(y[id]), p.inv_t) : 0.0;
      }
      if (!(there && p.accept_u[b * p.drafts + a] * q < px.of(T::get(x[id]), p.inv_t))) break;
      if (tid == 0) p.tokens[b * (p.drafts + 1) + a] = id;
    }
    bool minus = a < n;                     // w = max(p - q, 0), or p
    auto weight = [&](int v) -> double {
      const double pv = px.of(T::get(x[v]), p.inv_t);
      if (!minus) return pv;
      const double d = pv - (p.draft.data ? qx.of(T::get(y[v]), p.inv_t) : v == id ? 1.0 : 0.0);
      return d > 0 ? d : 0.0;
    };
    double total = 0;
    for (int v = tid; v < V; v += NT) total += weight(v);
    total = block_reduce<Sum>(total, shd);
    if (minus && !(total > 0)) {
      minus = false;
      total = px.s > 0 ? 1 : 0;
    }
    const double line = p.sample_u[b] * total;
    double before = 0;
    int token = -1, last = -1;
    for (int v0 = 0; v0 < V && token < 0; v0 += NT) {
      const int v = v0 + tid;
      const double w = v < V ? weight(v) : 0.0;
      double cum = w;
      for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(cum, o, 64);
        if (lane >= o) cum += u;
      }
      if (lane == 63) shd[wave] = cum;
      if (tid == 0) sh_last = 0x7fffffff;
      __syncthreads();
      cum += before;
      for (int i = 0; i < NW; ++i) {
        if (i < wave) cum += shd[i];
        before += shd[i];
      }
      if (w > 0) {
        last = v;
        if (cum > line) atomicMin(&sh_last, v);
      }
      __syncthreads();
      if (sh_last != 0x7fffffff) token = sh_last;
      __syncthreads();
    }
    if (token < 0) {
      if (tid == 0) sh_last = -1;
      __syncthreads();
      atomicMax(&sh_last, last);
      __syncthreads();
      token = sh_last;
      __syncthreads();
    }
    if (tid == 0) p.accepted[b] = a;
    for (int i = a + tid; i <= p.drafts; i += NT) p.tokens[b * (p.drafts + 1) + i] = i == a ? token : -1;
  }
}

// ---- host ------------------------------------------------------------------
#define BAD(...) return lt::set_error(LT_EINVAL, __VA_ARGS__)

int dtype_bytes(int d) { return d == LT_F32 ? 4 : 2; }

bool rows_ok(const lt_rows* x, const char* what, lt_status* st) {
  *st = LT_OK;
  if (!x) *st = lt::set_error(LT_EINVAL, "%s: NULL", what);
  else if (x->dtype < LT_F32 || x->dtype > LT_BF16) *st = lt::set_error(LT_EINVAL, "%s: dtype %d", what, x->dtype);
  else if (x->rows < 0 || x->inner < 1) *st = lt::set_error(LT_EINVAL, "%s: rows %lld, inner %lld", what, (long long)x->rows, (long long)x->inner);
  else if (x->vocab < 1 || x->vocab > 0x7fffffff) *st = lt::set_error(LT_EINVAL, "%s: vocab %lld", what, (long long)x->vocab);
  else if (x->rows > 0 && (!x->data || (uintptr_t)x->data % dtype_bytes(x->dtype)))
    *st = lt::set_error(LT_EINVAL, "%s: data is NULL or not aligned to its type", what);
  return *st == LT_OK;
}

bool temperature_ok(double t) { return t >= 1e-6 && t <= 1e6; }

Rows rows_of(const lt_rows* x) {
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

template <class P>
lt_status launch(void (*kernel)(P), int64_t blocks, int threads, P& p, void* stream, const char* what) {
  void* args[] = {&p};
  const hipError_t e = hipLaunchKernel((const void*)kernel, dim3((uint32_t)blocks), dim3(threads), args, 0, (hipStream_t)stream);
  if (e != hipSuccess) return lt::set_error(LT_EHIP, "%s: %s", what, hipGetErrorString(e));
  return LT_OK;
}

#define BY_TYPE(dtype, kernel) ((dtype) == LT_F32 ? kernel<F32> : (dtype) == LT_F16 ? kernel<F16> : kernel<BF16>)
#define ON_DEVICE(d)                                                                                   \
  OnDevice on(d);                                                                                      \
  if (on.err != hipSuccess) return lt::set_error(LT_EHIP, "device %d: %s", (int)(d), hipGetErrorString(on.err))

constexpr int64_t MAX_BLOCKS = 1 << 20;

constexpr double LOG2E = 1.4426950408889634;

lt_status distill_check(const lt_rows* z, const lt_teacher* t, double temperature) {
  lt_status st;
  if (!rows_ok(z, "logits", &st)) return st;
  if (!t) BAD("teacher: NULL");
  if (t->entries < 1 || t->entries > MAXK) BAD("teacher: %d entries (1 .. %d)", t->entries, MAXK);
  if (t->ids_bytes != 4 && t->ids_bytes != 8) BAD("teacher: ids of %d bytes", t->ids_bytes);
  if (t->top_dtype < LT_F32 || t->top_dtype > LT_BF16) BAD("teacher: dtype %d", t->top_dtype);
  if (z->rows > 0 && (!t->ids || !t->top)) BAD("teacher: NULL");
  if (!temperature_ok(temperature)) BAD("temperature %g (1e-6 .. 1e6)", temperature);
  return LT_OK;
}

lt_status grad_check(const lt_rows* z, const lt_rows* g, const float* weight, int64_t weight_stride) {
  lt_status st;
  if (!rows_ok(g, "grad", &st)) return st;
  if (g->rows != z->rows || g->vocab != z->vocab || g->dtype != z->dtype || g->device != z->device)
    BAD("grad: not the logits' rows, vocab, dtype and device");
  if (z->rows > 0 && !weight) BAD("weight: NULL");
  if (weight_stride != 0 && weight_stride != 1) BAD("weight_stride %lld", (long long)weight_stride);
  return LT_OK;
}

DistillParams distill_params(const lt_rows* z, const lt_teacher* t, double temperature) {
  DistillParams p{};
  p.z = rows_of(z);
  p.t = Teacher{t->ids, t->top, t->top_lse, t->entries, t->ids_bytes, t->top_dtype};
  p.rows = z->rows;
  p.inv_t = 1 / temperature;
  p.c = (float)(LOG2E / temperature);
  return p;
}

}  // namespace

extern "C" {

const char* lt_hip_library(void) {
  static const char* path = [] {
    Dl_info info;
    return dladdr(reinterpret_cast<void*>(&hipGetDeviceCount), &info) && info.dli_fname ? info.dli_fname : "";
  }();
  return path;
}

int64_t lt_top_logits_workspace(const lt_rows*, int32_t) { return 0; }

lt_status lt_top_logits(const lt_rows* x, int32_t k, double temperature, void* values, int64_t* ids, float* lse,
                        void*, int64_t, void* stream) {
  lt_status st;
  if (!rows_ok(x, "logits", &st)) return st;
  if (k < 1 || k > MAXK || k > x->vocab) BAD("k %d (1 .. min(vocab, %d))", k, MAXK);
  if (!temperature_ok(temperature)) BAD("temperature %g (1e-6 .. 1e6)", temperature);
  if (x->rows == 0) return LT_OK;
  if (!values || !ids || !lse) BAD("output: NULL");
  ON_DEVICE(x->device);
  TopParams p{};
  p.x = rows_of(x);
  p.rows = x->rows;
  p.k = k;
  p.c = (float)(LOG2E / temperature);
  p.values = values;
  p.ids = ids;
  p.lse = lse;
  return launch(BY_TYPE(x->dtype, lt_top_k), x->rows < MAX_BLOCKS ? x->rows : MAX_BLOCKS, NT, p, stream, "lt_top_logits");
}

int64_t lt_distill_workspace(const lt_rows* z, int32_t) {
  return z ? z->rows * LT_DISTILL_STATS * (int64_t)sizeof(float) : 0;
}

lt_status lt_distill_forward(const lt_rows* z, const lt_teacher* t, double temperature, float* loss, float* stats,
                             void*, int64_t, void* stream) {
  const lt_status st = distill_check(z, t, temperature);
  if (st != LT_OK || z->rows == 0) return st;
  if (!loss || !stats) BAD("output: NULL");
  ON_DEVICE(z->device);
  DistillParams p = distill_params(z, t, temperature);
  p.loss = loss;
  p.stats = stats;
  return launch(BY_TYPE(z->dtype, lt_distill_fwd), z->rows < MAX_BLOCKS ? z->rows : MAX_BLOCKS, NT, p, stream, "lt_distill_forward");
}

lt_status lt_distill_backward(const lt_rows* z, const lt_teacher* t, double temperature, const float* stats,
                              const float* weight, int64_t weight_stride, const lt_rows* grad, void* stream) {
  lt_status st = distill_check(z, t, temperature);
  if (st == LT_OK) st = grad_check(z, grad, weight, weight_stride);
  if (st != LT_OK || z->rows == 0) return st;
  if (!stats) BAD("stats: NULL");
  ON_DEVICE(z->device);
  DistillParams p = distill_params(z, t, temperature);
  p.stats = const_cast<float*>(stats);
  p.weight = weight;
  p.weight_stride = weight_stride;
  p.grad = rows_of(grad);
  return launch(BY_TYPE(z->dtype, lt_distill_bwd), z->rows < MAX_BLOCKS ? z->rows : MAX_BLOCKS, NT, p, stream, "lt_distill_backward");
}

lt_status lt_distill_fused(const lt_rows* z, const lt_teacher* t, double temperature, const float* weight,
                           int64_t weight_stride, float* loss, const lt_rows* grad, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  lt_status st = distill_check(z, t, temperature);
  if (st == LT_OK) st = grad_check(z, grad, weight, weight_stride);
  if (st != LT_OK || z->rows == 0) return st;
  if (!workspace || workspace_bytes < lt_distill_workspace(z, t->entries)) BAD("workspace: %lld bytes", (long long)workspace_bytes);
  st = lt_distill_forward(z, t, temperature, loss, (float*)workspace, nullptr, 0, stream);
  if (st != LT_OK) return st;
  return lt_distill_backward(z, t, temperature, (const float*)workspace, weight, weight_stride, grad, stream);
}

int64_t lt_verify_workspace(const lt_draft*) { return 0; }

lt_status lt_verify_draft(const lt_draft* d, double temperature, int64_t* tokens, int64_t* accepted, void*, int64_t,
                          void* stream) {
  lt_status st;
  if (!d) BAD("draft: NULL");
  if (!rows_ok(d->target, "target", &st)) return st;
  if (d->batch < 0 || d->drafts < 0 || d->drafts > LT_MAX_DRAFTS) BAD("batch %lld, drafts %d (0 .. %d)", (long long)d->batch, d->drafts, LT_MAX_DRAFTS);
  if (d->target->rows != d->batch * (d->drafts + 1)) BAD("target: %lld rows, batch * (drafts + 1) = %lld", (long long)d->target->rows, (long long)(d->batch * (d->drafts + 1)));
  if (d->ids_bytes != 4 && d->ids_bytes != 8) BAD("ids of %d bytes", d->ids_bytes);
  if (d->draft) {
    if (!rows_ok(d->draft, "draft", &st)) return st;
    if (d->draft->rows != d->batch * d->drafts || d->draft->vocab != d->target->vocab || d->draft->dtype != d->target->dtype ||
        d->draft->device != d->target->device)
      BAD("draft: not batch * drafts rows of the target's vocab, dtype and device");
  }
  if (!temperature_ok(temperature)) BAD("temperature %g (1e-6 .. 1e6)", temperature);
  if (d->batch == 0) return LT_OK;
  if (!tokens || !accepted || !d->sample_u || (d->drafts > 0 && (!d->ids || !d->accept_u))) BAD("NULL argument");
  ON_DEVICE(d->target->device);
  VerifyParams p{};
  p.target = rows_of(d->target);
  if (d->draft && d->drafts > 0) p.draft = rows_of(d->draft);
  p.ids = d->ids;
  p.accept_u = d->accept_u;
  p.sample_u = d->sample_u;
  p.lengths = d->lengths;
  p.batch = d->batch;
  p.drafts = d->drafts;
  p.ids_bytes = d->ids_bytes;
  p.inv_t = 1 / temperature;
  p.tokens = tokens;
  p.accepted = accepted;
  return launch(BY_TYPE(d->target->dtype, lt_verify), d->batch < MAX_BLOCKS ? d->batch : MAX_BLOCKS, NT, p, stream, "lt_verify_draft");
}

}  // extern "C"
