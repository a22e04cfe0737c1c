// lt_distill.hip -- the distillation loss against a teacher's top logits and
// its gradient (include/lattice_logits.h lt_distill_*).
#include "lt_logits.h"

namespace {

constexpr int NT = 256;                   // threads of a block
constexpr int NW = NT / 64;               // its waves

// ---- distillation ----------------------------------------------------------
struct Teacher {
  const void* ids;
  const void* top;
  const float* top_lse;
  int32_t entries, ids_bytes, top_dtype;
};

struct DistillParams {
  int64_t block0;         // of this launch
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
  double ref = t.top_lse ? (double)t.top_lse[r] : block_reduce<NT, Max>(m, o.sh);
  if (!t.top_lse && ref == -INFINITY) ref = 0;
  double s = 0;
  for (int j = threadIdx.x; j < t.entries; j += NT) {
    const double e = o.id[j] < 0 ? 0.0 : exp(o.p[j] - ref);
    o.p[j] = e;
    s += e;
  }
  psum = block_reduce<NT, Sum>(s, o.sh);
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
  {
    const int64_t r = p.block0 + blockIdx.x;
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
    const float m = block_reduce<NT, Max>(all.m, shf);
    const float s = block_reduce<NT, Sum>(all.s * exp2f((all.m - m) * p.c), shf);
    const float sr = block_reduce<NT, Sum>(rest.s * exp2f((rest.m - m) * p.c), shf);
    const double logs = log((double)s);
    double loss = 0;
    for (int j = threadIdx.x; j < p.t.entries; j += NT) {
      const double pj = t.p[j];
      if (t.id[j] >= 0 && pj != 0) loss += pj * (log(pj) - ((double)T::get(z[t.id[j]]) - m) * p.inv_t + logs);
    }
    loss = block_reduce<NT, Sum>(loss, t.sh);
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
  {
    const int64_t r = p.block0 + blockIdx.x;
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
  return launch(BY_TYPE(z->dtype, lt_distill_fwd), z->rows, NT, p, stream, "lt_distill_forward");
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
  return launch(BY_TYPE(z->dtype, lt_distill_bwd), z->rows, NT, p, stream, "lt_distill_backward");
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

}  // extern "C"
