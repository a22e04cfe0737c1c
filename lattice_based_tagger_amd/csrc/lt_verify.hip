// lt_verify.hip -- the verification of drafted tokens
// (include/lattice_logits.h lt_verify_draft).
#include "lt_logits.h"

namespace {

constexpr int NT = 256;                   // threads of a block
constexpr int NW = NT / 64;               // its waves

// ---- verification ----------------------------------------------------------
struct VerifyParams {
  int64_t block0;         // of this launch
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
  m = block_reduce<NT, Max>(m, shf);
  double s = 0;
  for (int v = threadIdx.x; v < vocab; v += NT) s += exp(((double)T::get(x[v]) - m) * inv_t);
  return Soft{m, block_reduce<NT, Sum>(s, shd)};
}

template <class T>
__global__ __launch_bounds__(NT) void lt_verify(VerifyParams p) {
  using raw = typename T::raw;
  __shared__ float shf[NW];
  __shared__ double shd[NW];
  __shared__ int sh_last;
  const int V = p.target.vocab;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  {
    const int64_t b = p.block0 + blockIdx.x;
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
    total = block_reduce<NT, Sum>(total, shd);
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

}  // namespace

extern "C" {

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
  return launch(BY_TYPE(d->target->dtype, lt_verify), d->batch, NT, p, stream, "lt_verify_draft");
}

}  // extern "C"
