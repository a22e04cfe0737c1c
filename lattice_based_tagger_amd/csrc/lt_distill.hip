// lt_distill.hip -- the distillation loss against a teacher's top logits and
// its gradient (include/lattice_logits.h lt_distill_*).
#include <type_traits>

#include "lt_logits.h"

namespace {

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
  int32_t splits;         // blocks of a row
  int32_t chunk;          // of a row's numbers, to a block (a multiple of its step)
  float* loss;
  float* stats;           // [rows][LT_DISTILL_STATS]: Factors
  float2* part;           // splits > 1: [rows][splits] reference and sum, its sign set where an id came again
  float scale;
  const float* weight;    // NULL: 1
  int64_t weight_stride;
  Rows grad;
  bool past;              // the gradient is written past the caches
};

__device__ __forceinline__ float weight_of(const DistillParams& p, int64_t r) {
  return p.weight ? p.scale * p.weight[r * p.weight_stride] : p.scale;
}

// What a block keeps in LDS: the entries, and
// a bit for each logit of a window that says whether it is one.
template <int NT, int WINDOW>
struct DistillShared {
  alignas(16) int id[MAXK];                // (read four at a time)
  float mass[MAXK];
  uint32_t bits[WINDOW / 32];
  double sh[NT / 64];
  int again;                               // an id came more than once
};

// A thread's entries of the teacher's row, j = i * NT + thread: logits that are
// no entry have id -1 and p 0.  p in 64 bits: what is left of 1 is used.
// Logarithms are to the base 2.  (A library's logarithm or exponential of 64
// bits takes 60 operations or more of two slots each: for every row of 2000
// logits they took longer than the logits.)
template <int NT, int N_ = (MAXK / NT > 1 ? MAXK / NT : 1)>
struct Entries {
  static constexpr int N = N_;
  int id[N];
  double p[N], logp[N];
  double sum, rest;       // of the row
  // Nothing to learn: no entry, or none with a weight.  Loss and gradient are 0
  // whatever the logits are (a padded position's are often NaN); they are not read.
  __device__ __forceinline__ bool blank() const { return sum == 0 && rest == 0; }
};

// With top_lse, an entry too unlikely for its p to be more than 0 still tells its
// row from one without entries.
constexpr double TRACE = 1e-300;

// 2^t; 0 far below, infinite far above (a log-sum-exp that is not the entries').
__device__ __forceinline__ double exp2_or_0(double t) { return t < -1000 ? 0.0 : t > 1000 ? INFINITY : exp2_64(t); }

template <int NT, int N>
__device__ __forceinline__ void load_entries(const Teacher& t, int64_t r, int vocab, double inv_t, Entries<NT, N>& o,
                                             double* sh) {
  const double c = inv_t * LOG2E;
  float m = -INFINITY, top[N];
  double s = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = i * NT + thread_of<NT>();
    o.id[i] = -1;
    top[i] = -INFINITY;
    if (j < t.entries) {
      const int64_t id = any_id(t.ids, r * t.entries + j, t.ids_bytes);
      if (id >= 0 && id < vocab) {
        o.id[i] = (int)id;
        top[i] = any_float(t.top, r * t.entries + j, t.top_dtype);
      }
    }
    m = max2(m, top[i]);
  }
  double ref;
  if (t.top_lse) {
    ref = (double)t.top_lse[r] * LOG2E;
  } else {
    m = block_reduce<NT, Max>(m, (float*)sh);
    ref = m == -INFINITY ? 0 : m * c;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    o.logp[i] = top[i] * c - ref;
    o.p[i] = 0;
    if (i * NT < t.entries) {              // (for all threads)
      o.p[i] = o.id[i] < 0 ? 0.0 : exp2_or_0(o.logp[i]);
      s += t.top_lse && o.id[i] >= 0 && o.p[i] == 0 ? TRACE : o.p[i];
    }
  }
  o.sum = block_reduce<NT, Sum>(s, sh);
  o.rest = 0;
  if (t.top_lse) {
    if (o.sum > 0 && o.sum < 1) o.rest = 1 - o.sum;
  } else if (o.sum != 0) {
    // (a reciprocal good to 2^-20 or so, and two steps of Newton's: a division
    // takes three times as long)
    double inv = __builtin_amdgcn_rcp(o.sum);
    inv = fma(fma(-o.sum, inv, 1.0), inv, inv);
    inv = fma(fma(-o.sum, inv, 1.0), inv, inv);
    const double logs = log2_((float)o.sum);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o.logp[i] -= logs;
      o.p[i] *= inv;
    }
    o.sum = o.sum > 0 ? 1 : o.sum;         // (a NaN stays)
  }
}

// first: of a block's entries that are one logit the first alone (ids: MAXK in LDS,
// -1 behind the row's).  Which of several waves' an atomic finds first varies from
// call to call, and so would the order of a sum.
template <int NT>
__device__ __forceinline__ void only_first(const Entries<NT>& t, const int* ids, int entries, bool (&first)[1]) {
  const int own = threadIdx.x, id = t.id[0];
  bool before = false;
  for (int j = 0; j < entries; j += 16) {
    int4 o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = ((const int4*)&ids[j])[k];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int left = own - (j + k * 4);
      before |= (o[k].x == id && left > 0) | (o[k].y == id && left > 1) | (o[k].z == id && left > 2) | (o[k].w == id && left > 3);
    }
  }
  first[0] = id >= 0 && !before;
}

// A sum of exp2((z - m) c), and its reference m.
struct Sums {
  float m = LOWEST, s = 0.f;
};

// One pass over a row's logits with numbers in [v0, v1), from c0 on: the sum of
// all, or, with the tail (TAIL), of all that are no entries.  These have a
// reference of their own: beside a larger entry's their sum would lose its bits,
// or all of it -- 87 temperatures below it nothing is left of it in 32 bits, where
// the loss is to be 87 and the gradient p_rest.  first: of the entries in these
// windows that are one logit, whether it is the one that was seen first
// (sh.again: some were seen again).
template <class T, int NT, int U, int WINDOW, bool TAIL>
__device__ __forceinline__ Sums sum_row(const typename T::raw* row, int lead, int c0, int v0, int v1, float c, const Entries<NT>& t,
                                        DistillShared<NT, WINDOW>& sh, bool (&first)[Entries<NT>::N]) {
  constexpr int E = Vec<T>::E, STEP = NT * U * E;
  static_assert(WINDOW % STEP == 0 || WINDOW >= STEP, "a step lies in a window");
  const int tid = thread_of<NT>();
  const typename T::raw* const z = row - lead;
  Sums o;
  for (int w0 = c0; w0 < v1; w0 += WINDOW) {
    const int w1 = min(v1, w0 + WINDOW);
    if (TAIL) {
      for (int i = tid; i < (w1 - w0 + 31) / 32; i += NT) sh.bits[i] = 0;
      sync<NT>();
#pragma unroll
      for (int i = 0; i < Entries<NT>::N; ++i) {
        const int at = t.id[i] + lead - w0;
        if (t.id[i] >= 0 && at >= 0 && at < w1 - w0) {
          first[i] = !(atomicOr(&sh.bits[at >> 5], 1u << (at & 31)) >> (at & 31) & 1);
          if (!first[i]) sh.again = 1;
        }
      }
      sync<NT>();
    }
    for (int base = w0; base < w1; base += STEP) {
      Vec<T> v[U];
      load_step<T, NT, U>(v, z, base, tid, v0, w1);
      float t = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (TAIL) {
          const int at = min(base + (u * NT + tid) * E, w1 - 1) - w0;
          const uint32_t in = (sh.bits[at >> 5] >> (at & 31 & ~(E - 1))) & ((1u << E) - 1);
          if (__any(in)) v[u].mask(in);
        }
        t = max2(t, max_of(v[u]));
        v[u].keep();
      }
      if ((t - o.m) * c > 32.f) {
        o.s *= exp2_((o.m - t) * c);
        o.m = t;
      }
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          s0 += exp2_((v[u].get(e) - o.m) * c);
          s1 += exp2_((v[u].get(e + 1) - o.m) * c);
        }
      o.s += s0 + s1;
    }
    if (TAIL) sync<NT>();
  }
  return o;
}

// 2^t, t <= 0.
__device__ __forceinline__ float exp2_of(double t) {
  if (t < -160) return 0.f;
  const double n = rint(t);
  return ldexpf(exp2_((float)(t - n)), (int)n);
}

// How far the others' reference lies below the row's, to the base 2, and 2 to that
// (from 64 bits: an error here is all of the others').
struct Apart {
  double t;
  float far;
};
__device__ __forceinline__ Apart apart(float other_m, float m, double inv_t) {
  if (other_m == m) return {0, 1.f};
  const double t = ((double)other_m - m) * (inv_t * LOG2E);
  return {t, exp2_of(t)};
}

// Two at once: a thread's sum and, of the entries beside it, the row's.
struct Two {
  float a, b;
};
struct Max2 {
  static __device__ __forceinline__ Two of(Two x, Two y) { return {max2(x.a, y.a), max2(x.b, y.b)}; }
};
struct Sum2 {
  static __device__ __forceinline__ Two of(Two x, Two y) { return {x.a + y.a, x.b + y.b}; }
};
template <> __device__ __forceinline__ Two neutral<Max2, Two>() { return {-INFINITY, -INFINITY}; }
template <> __device__ __forceinline__ Two neutral<Sum2, Two>() { return {0.f, 0.f}; }

// The sums of a group's threads, or of a row's chunks.
template <int NT>
__device__ __forceinline__ Sums join(Sums o, float c, double* sh) {
  const float m = block_reduce<NT, Max>(o.m, (float*)sh);
  return {m, block_reduce<NT, Sum>(o.s * exp2_((o.m - m) * c), (float*)sh)};
}
// The same of all but the entries, and, with the entries' logits zi, each once
// (`first` tells) however often the row repeats it, of the row.
template <int NT>
__device__ __forceinline__ Sums join(Sums o, const float (&zi)[Entries<NT>::N], const bool (&first)[Entries<NT>::N], float c,
                                     double inv_t, double* sh, Sums& all, Apart& ap) {
  float in = -INFINITY;
#pragma unroll
  for (int i = 0; i < Entries<NT>::N; ++i) in = first[i] ? max2(in, zi[i]) : in;
  const Two m = block_reduce<NT, Max2>(Two{o.m, max2(o.m, in)}, (Two*)sh);
  in = 0.f;
#pragma unroll
  for (int i = 0; i < Entries<NT>::N; ++i) in += first[i] ? exp2_((zi[i] - m.b) * c) : 0.f;
  const Two s = block_reduce<NT, Sum2>(Two{o.s * exp2_((o.m - m.a) * c), in}, (Two*)sh);
  ap = apart(m.a, m.b, inv_t);
  all = {m.b, s.b + s.a * ap.far};
  return {m.a, s.a};
}

// What the gradient of a row is made of: an entry's is exp2((z - m) entry) less
// its mass, another's exp2((z - other_m) other).
struct Factors {
  float other_m, other, m, entry;
};
__device__ __forceinline__ Factors of_stats(const float* stats, int64_t r) {
  const float4 v = *(const float4*)(stats + r * LT_DISTILL_STATS);
  return {v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ void put_stats(float* stats, int64_t r, Factors f) {
  *(float4*)(stats + r * LT_DISTILL_STATS) = make_float4(f.other_m, f.other, f.m, f.entry);
}

// From the row's sum and that of all but its entries (where that is not known,
// the row's).  p_rest becomes 0 where these have nothing: all of them are -inf, or
// all the type's lowest value -- a mask -- and so far below the largest logit that
// 64 bits hold nothing of them.  Else q_rest may lie as far below as logits can:
// log_rest is its logarithm to the base 2, and with
//   q_v = q_rest r_v,  r_v = exp2((z - other_m) c) / others.s
// the gradient (P - p_rest / q_rest) q_v is (P q_rest - p_rest) r_v, which neither
// under- nor overflows.
// A sum that is not above 0 -- logits of NaN or +inf, or -inf throughout -- has no
// softmax: all of the gradient is NaN, and the loss.
constexpr double GONE = 745;               // exp(-745) is the least in 64 bits
template <class T, bool TAIL>
__device__ __forceinline__ Factors factors(Sums all, Sums others, Apart ap, double sum, double& rest, double inv_t, double& log_rest) {
  if (!TAIL) {
    const float entry = all.s > 0 ? (float)(sum * inv_t) * (1 / all.s) : NAN;
    return {all.m, entry, all.m, entry};
  }
  if (!(others.s > 0) || (others.m <= T::lowest && -ap.t > GONE * LOG2E)) rest = 0;
  const double whole = sum + rest;
  if (!(all.s > 0)) return {others.m, NAN, all.m, NAN};
  const float inv = 1 / all.s, entry = (float)(whole * inv_t) * inv, share = others.s * inv;
  log_rest = ap.t + log2_(share);             // (one logarithm: each is off by 2^-23)
  if (!(rest > 0)) return {others.m, entry * ap.far, all.m, entry};
  return {others.m, (float)((whole * (share * ap.far) - rest) * inv_t) / others.s, all.m, entry};
}

// Loss and the gradient's factors of a row from its sums (zi: the logits of the
// entries).
template <class T, bool TAIL, int NT, int N>
__device__ __forceinline__ Factors finish_row(const Entries<NT, N>& t, const float (&zi)[N], Sums all, Sums others, Apart ap, double inv_t,
                                              double* sh, float& loss) {
  const double logs = log2_(all.s), c = inv_t * LOG2E;
  double l = 0, rest = t.rest, log_rest;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (t.id[i] >= 0 && t.p[i] != 0) l += t.p[i] * (t.logp[i] - ((double)zi[i] - all.m) * c + logs);
  l = block_reduce<NT, Sum>(l, sh);
  const Factors f = factors<T, TAIL>(all, others, ap, t.sum, rest, inv_t, log_rest);
  if (TAIL && rest > 0) l += rest * (log2_((float)rest) - log_rest);
  loss = all.s > 0 ? (float)(l * LN2) : t.blank() ? 0.f : NAN;
  return f;
}

// (z: the row.)
template <class T, int NT, int N>
__device__ __forceinline__ void load_zi(const Entries<NT, N>& t, const typename T::raw* z, float (&zi)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) zi[i] = t.id[i] >= 0 ? T::get(z[t.id[i]]) : 0.f;
}

// The gradient of the logits with numbers in [v0, v1), from c0 on; w: the row's
// weight.  The entries' own are written behind a barrier over what the others
// were given.
template <class T, int NT, int U, int WINDOW, bool AGAIN>
__device__ __forceinline__ void grad_row(const typename T::raw* row, typename T::raw* grad, int lead, int c0, int v0,
                                         int v1, float c, Factors st, float w, double inv_t, const Entries<NT>& t,
                                         DistillShared<NT, WINDOW>& sh, int entries, bool past) {
  constexpr int E = Vec<T>::E, STEP = NT * U * E;
  const int tid = thread_of<NT>();
  const float out = st.other * w;
  const typename T::raw* const z = row - lead;
  typename T::raw* const g = grad - lead;
  if (t.blank()) {
    Vec<T> none;
    none.b = {};
    for (int at = c0 + tid * E; at < v1; at += NT * E) {
      if (at >= v0 && at + E <= v1) none.store(g + at);
      else none.store_part(g, at, v0, v1);
    }
    return;
  }
  for (int base = c0; base < v1; base += STEP) {
    Vec<T> v[U];
    load_step<T, NT, U, AGAIN>(v, z, base, tid, v0, v1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = exp2_((v[u].get(e) - st.other_m) * c) * out;
      v[u].put(f);
      const int at = base + (u * NT + tid) * E;
      if (at >= v0 && at + E <= v1) {
        if (past) v[u].store_past(g + at);
        else v[u].store(g + at);
      } else if (at < v1) {
        v[u].store_part(g, at, v0, v1);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < Entries<NT>::N; ++i) {
    const int j = i * NT + tid;
    if (j < MAXK) {
      sh.id[j] = t.id[i];
      sh.mass[j] = (float)(t.p[i] * inv_t);
    }
  }
  sync<NT>();
#pragma unroll
  for (int i = 0; i < Entries<NT>::N; ++i) {
    const int id = t.id[i];
    if (id < 0 || id + lead < v0 || id + lead >= v1) continue;
    int alike = 0;                         // entries with this id, itself among them
    for (int j = 0; j < entries; j += 4) {
      const int4 o = *(const int4*)&sh.id[j];
      alike += (o.x == id) + (o.y == id) + (o.z == id) + (o.w == id);
    }
    float mass = (float)(t.p[i] * inv_t);
    if (alike > 1) {
      mass = 0;
      for (int j = 0; j < entries; ++j) mass += sh.id[j] == id ? sh.mass[j] : 0.f;
    }
    grad[id] = T::put((exp2_((T::get(row[id]) - st.m) * c) * st.entry - mass) * w);
  }
}

// A block's row, and the part of it that is the block's.
#define BLOCK_HEAD                                                                                        \
  __shared__ DistillShared<NT, WINDOW> sh;                                                                \
  const int64_t blk = p.block0 + blockIdx.x, r = p.splits == 1 ? blk : blk / p.splits;                    \
  const typename T::raw* z = (const typename T::raw*)p.z.data + p.z.at(r);                                \
  const int lead = lead_of<T>(z), c0 = p.splits == 1 ? 0 : (int)(blk % p.splits) * p.chunk;               \
  const int v0 = max(lead, c0), v1 = min(lead + p.z.vocab, c0 + p.chunk);                                 \
  Entries<NT> t;                                                                                          \
  load_entries(p.t, r, p.z.vocab, p.inv_t, t, sh.sh)

// Its pass: o, the sum of all that are no entries (without the tail: of all), and
// the row's.
#define PASS                                                                                              \
  float zi[Entries<NT>::N];                                                                               \
  bool first[Entries<NT>::N] = {};                                                                        \
  load_zi<T>(t, z, zi);                                                                                   \
  Sums o, all;                                                                                            \
  Apart ap{0, 1.f};                                                                                       \
  if (threadIdx.x == 0) sh.again = 0;                                                                     \
  if (!t.blank()) {                                                                                       \
    o = sum_row<T, NT, U, WINDOW, TAIL>(z, lead, c0, v0, v1, p.c, t, sh, first);                          \
    if (TAIL && p.splits == 1) {                                                                          \
      if (sh.again) {                                                                                     \
        if ((int)threadIdx.x < MAXK) sh.id[threadIdx.x] = t.id[0];                                        \
        __syncthreads();                                                                                  \
        only_first<NT>(t, sh.id, p.t.entries, first);                                                     \
      }                                                                                                   \
      o = join<NT>(o, zi, first, p.c, p.inv_t, sh.sh, all, ap);                                           \
    } else {                                                                                              \
      all = o = join<NT>(o, p.c, sh.sh);                                                                  \
    }                                                                                                     \
  }

// Loss and statistics, or the gradient from them: one pass each, bound by memory
// (2039 x 50261 bf16, 32 entries with the tail: 50 us, 4.1 TB/s, and 66 us, 6.2
// TB/s with what of the logits is still in the last cache).
template <class T, int NT, int U, int WINDOW, bool TAIL>
__global__ __launch_bounds__(NT) void lt_distill_sums(DistillParams p) {
  BLOCK_HEAD;
  PASS;
  if (p.splits > 1) {
    if (threadIdx.x == 0) p.part[blk] = make_float2(o.m, TAIL && !t.blank() && sh.again ? -o.s : o.s);
    return;
  }
  float loss;
  const Factors st = finish_row<T, TAIL>(t, zi, all, o, ap, p.inv_t, sh.sh, loss);
  if (threadIdx.x == 0) {
    p.loss[r] = loss;
    put_stats(p.stats, r, st);
  }
}

// A row's chunks joined.
template <class T, bool TAIL>
__global__ __launch_bounds__(256) void lt_distill_join(DistillParams p) {
  constexpr int NT = 256;
  __shared__ DistillShared<NT, 32> sh;
  const int64_t r = p.block0 + blockIdx.x;
  Entries<NT> t;
  load_entries(p.t, r, p.z.vocab, p.inv_t, t, sh.sh);
  Sums o;
  bool again = false;
  if ((int)threadIdx.x < p.splits) {       // (at most NT chunks)
    const float2 part = p.part[r * p.splits + threadIdx.x];
    o.m = part.x;
    o.s = fabsf(part.y);
    again = signbit(part.y);
  }
  float zi[Entries<NT>::N];
  load_zi<T>(t, (const typename T::raw*)p.z.data + p.z.at(r), zi);
  Sums all;
  Apart ap{0, 1.f};
  if (TAIL) {
    bool first[1] = {t.id[0] >= 0};
    sh.id[threadIdx.x] = t.id[0];
    if (__syncthreads_or(again)) only_first<NT>(t, sh.id, p.t.entries, first);
    o = join<NT>(o, zi, first, p.c, p.inv_t, sh.sh, all, ap);
  } else {
    all = o = join<NT>(o, p.c, sh.sh);
  }
  float loss;
  const Factors st = finish_row<T, TAIL>(t, zi, all, o, ap, p.inv_t, sh.sh, loss);
  if (threadIdx.x == 0) {
    p.loss[r] = loss;
    put_stats(p.stats, r, st);
  }
}

template <class T, int NT, int U, int WINDOW>
__global__ __launch_bounds__(NT) void lt_distill_grad(DistillParams p) {
  BLOCK_HEAD;
  grad_row<T, NT, U, WINDOW, false>(z, (typename T::raw*)p.grad.data + p.grad.at(r), lead, c0, v0, v1, p.c,
                                    of_stats(p.stats, r), weight_of(p, r), p.inv_t, t, sh, p.t.entries, p.past);
}

// Both: the second pass finds the row in the caches.  It reads past them, and
// the gradient is written past them: kept, they push out the rows that other
// blocks are about to read again (4096 x 131072 bf16: 570 us; with the stores
// past the caches 500, with the loads too 467, 4.6 TB/s; 32768 x 16000: 518 and
// 464).
template <class T, int NT, int U, int WINDOW, bool TAIL>
__global__ __launch_bounds__(NT, 8) void lt_distill_both(DistillParams p) {
  BLOCK_HEAD;
  PASS;
  float loss;
  const Factors st = finish_row<T, TAIL>(t, zi, all, o, ap, p.inv_t, sh.sh, loss);
  if (threadIdx.x == 0) p.loss[r] = loss;
  grad_row<T, NT, U, WINDOW, true>(z, (typename T::raw*)p.grad.data + p.grad.at(r), lead, c0, v0, v1, p.c, st,
                                   weight_of(p, r), p.inv_t, t, sh, p.t.entries, p.past);
}

// Rows that a wave holds in its registers, U vectors a lane: read once, their
// exponentials too taken once for the loss and the gradient.  N * 64 entries at
// most.  The sum within the entries is that of the entries' own logits, each
// once; the row's others are summed beside the largest of their own, with -inf in
// the entries' places (a mask of bits in LDS tells them).
template <int N>
struct WaveShared {
  uint32_t bits[128];
  int id[N * 64];
  float mass[N * 64];
};

// (Of 16-bit rows up to 2048 with many entries and the tail the compiler takes one
// register more than six waves a SIMD leave: 65536 x 2000 bf16, 100 entries 152 us
// by six, 159 by five.)
template <class T, class V, int U, int N, bool TAIL, bool LOSS, bool GRAD>
__global__ __launch_bounds__(256, (TAIL && N > 1 && U == 4 && V::E == 8 ? 6 : 1)) void lt_distill_wave(DistillParams p) {
  using raw = typename T::raw;
  constexpr int E = V::E;
  __shared__ WaveShared<N> shared[4];
  WaveShared<N>& sh = shared[group_of<64>()];
  const int lane = threadIdx.x & 63, vocab = p.z.vocab;
  const int64_t r = (p.block0 + blockIdx.x) * 4 + group_of<64>();
  if (r >= p.rows) return;                 // (a wave as a whole)
  const raw* const x = (const raw*)p.z.data + p.z.at(r);
  V v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * 64 + lane) * E;
    if ((u + 1) * 64 * E <= vocab) v[u].load(x + at);
    else v[u].load(x, at, 0, vocab, T::put(-INFINITY));
  }
  Entries<64, N> t;
  load_entries(p.t, r, vocab, p.inv_t, t, nullptr);
  const bool blank = t.blank();
  float zi[N];
  load_zi<T>(t, x, zi);
  // a bit for each logit that is an entry; `first`: of those with this id
  bool first[N];
  for (int i = lane; i < U * 2 * E; i += 64) sh.bits[i] = 0;
  sync<64>();
#pragma unroll
  for (int i = 0; i < N; ++i)
    first[i] = t.id[i] >= 0 && !(atomicOr(&sh.bits[t.id[i] >> 5], 1u << (t.id[i] & 31)) >> (t.id[i] & 31) & 1);
  sync<64>();
  Factors st{0.f, 0.f, 0.f, 0.f};
  if (LOSS) {
    float m = -INFINITY, in = -INFINITY;
    if (TAIL) {
#pragma unroll
      for (int i = 0; i < N; ++i) in = first[i] ? max2(in, zi[i]) : in;
      in = wave_reduce<Max>(in, -INFINITY);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (TAIL) {
        const int at = min((u * 64 + lane) * E, vocab - 1);
        v[u].mask(sh.bits[at >> 5] >> (at & 31 & ~(E - 1)));
      }
      m = max2(m, max_of(v[u]));
      v[u].keep();
    }
    st.other_m = max2(wave_reduce<Max>(m, -INFINITY), LOWEST);
    st.m = TAIL ? max2(st.other_m, in) : st.other_m;
  } else {
    st = of_stats(p.stats, r);
  }
  float f[U][E], out[2] = {0.f, 0.f};
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      f[u][e] = exp2_((v[u].get(e) - st.other_m) * p.c);
      if (LOSS) out[e & 1] += f[u][e];
    }
  if (LOSS) {
    Sums rest{st.other_m, wave_reduce<Sum>(out[0] + out[1], 0.f)}, all = rest;
    Apart ap{0, 1.f};
    if (TAIL) {
      float in = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) in += first[i] ? exp2_((zi[i] - st.m) * p.c) : 0.f;
      ap = apart(rest.m, st.m, p.inv_t);
      all = {st.m, wave_reduce<Sum>(in, 0.f) + rest.s * ap.far};
    }
    float loss;
    st = finish_row<T, TAIL>(t, zi, all, rest, ap, p.inv_t, nullptr, loss);
    if (lane == 0) {
      p.loss[r] = blank ? 0.f : loss;
      if (!GRAD) put_stats(p.stats, r, st);
    }
  }
  if (!GRAD) return;
  const float w = weight_of(p, r), all = st.other * w;
  raw* const g = (raw*)p.grad.data + p.grad.at(r);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * 64 + lane) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) f[u][e] = blank ? 0.f : f[u][e] * all;
    if constexpr (E == 1) {
      if (at < vocab) g[at] = T::put(f[u][0]);
    } else {
      v[u].put(f[u]);
      if (at + E <= vocab) v[u].store(g + at);
      else if (at < vocab) v[u].store_part(g, at, 0, vocab);
    }
  }
  if (blank) return;
  // the entries' own, over that
  float mass[N];
  bool again = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mass[i] = (float)(t.p[i] * p.inv_t);
    again |= t.id[i] >= 0 && !first[i];
  }
  if (__any(again)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      sh.id[i * 64 + lane] = t.id[i];
      sh.mass[i * 64 + lane] = mass[i];
      mass[i] = 0;
    }
    sync<64>();
#pragma nounroll
    for (int j = 0; j < p.t.entries; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) mass[i] += sh.id[j] == t.id[i] ? sh.mass[j] : 0.f;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (t.id[i] >= 0) g[t.id[i]] = T::put((exp2_((zi[i] - st.m) * p.c) * st.entry - mass[i]) * w);
}

// Rows of at most FEW logits: a thread a row, the row in LDS, its entries a
// mask of 64 bits.  The others' sum is taken with the row's, and again beside the
// largest of their own where it is LITTLE beside that: there its exponents'
// roundings cost more than 2^-18 of it, further down it vanishes.  The gradient is
// made of the logits alone (no stats).  131072 x
// 41 float32, 5 entries: loss 20 us, gradient 26, where reading the logits and
// writing the gradient take 4 each: two waves a SIMD, 7 and 10 us of instructions
// and the rest waiting, for the entries' loads foremost.
constexpr float LITTLE = 0x1p-24f;

template <class T, bool LOSS, bool GRAD>
__global__ __launch_bounds__(64) void lt_distill_few(DistillParams p) {
  using raw = typename T::raw;
  extern __shared__ float few[];           // [64][few_pitch(vocab)]
  const int lane = threadIdx.x, vocab = p.z.vocab, pitch = few_pitch(vocab), n = p.t.entries;
  const int64_t r0 = (p.block0 + blockIdx.x) * 64;
  const int rows = (int)min((int64_t)64, p.rows - r0);
  load_few<T>(p.z, r0, rows, few, pitch);
  __syncthreads();
  const int64_t r = r0 + min(lane, rows - 1);
  float* z = few + min(lane, rows - 1) * pitch;
  const int64_t first = r * n;
  const double c = p.inv_t * LOG2E;
  // (the entries are read again where they are used: a cache line or two a row)
  auto entry = [&](int j, int& id, double& v) {
    const int64_t i = any_id(p.t.ids, first + j, p.t.ids_bytes);
    if (i < 0 || i >= vocab) return false;
    id = (int)i;
    v = any_float(p.t.top, first + j, p.t.top_dtype) * c;
    return true;
  };
  int id = 0;
  double v, ref = -INFINITY, sum = 0, rest = 0, norm = 0;
  uint64_t mask = 0;
  if (p.t.top_lse) ref = p.t.top_lse[r] * LOG2E;
  else
    for (int j = 0; j < n; ++j)
      if (entry(j, id, v)) ref = v > ref || v != v ? v : ref;
  if (!p.t.top_lse && ref == -INFINITY) ref = 0;
  for (int j = 0; j < n; ++j)
    if (entry(j, id, v)) {
      mask |= 1ull << id;
      const double pj = exp2_or_0(v - ref);
      sum += p.t.top_lse && pj == 0 ? TRACE : pj;
    }
  if (p.t.top_lse) {
    if (sum > 0 && sum < 1) rest = 1 - sum;
  } else if (sum != 0) {
    norm = log2_((float)sum);
    sum = sum > 0 ? 1 : sum;               // (a NaN stays)
  }
  const bool blank = sum == 0 && rest == 0;
  Sums all, others;
  for (int i = 0; i < vocab; i += 4) all.m = max2(max3(all.m, z[i], z[i + 1]), max2(z[i + 2], z[i + 3]));
  others.m = all.m;
  for (int i = 0; i < vocab; i += 4) {
    float e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = exp2_((z[i + j] - all.m) * p.c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool entry = mask >> (i + j) & 1;
      all.s += entry ? e[j] : 0.f;
      others.s += entry ? 0.f : e[j];
    }
  }
  all.s += others.s;
  if (__builtin_expect(rest > 0 && others.s < LITTLE, 0)) {
    others = Sums{};
    for (int i = 0; i < vocab; i += 4) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = mask >> (i + j) & 1 ? -INFINITY : z[i + j];
      others.m = max2(max3(others.m, f[0], f[1]), max2(f[2], f[3]));
    }
    for (int i = 0; i < vocab; i += 4) {
      float f[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = exp2_(((mask >> (i + j) & 1 ? -INFINITY : z[i + j]) - others.m) * p.c);
      others.s += (f[0] + f[1]) + (f[2] + f[3]);
    }
  }
  double log_rest;
  const Factors st = factors<T, true>(all, others, apart(others.m, all.m, p.inv_t), sum, rest, p.inv_t, log_rest);
  if (LOSS) {
    double loss = 0;
    const double logs = log2_(all.s);
    for (int j = 0; j < n; ++j)
      if (entry(j, id, v)) {
        const double logp = v - ref - norm, pj = exp2_or_0(logp);
        if (pj != 0) loss += pj * (logp - ((double)z[id] - all.m) * c + logs);
      }
    if (rest > 0) loss += rest * (log2_((float)rest) - log_rest);
    if (lane < rows) {
      p.loss[r] = all.s > 0 ? (float)(loss * LN2) : blank ? 0.f : NAN;
      if (p.stats) put_stats(p.stats, r, st);
    }
  }
  if (GRAD) {
    const float w = weight_of(p, r);
    if (lane < rows) {
      // (two references in a row are rare: for a wave without, one less selection)
      auto each = [&](auto two) {
        for (int i = 0; i < vocab; i += 4) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool entry = mask >> (i + j) & 1;
            e[j] = exp2_((z[i + j] - (decltype(two)::value && entry ? st.m : st.other_m)) * p.c) * (entry ? st.entry : st.other) * w;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) z[i + j] = blank ? 0.f : e[j];
        }
      };
      if (__any(st.m != st.other_m)) each(std::true_type());
      else each(std::false_type());
      for (int j = 0; j < n && !blank; ++j)
        if (entry(j, id, v)) z[id] -= (float)(exp2_or_0(v - ref - norm) * p.inv_t) * w;
    }
    __syncthreads();
    raw* const g = (raw*)p.grad.data;
    if (p.grad.inner == 1 && p.grad.stride_outer == vocab)
      each_of_rows(rows, vocab, [&](int r, int v, int i) { g[r0 * vocab + i] = T::put(few[r * pitch + v]); });
    else
      each_of_rows(rows, vocab, [&](int r, int v, int) { g[p.grad.at(r0 + r) + v] = T::put(few[r * pitch + v]); });
  }
}

// ---- host ------------------------------------------------------------------
enum Pass { SUMS, GRAD, BOTH };

// Chunks of a row, of a whole number of steps of a block.
void split_rows(DistillParams& p, int step, int64_t n) {
  const int64_t steps = (p.z.vocab + LEAD + n * step - 1) / (n * step);
  p.chunk = (int32_t)(n <= 1 ? 0x7fffff80 : steps * step);
  p.splits = (int32_t)(((int64_t)p.z.vocab + LEAD + p.chunk - 1) / p.chunk);
}

// For the sums: one where the rows fill the card or a row is a few steps --
// chunks have to be joined, in a launch of its own.  (Loss and gradient of 8 x
// 32000 bf16 in one launch 11 us, in three 16 and the gaps between them; of 64 x
// 131072 in three 25 us, in one 28; of 200 42 and 39.)
void split_sums(DistillParams& p, int dtype) {
  const int step = 512 * 4 * (dtype == LT_F32 ? 4 : 8);
  int64_t n = 1;
  if (p.z.vocab > 6 * step && p.rows < 256) {
    n = (p.z.vocab + step - 1) / step;
    n = n < 512 / p.rows ? n : 512 / p.rows;
    n = n < 256 ? n : 256;
  }
  split_rows(p, step, n);
}

// For the gradient, which needs no joining: blocks enough for the card.  (Loss and
// gradient of 64 x 131072 bf16 25 us, with a block a row's gradient 31; of 200 42
// and 43.)
void split_grad(DistillParams& p, int dtype) {
  const int step = 512 * 4 * (dtype == LT_F32 ? 4 : 8);
  int64_t n = 1;
  if (p.z.vocab > 16384 && p.rows < 512) {
    n = (p.z.vocab + step - 1) / step;
    n = n < 1024 / p.rows ? n : 1024 / p.rows;
  }
  split_rows(p, step, n);
}

// (whole 16 bytes: the statistics lie behind them)
int64_t parts_bytes(const DistillParams& p) { return p.splits == 1 ? 0 : (p.rows * p.splits * (int64_t)sizeof(float2) + 15) / 16 * 16; }

template <class T, int NT, int U, int WINDOW>
lt_status launch_block(const DistillParams& p, Pass pass, void* stream, const char* what) {
  const int64_t blocks = p.rows * p.splits;
  if (pass == GRAD) return launch(lt_distill_grad<T, NT, U, WINDOW>, blocks, NT, p, stream, what);
  if (pass == SUMS)
    return p.t.top_lse ? launch(lt_distill_sums<T, NT, U, WINDOW, true>, blocks, NT, p, stream, what)
                       : launch(lt_distill_sums<T, NT, U, WINDOW, false>, blocks, NT, p, stream, what);
  return p.t.top_lse ? launch(lt_distill_both<T, NT, U, WINDOW, true>, blocks, NT, p, stream, what)
                     : launch(lt_distill_both<T, NT, U, WINDOW, false>, blocks, NT, p, stream, what);
}

template <class T, class V, int U, int N, bool TAIL>
lt_status launch_wave(const DistillParams& p, Pass pass, void* stream, const char* what) {
  const int64_t blocks = (p.rows + 3) / 4;
  return pass == SUMS   ? launch(lt_distill_wave<T, V, U, N, TAIL, true, false>, blocks, 256, p, stream, what)
         : pass == GRAD ? launch(lt_distill_wave<T, V, U, N, false, false, true>, blocks, 256, p, stream, what)
                        : launch(lt_distill_wave<T, V, U, N, TAIL, true, true>, blocks, 256, p, stream, what);
}

// (Room for 64 entries or 256: 65536 x 200 bf16, 8 entries 48 us and 53.)
template <class T, class V, int U>
lt_status launch_wave(const DistillParams& p, Pass pass, void* stream, const char* what) {
  if (p.t.entries <= 64)
    return p.t.top_lse ? launch_wave<T, V, U, 1, true>(p, pass, stream, what) : launch_wave<T, V, U, 1, false>(p, pass, stream, what);
  return p.t.top_lse ? launch_wave<T, V, U, 4, true>(p, pass, stream, what) : launch_wave<T, V, U, 4, false>(p, pass, stream, what);
}

template <class T>
lt_status launch_pass(const DistillParams& p, Pass pass, void* stream, const char* what) {
  // Rows of few logits, and enough of them: a thread a row, which goes through
  // its entries one after another.  (Loss and gradient of float32, us, a wave a
  // row the second: 131072 x 41, 3 entries 24, 70; 12 entries 44, 68; 16384 x 41,
  // 12 entries 28, 17.)
  if (p.z.vocab <= FEW && p.rows >= 65536 && p.t.entries <= 16) {
    const int64_t blocks = (p.rows + 63) / 64;
    const int lds = 64 * few_pitch(p.z.vocab) * 4;
    return pass == SUMS   ? launch(lt_distill_few<T, true, false>, blocks, 64, p, stream, what, lds)
           : pass == GRAD ? launch(lt_distill_few<T, false, true>, blocks, 64, p, stream, what, lds)
                          : launch(lt_distill_few<T, true, true>, blocks, 64, p, stream, what, lds);
  }
  // Rows that fit a wave's registers.  (65536 x 2000 bf16, 32 entries: 120 us, 4.5
  // TB/s; 65536 x 200, 8 entries: 48, by its instructions; a wave that reads the
  // row twice 190 and 82.  16384 x 4000: 55 us, a block of 256 threads 105.)
  using W = Vec<T>;
  if (p.z.vocab <= 128) return launch_wave<T, One<T>, 2>(p, pass, stream, what);
  if (p.z.vocab <= 256) return launch_wave<T, One<T>, 4>(p, pass, stream, what);
  if (p.z.vocab <= 64 * W::E) return launch_wave<T, W, 1>(p, pass, stream, what);
  if (p.z.vocab <= 128 * W::E) return launch_wave<T, W, 2>(p, pass, stream, what);
  if (p.z.vocab <= 256 * W::E) return launch_wave<T, W, 4>(p, pass, stream, what);
  if (p.z.vocab <= 512 * W::E) return launch_wave<T, W, 8>(p, pass, stream, what);
  // (4096 x 8000 bf16: 39 us by 256 threads, 56 by 512; 4096 x 131072: 504 and 467.)
  if (p.z.vocab <= 16384) return launch_block<T, 256, 4, 16384>(p, pass, stream, what);
  const lt_status st = launch_block<T, 512, 4, 1 << 18>(p, pass, stream, what);
  if (st != LT_OK || pass != SUMS || p.splits == 1) return st;
  return p.t.top_lse ? launch(lt_distill_join<T, true>, p.rows, 256, p, stream, what)
                     : launch(lt_distill_join<T, false>, p.rows, 256, p, stream, what);
}

lt_status launch_pass(const DistillParams& p, int dtype, Pass pass, void* stream, const char* what) {
  return dtype == LT_F32   ? launch_pass<F32>(p, pass, stream, what)
         : dtype == LT_F16 ? launch_pass<F16>(p, pass, stream, what)
                           : launch_pass<BF16>(p, pass, stream, what);
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

lt_status grad_check(const lt_rows* z, const lt_rows* g, double scale, int64_t weight_stride) {
  lt_status st;
  if (!rows_ok(g, "grad", &st)) return st;
  if (g->rows != z->rows || g->vocab != z->vocab || g->dtype != z->dtype || g->device != z->device)
    BAD("grad: not the logits' rows, vocab, dtype and device");
  if (z->rows > 0 && !g->data) BAD("grad: NULL");
  if (!isfinite(scale)) BAD("scale %g", scale);
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
  split_sums(p, z->dtype);
  // Logits and gradient of more than the last cache's 256 MB: by the time that
  // the gradient is read, it would be gone; a smaller one is left there.
  p.past = 2 * p.rows * p.z.vocab * dtype_bytes(z->dtype) > (int64_t)256 << 20;
  return p;
}

bool workspace_ok(const DistillParams& p, const void* at, int64_t bytes) {
  return p.splits == 1 || (at && (uintptr_t)at % 16 == 0 && bytes >= p.rows * LT_DISTILL_STATS * (int64_t)sizeof(float) + parts_bytes(p));
}

}  // namespace

extern "C" {

int64_t lt_distill_workspace(const lt_rows* z, int32_t) {
  if (!z || z->rows < 1 || z->vocab < 1 || z->vocab > LT_MAX_VOCAB) return 0;
  DistillParams p{};
  p.z = rows_of(z);
  p.rows = z->rows;
  split_sums(p, z->dtype);
  return p.splits == 1 ? 0 : p.rows * LT_DISTILL_STATS * (int64_t)sizeof(float) + parts_bytes(p);
}

lt_status lt_distill_forward(const lt_rows* z, const lt_teacher* t, double temperature, float* loss, float* stats,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const lt_status st = distill_check(z, t, temperature);
  if (st != LT_OK || z->rows == 0) return st;
  if (!loss || !stats || (uintptr_t)stats % 16) BAD("output: NULL, or stats not 16 B aligned");
  DistillParams p = distill_params(z, t, temperature);
  if (!workspace_ok(p, workspace, workspace_bytes))
    BAD("workspace: %lld bytes, 16 B aligned, are needed", (long long)lt_distill_workspace(z, t->entries));
  p.part = (float2*)workspace;
  p.loss = loss;
  p.stats = stats;
  ON_DEVICE(z->device);
  return launch_pass(p, z->dtype, SUMS, stream, "lt_distill_forward");
}

lt_status lt_distill_backward(const lt_rows* z, const lt_teacher* t, double temperature, const float* stats,
                              double scale, const float* weight, int64_t weight_stride, const lt_rows* grad,
                              void* stream) {
  lt_status st = distill_check(z, t, temperature);
  if (st == LT_OK) st = grad_check(z, grad, scale, weight_stride);
  if (st != LT_OK || z->rows == 0) return st;
  if (!stats || (uintptr_t)stats % 16) BAD("stats: NULL or not 16 B aligned");
  DistillParams p = distill_params(z, t, temperature);
  p.stats = const_cast<float*>(stats);
  p.scale = (float)scale;
  p.weight = weight;
  p.weight_stride = weight_stride;
  p.grad = rows_of(grad);
  split_grad(p, z->dtype);
  ON_DEVICE(z->device);
  return launch_pass(p, z->dtype, GRAD, stream, "lt_distill_backward");
}

lt_status lt_distill_fused(const lt_rows* z, const lt_teacher* t, double temperature, double scale,
                           const float* weight, int64_t weight_stride, float* loss, const lt_rows* grad,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  lt_status st = distill_check(z, t, temperature);
  if (st == LT_OK) st = grad_check(z, grad, scale, weight_stride);
  if (st != LT_OK || z->rows == 0) return st;
  if (!loss) BAD("output: NULL");
  DistillParams p = distill_params(z, t, temperature);
  if (!workspace_ok(p, workspace, workspace_bytes))
    BAD("workspace: %lld bytes, 16 B aligned, are needed", (long long)lt_distill_workspace(z, t->entries));
  p.part = (float2*)workspace;
  p.loss = loss;
  p.stats = p.splits > 1 ? (float*)((char*)workspace + parts_bytes(p)) : nullptr;
  p.scale = (float)scale;
  p.weight = weight;
  p.weight_stride = weight_stride;
  p.grad = rows_of(grad);
  ON_DEVICE(z->device);
  if (p.splits == 1) return launch_pass(p, z->dtype, BOTH, stream, "lt_distill_fused");
  st = launch_pass(p, z->dtype, SUMS, stream, "lt_distill_fused");
  split_grad(p, z->dtype);
  return st != LT_OK ? st : launch_pass(p, z->dtype, GRAD, stream, "lt_distill_fused");
}

}  // extern "C"
