// lt_verify.hip -- the verification of drafted tokens
// (include/lattice_logits.h lt_verify_draft).
//
// A token is drawn where a running sum over the vocabulary crosses a line, so a
// relative error e of the sums moves it with a probability of about e times the
// number of tokens that the line may fall beside: 131072 e.  A float32
// exponential (1e-7) would move one in a hundred; all sums are held in 64 bits
// and the exponential is good to 1.1e-12.  It is what bounds these kernels: 18
// instructions a logit, where memory would allow 14.
#include "lt_logits.h"

namespace {

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

// Four at a time: a step of one takes 8 cycles or more until the next may use
// it, and few waves are there to fill them.
__device__ __forceinline__ void exp2_64(double (&t)[4]) {
  constexpr double BIG = 6755399441055744.0;
  constexpr double C[9] = {0.9999999999999997, 0.6931471805459343, 0.24022650695821055, 0.055504109412010456, 0.009618129157656703,
                           0.0013333450573018062, 0.00015403457039410448, 1.531007807039615e-05, 1.325497460306718e-06};
  double b[4], r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = t[i] + BIG;
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] -= b[i] - BIG;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = fma(C[8], t[i], C[7]);
#pragma unroll
  for (int k = 6; k >= 0; --k)
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fma(r[i], t[i], C[k]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, r[i]);
    const uint32_t hi = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(uint64_t, b[i]) << 20);
    t[i] = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)bits);
  }
}

// exp2((x - m) c) of logits no further than 1000 (in the exponent) below m;
// lower ones are taken as that: 1e-301.
constexpr double DEPTH = 1000;
__device__ __forceinline__ float floor_of(float m, double c) { return (float)fmax((double)m - DEPTH / c, (double)LOWEST); }
__device__ __forceinline__ double soft_exp(float x, float floor, double m, double c) {
  return exp2_64(((double)max2(x, floor) - m) * c);
}

// Where a sequence stops, for the kernels that follow.
struct StopNote {
  double ps, qs;          // sums of the target's row, of the drafter's
  float pm, qm;
  int32_t a, pad;
};

struct VerifyParams {
  int64_t block0;         // of this launch
  Rows target, draft;     // draft.data NULL: certain tokens
  const void* ids;
  const float* accept_u;
  const float* sample_u;
  const int32_t* lengths;
  int64_t batch;
  int32_t drafts, ids_bytes;
  double c;               // log2(e) / temperature
  int64_t* tokens;
  int64_t* accepted;
  int32_t splits, chunk;  // blocks of a row, a block's numbers of it
  int32_t segments;       // of a row: 64 vectors each
  int32_t weigh_splits, weigh_chunk;       // of the row that the token is drawn from
  double* weight;         // [batch][segments]: the weights' sums
  struct StopNote* stop;  // [batch]
  double2* part;          // [batch * (2 drafts + 1)][splits]: reference and sum, targets first
};

// A row's softmax: exp2((x - m) c) * inv, inv 0 for a row of -inf; 0 below the
// floor.
struct Soft {
  float m = LOWEST, floor = LOWEST;
  double s = 0, inv = 0;
  __device__ __forceinline__ double of(float x, double c) const { return x >= floor ? soft_exp(x, floor, m, c) * inv : 0; }
  __device__ __forceinline__ void finish(double c) {
    floor = floor_of(m, c);
    inv = s > 0 ? 1 / s : 0;
  }
};

// The sum of exp2((x - m) c) over a row's numbers [v0, v1), from c0 on; a
// thread's m is any logit not far below its largest.
template <class T, int NT, int U>
__device__ __forceinline__ Soft soft_part(const typename T::raw* row, int lead, int c0, int v0, int v1, double c,
                                          float* shf, double* shd) {
  constexpr int E = Vec<T>::E, STEP = NT * U * E;
  Soft o;
  for (int base = c0; base < v1; base += STEP) {
    Vec<T> v[U];
    load_step<T, NT, U>(v, row - lead, base, threadIdx.x, v0, v1);
    float t = LOWEST;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      t = max2(t, max_of(v[u]));
      v[u].keep();
    }
    if (((double)t - o.m) * c > 300) {
      o.s *= exp2_64(fmax(((double)o.m - t) * c, -DEPTH));
      o.m = t;
      o.floor = floor_of(t, c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        double t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = ((double)max2(v[u].get(e + i), o.floor) - o.m) * c;
        exp2_64(t);
        o.s += (t[0] + t[1]) + (t[2] + t[3]);
      }
  }
  const float m = block_reduce<NT, Max>(o.m, shf);
  o.s = block_reduce<NT, Sum>(o.m > -1e38f ? o.s * exp2_64(fmax(((double)o.m - m) * c, -DEPTH)) : 0, shd);
  o.m = m;
  if (m <= -1e38f) {
    // nothing but -inf and the type's lowest value: of these the sum above
    // made one
    double s = 0;
    for (int at = v0 + threadIdx.x; at < v1; at += NT) {
      const float x = T::get(row[at - lead]);
      if (x >= LOWEST) s += exp2_64(fmax(((double)x - m) * c, -DEPTH));
    }
    o.s = block_reduce<NT, Sum>(s, shd);
  }
  o.finish(c);
  return o;
}

// Where a sequence stops: its rows there, and what the next token is drawn by.
template <class T>
struct Stop {
  const typename T::raw *x = nullptr, *y = nullptr;        // the target's row; the drafter's
  Soft p, q;
  int64_t id = -1;        // the token that was not accepted
  bool minus = false;     // weight max(p - q, 0); else p
  __device__ __forceinline__ double weight(float fx, float fy, int v, double c) const {
    const double w = p.of(fx, c);
    if (!minus) return w;
    return fmax(w - (y ? q.of(fy, c) : v == id ? 1.0 : 0.0), 0.0);
  }
};

// The weights' sums of 64 vectors each, of the numbers [v0, v1) from c0 on.
template <class T, int NT>
__device__ __forceinline__ void weigh(const Stop<T>& st, int vocab, int c0, int c1, double c, double* weight) {
  constexpr int E = Vec<T>::E;
  const int lead = lead_of<T>(st.x), v1 = min(c1, lead + vocab);
  const typename T::raw* const x = st.x - lead;
  const typename T::raw* const y = st.y ? st.y - lead : nullptr;       // (at any address)
  for (int base = c0; base < v1; base += NT * E) {
    const int at = base + threadIdx.x * E;
    Vec<T> vx, vy;
    vx.load(x, at, lead, lead + vocab, T::put(-INFINITY));
    if (st.minus && y) vy.load(y, at, lead, lead + vocab, T::put(-INFINITY));
    else vy = vx;
    double s = 0;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      double t[4], q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = ((double)max2(vx.get(e + i), st.p.floor) - st.p.m) * c;
      exp2_64(t);
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = vx.get(e + i) >= st.p.floor ? t[i] * st.p.inv : 0;
      if (st.minus && y) {
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = ((double)max2(vy.get(e + i), st.q.floor) - st.q.m) * c;
        exp2_64(q);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = fmax(t[i] - (vy.get(e + i) >= st.q.floor ? q[i] * st.q.inv : 0), 0.0);
      } else if (st.minus) {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = at + e + i - lead == st.id ? fmax(t[i] - 1.0, 0.0) : t[i];
      }
      s += (t[0] + t[1]) + (t[2] + t[3]);
    }
    s = wave_reduce<Sum>(s, 0.0);
    if ((threadIdx.x & 63) == 0 && at < v1) weight[at / (64 * E)] = s;
  }
}

// The token: the first whose running sum of weights passes u of the whole,
// else the last with a weight.  All of a block gets it.
template <class T, int NT>
__device__ __forceinline__ int draw(Stop<T>& st, int vocab, float u, double c, const double* weight, int segments,
                                    double* shd, int* shi) {
  constexpr int SEG = 64 * Vec<T>::E;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lead = lead_of<T>(st.x);
  // sums of the segments, `before` each NT of them, in their order
  auto scan = [&](double w, double before, double& all) {
    double cum = wave_scan<Sum>(w, 0.0);
    if (lane == 63) shd[wave] = cum;
    __syncthreads();
    cum += before;
    all = before;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
      if (i < wave) cum += shd[i];
      all += shd[i];
    }
    __syncthreads();
    return cum;
  };
  double total = 0;
  for (int s0 = 0; s0 < segments; s0 += NT) total += s0 + tid < segments ? weight[s0 + tid] : 0.0;
  total = block_reduce<NT, Sum>(total, shd);
  int begin = lead, end = lead + vocab;
  double before = 0;
  const bool whole = !(total > 0);         // p and q alike: then it is drawn by p
  if (whole) {
    st.minus = false;
    total = st.p.inv > 0 ? 1 : 0;
  }
  const double line = u * total;
  if (!whole) {
    if (tid == 0) shi[0] = 0x7fffffff, shi[1] = -1;
    __syncthreads();
    double ahead = 0;
    for (int s0 = 0; s0 < segments; s0 += NT) {
      const int s = s0 + tid;
      const double w = s < segments ? weight[s] : 0.0;
      double all;
      const double cum = scan(w, ahead, all);
      if (w > 0) {
        if (cum > line) atomicMin(&shi[0], s);
        atomicMax(&shi[1], s);
      }
      ahead = all;
    }
    __syncthreads();
    const int s = shi[0] != 0x7fffffff ? shi[0] : shi[1];
    __syncthreads();
    // what lies before it, summed as above
    double part = 0;
    for (int s0 = 0; s0 < s; s0 += NT) {
      double all;
      (void)scan(s0 + tid < s ? weight[s0 + tid] : 0.0, part, all);
      part = all;
    }
    before = part;
    begin = max(begin, s * SEG);
    end = min(end, (s + 1) * SEG);
  }
  if (tid == 0) shi[0] = 0x7fffffff, shi[1] = -1;
  __syncthreads();
  for (int base = begin; base < end; base += NT) {
    const int at = base + tid, v = at - lead;
    double w = 0;
    if (at < end) w = st.weight(T::get(st.x[v]), st.y ? T::get(st.y[v]) : 0.f, v, c);
    double all;
    const double cum = scan(w, before, all);
    if (w > 0) {
      if (cum > line) atomicMin(&shi[0], v);
      atomicMax(&shi[1], v);
    }
    before = all;
    __syncthreads();
    if (shi[0] != 0x7fffffff) break;
  }
  __syncthreads();
  return shi[0] != 0x7fffffff ? shi[0] : shi[1];
}

template <class T>
__device__ __forceinline__ const typename T::raw* target_row(const VerifyParams& p, int64_t b, int i) {
  return (const typename T::raw*)p.target.data + p.target.at(b * (p.drafts + 1) + i);
}
template <class T>
__device__ __forceinline__ const typename T::raw* draft_row(const VerifyParams& p, int64_t b, int i) {
  return (const typename T::raw*)p.draft.data + p.draft.at(b * p.drafts + i);
}
__device__ __forceinline__ int length_of(const VerifyParams& p, int64_t b) {
  return p.lengths ? max(0, min(p.lengths[b], p.drafts)) : p.drafts;
}

template <int NT>
__device__ __forceinline__ void write_tokens(const VerifyParams& p, int64_t b, int a, int token) {
  if (threadIdx.x == 0) p.accepted[b] = a;
  for (int i = threadIdx.x; i <= p.drafts; i += NT)
    p.tokens[b * (p.drafts + 1) + i] = i < a ? any_id(p.ids, b * p.drafts + i, p.ids_bytes) : i == a ? token : -1;
}

// Batches that fill the card: a block takes a sequence, row by row up to where
// it stops; what lies behind is not read.
template <class T, int NT, int U>
__global__ __launch_bounds__(NT, 4) void lt_verify_walk(VerifyParams p) {
  __shared__ float shf[NT / 64];
  __shared__ double shd[NT / 64];
  __shared__ int shi[2];
  const int V = p.target.vocab;
  const int64_t b = p.block0 + blockIdx.x;
  const int n = length_of(p, b);
  Stop<T> st;
  int a = 0;
  for (;; ++a) {
    st.x = target_row<T>(p, b, a);
    int lead = lead_of<T>(st.x);
    st.p = soft_part<T, NT, U>(st.x, lead, 0, lead, lead + V, p.c, shf, shd);
    st.y = nullptr;
    if (a == n) break;
    st.id = any_id(p.ids, b * p.drafts + a, p.ids_bytes);
    const bool there = st.id >= 0 && st.id < V;
    double q = 1;
    if (p.draft.data) {
      st.y = draft_row<T>(p, b, a);
      lead = lead_of<T>(st.y);
      st.q = soft_part<T, NT, U>(st.y, lead, 0, lead, lead + V, p.c, shf, shd);
      q = there ? st.q.of(T::get(st.y[st.id]), p.c) : 0.0;
    }
    st.minus = true;
    if (!(there && p.accept_u[b * p.drafts + a] * q < st.p.of(T::get(st.x[st.id]), p.c))) break;
    st.minus = false;
  }
  double* const weight = p.weight + b * p.segments;
  const int lead = lead_of<T>(st.x), segments = (lead + V + 64 * Vec<T>::E - 1) / (64 * Vec<T>::E);
  weigh<T, NT>(st, V, 0, lead + V, p.c, weight);
  __syncthreads();
  const int token = draw<T, NT>(st, V, p.sample_u[b], p.c, weight, segments, shd, shi);
  write_tokens<NT>(p, b, a, token);
}

// ---- smaller batches: all rows at once, in chunks --------------------------------
constexpr int SMALL_NT = 256;

// Chunks' sums of every row that counts.
template <class T, int U>
__global__ __launch_bounds__(SMALL_NT) void lt_verify_sums(VerifyParams p) {
  constexpr int NT = SMALL_NT;
  __shared__ float shf[NT / 64];
  __shared__ double shd[NT / 64];
  const int64_t blk = p.block0 + blockIdx.x, row = blk / p.splits, targets = p.batch * (p.drafts + 1);
  const bool target = row < targets;
  const int64_t b = target ? row / (p.drafts + 1) : (row - targets) / p.drafts;
  const int i = (int)(target ? row - b * (p.drafts + 1) : row - targets - b * p.drafts), n = length_of(p, b);
  if (target ? i > n : i >= n) return;
  const typename T::raw* x = target ? target_row<T>(p, b, i) : draft_row<T>(p, b, i);
  const int lead = lead_of<T>(x), c0 = (int)(blk - row * p.splits) * p.chunk;
  const int v1 = min(lead + p.target.vocab, c0 + p.chunk);
  const Soft o = soft_part<T, NT, U>(x, lead, c0, max(lead, c0), v1, p.c, shf, shd);
  if (threadIdx.x == 0) p.part[blk] = make_double2(o.m, o.s);
}

// A row's chunks, one after another.
__device__ __forceinline__ Soft join_parts(const double2* part, int splits, double c) {
  Soft o;
  for (int i = 0; i < splits; ++i) o.m = fmaxf(o.m, (float)part[i].x);
  for (int i = 0; i < splits; ++i) o.s += part[i].y * exp2_64(fmax((part[i].x - o.m) * c, -DEPTH));
  o.finish(c);
  return o;
}

// Where sequence b stops, from the chunks' sums (every block that needs it does
// the same): a thread a place.
template <class T>
__device__ __forceinline__ Stop<T> find_stop(const VerifyParams& p, int64_t b, int* sh_a, int& a) {
  const int n = length_of(p, b), V = p.target.vocab;
  if (threadIdx.x == 0) *sh_a = n;
  __syncthreads();
  const int64_t targets = p.batch * (p.drafts + 1);
  for (int i0 = 0; i0 < n; i0 += SMALL_NT) {
    const int i = i0 + threadIdx.x;
    if (i < n) {
      const int64_t id = any_id(p.ids, b * p.drafts + i, p.ids_bytes);
      const bool there = id >= 0 && id < V;
      double px = 0, qx = there ? 1 : 0;
      if (there) {
        px = join_parts(p.part + (b * (p.drafts + 1) + i) * p.splits, p.splits, p.c).of(T::get(target_row<T>(p, b, i)[id]), p.c);
        if (p.draft.data)
          qx = join_parts(p.part + (targets + b * p.drafts + i) * p.splits, p.splits, p.c).of(T::get(draft_row<T>(p, b, i)[id]), p.c);
      }
      if (!(there && p.accept_u[b * p.drafts + i] * qx < px)) atomicMin(sh_a, i);
    }
  }
  __syncthreads();
  a = *sh_a;
  Stop<T> st;
  st.x = target_row<T>(p, b, a);
  st.p = join_parts(p.part + (b * (p.drafts + 1) + a) * p.splits, p.splits, p.c);
  if (a < n) {
    st.minus = true;
    st.id = any_id(p.ids, b * p.drafts + a, p.ids_bytes);
    if (p.draft.data) {
      st.y = draft_row<T>(p, b, a);
      st.q = join_parts(p.part + (targets + b * p.drafts + a) * p.splits, p.splits, p.c);
    }
  }
  return st;
}

template <class T>
__global__ __launch_bounds__(SMALL_NT) void lt_verify_weigh(VerifyParams p) {
  __shared__ int sh_a;
  const int64_t blk = p.block0 + blockIdx.x, b = blk / p.weigh_splits;
  int a;
  const Stop<T> st = find_stop<T>(p, b, &sh_a, a);
  const int split = (int)(blk - b * p.weigh_splits), c0 = split * p.weigh_chunk;
  if (split == 0 && threadIdx.x == 0) p.stop[b] = StopNote{st.p.s, st.q.s, st.p.m, st.q.m, a, 0};
  weigh<T, SMALL_NT>(st, p.target.vocab, c0, c0 + p.weigh_chunk, p.c, p.weight + b * p.segments);
}

template <class T>
__global__ __launch_bounds__(SMALL_NT) void lt_verify_draw(VerifyParams p) {
  __shared__ double shd[SMALL_NT / 64];
  __shared__ int shi[2];
  const int64_t b = p.block0 + blockIdx.x;
  const StopNote note = p.stop[b];
  Stop<T> st;
  st.x = target_row<T>(p, b, note.a);
  st.p.m = note.pm;
  st.p.s = note.ps;
  st.p.finish(p.c);
  if (note.a < length_of(p, b)) {
    st.minus = true;
    st.id = any_id(p.ids, b * p.drafts + note.a, p.ids_bytes);
    if (p.draft.data) {
      st.y = draft_row<T>(p, b, note.a);
      st.q.m = note.qm;
      st.q.s = note.qs;
      st.q.finish(p.c);
    }
  }
  const int segments = (lead_of<T>(st.x) + p.target.vocab + 64 * Vec<T>::E - 1) / (64 * Vec<T>::E);
  const int token = draw<T, SMALL_NT>(st, p.target.vocab, p.sample_u[b], p.c, p.weight + b * p.segments, segments, shd, shi);
  write_tokens<SMALL_NT>(p, b, note.a, token);
}

// ---- host ------------------------------------------------------------------
constexpr int64_t MANY = 256;              // sequences that fill the card's CUs

void plan(VerifyParams& p, int dtype) {
  const int e = dtype == LT_F32 ? 4 : 8, step = SMALL_NT * 4 * e;
  const int64_t numbers = (int64_t)p.target.vocab + LEAD, rows = p.batch * (p.drafts + 1 + (p.draft.data ? p.drafts : 0));
  p.segments = (int32_t)((numbers + 64 * e - 1) / (64 * e));
  int64_t n = (numbers + step - 1) / step;
#ifndef XB
#define XB 8192
#endif
  n = n < XB / rows ? n : XB / rows;
  n = n > 1 ? n : 1;
  const int64_t steps = (numbers + n * step - 1) / (n * step);
  p.chunk = (int32_t)(steps * step);
  p.splits = (int32_t)((numbers + p.chunk - 1) / p.chunk);
  const int vectors = SMALL_NT * e;
  n = (numbers + vectors - 1) / vectors;
  n = n < 2048 / p.batch ? n : 2048 / p.batch;
  n = n > 1 ? n : 1;
  p.weigh_chunk = (int32_t)((numbers + n * vectors - 1) / (n * vectors) * vectors);
  p.weigh_splits = (int32_t)((numbers + p.weigh_chunk - 1) / p.weigh_chunk);
}

int64_t weights_bytes(const VerifyParams& p) { return (p.batch * p.segments * (int64_t)sizeof(double) + 15) / 16 * 16; }

int64_t parts_bytes(const VerifyParams& p) { return p.batch * (2 * p.drafts + 1) * p.splits * (int64_t)sizeof(double2); }

int64_t need_bytes(const VerifyParams& p) {
  return weights_bytes(p) + (p.batch >= MANY ? 0 : parts_bytes(p) + p.batch * (int64_t)sizeof(StopNote));
}

template <class T>
lt_status launch_verify(const VerifyParams& p, void* stream) {
  const char* what = "lt_verify_draft";
  if (p.batch >= MANY)
    return p.target.vocab > 8192 ? launch(lt_verify_walk<T, 512, 2>, p.batch, 512, p, stream, what)
                                 : launch(lt_verify_walk<T, 256, 2>, p.batch, 256, p, stream, what);
  const int64_t rows = p.batch * (p.drafts + 1 + (p.draft.data ? p.drafts : 0));
  lt_status st = launch(lt_verify_sums<T, 4>, rows * p.splits, SMALL_NT, p, stream, what);
  if (st == LT_OK) st = launch(lt_verify_weigh<T>, p.batch * p.weigh_splits, SMALL_NT, p, stream, what);
  return st != LT_OK ? st : launch(lt_verify_draw<T>, p.batch, SMALL_NT, p, stream, what);
}

lt_status check(const lt_draft* d) {
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
  return LT_OK;
}

VerifyParams verify_params(const lt_draft* d) {
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
  plan(p, d->target->dtype);
  return p;
}

}  // namespace

extern "C" {

int64_t lt_verify_workspace(const lt_draft* d) {
  if (check(d) != LT_OK || d->batch == 0) return 0;
  return need_bytes(verify_params(d));
}

lt_status lt_verify_draft(const lt_draft* d, double temperature, int64_t* tokens, int64_t* accepted, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  const lt_status st = check(d);
  if (st != LT_OK) return st;
  if (!temperature_ok(temperature)) BAD("temperature %g (1e-6 .. 1e6)", temperature);
  if (d->batch == 0) return LT_OK;
  if (!tokens || !accepted || !d->sample_u || (d->drafts > 0 && (!d->ids || !d->accept_u))) BAD("NULL argument");
  VerifyParams p = verify_params(d);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need_bytes(p))
    BAD("workspace: %lld bytes, 16 B aligned, are needed", (long long)need_bytes(p));
  p.weight = (double*)workspace;
  p.part = (double2*)((char*)workspace + weights_bytes(p));
  p.stop = (StopNote*)((char*)p.part + parts_bytes(p));
  p.c = LOG2E / temperature;
  p.tokens = tokens;
  p.accepted = accepted;
  ON_DEVICE(d->target->device);
  return d->target->dtype == LT_F32   ? launch_verify<F32>(p, stream)
         : d->target->dtype == LT_F16 ? launch_verify<F16>(p, stream)
                                      : launch_verify<BF16>(p, stream);
}

}  // extern "C"
