// lt_verify.hip -- the verification of drafted tokens
// (include/lattice_logits.h lt_verify_draft).
//
// A drafted token is accepted by comparing two probabilities with a random
// number: from sums in 32 bits, unless the two are within these sums' error
// (some 3e-5) of each other; then the rows are summed again in 64 bits.  A token
// is drawn where a running sum over the vocabulary crosses a
// line, so a relative error e of the sums moves it with a probability of about
// e times the number of tokens that the line may fall beside, 131072 e: the
// one or two rows that it is drawn from are summed in 64 bits with an
// exponential good to 1.1e-12.  That costs 35 issue slots a logit (a 64-bit
// operation takes two), where memory allows 14; the sums in 32 bits take 9.
//
// Three launches: sums, weigh, draw.  64 sequences of up to 5 drafts of 131072
// bf16: 22 us (4.6 TB/s), 27 and 8, half of it instructions; one of 4 drafts of
// 32000: 4, 9 and 6, which are latencies.  (The draw by a sequence's last block to weigh, which saves a launch,
// took 25 us longer with a fence of the whole card in every block.)
#include <type_traits>

#include "lt_logits.h"

namespace {

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
// (The float next above it where the nearest one lies below: at the lowest
// temperatures floats are hundreds of exponents apart.)
__device__ __forceinline__ float floor_of(float m, double c) {
  const float f = (float)fmax((double)m - DEPTH / c, (double)LOWEST);
  return ((double)f - m) * c >= -DEPTH ? f : nextafterf(f, INFINITY);
}
__device__ __forceinline__ double soft_exp(float x, float floor, double m, double c) {
  return exp2_64(((double)max2(x, floor) - m) * c);
}

// Where a sequence stops and what its next token is drawn by, for the last kernel.
struct StopNote {
  float pm, qm;           // references of the target's row, of the drafter's
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
  double margin;          // relative error of two probabilities by the sums in 32 bits
  int64_t* tokens;
  int64_t* accepted;
  int32_t rounds;         // a launch for every place of the drafts; else one for all
  int32_t place;          // of this launch
  int32_t splits, chunk;  // blocks of a row, a block's numbers of it
  int32_t segments;       // of a row: 64 vectors each
  int32_t weigh_splits, weigh_chunk;       // of the row that the token is drawn from
  float2* part;           // [batch * (2 drafts + 1)][splits]: reference and sum, targets first
  double2* weight;        // [batch][segments]: sums of e_p and e_q where p > q
  double2* sums;          // [batch][weigh_splits]: sums of e_p and e_q
  int32_t* stopped;       // [batch], rounds: the place of the first token not accepted, or -1
  StopNote* stop;         // [batch]
};

constexpr int NT = 256;

// A thread's part of the sum of exp2((x - m) c) over a row's numbers [v0, v1),
// from c0 on, in 32 bits; m is any logit not far below its largest.  CLEAN: with
// -inf for a NaN (a selection for every logit).
template <class T, int U, bool CLEAN>
__device__ __forceinline__ void sum_thread(const typename T::raw* row, int lead, int c0, int v0, int v1, float c, float& m, float& s) {
  constexpr int E = Vec<T>::E, STEP = NT * U * E;
  m = LOWEST;
  s = 0.f;
  auto of = [](float x) { return CLEAN && x != x ? -INFINITY : x; };
  for (int base = c0; base < v1; base += STEP) {
    Vec<T> v[U];
    load_step<T, NT, U>(v, row - lead, base, threadIdx.x, v0, v1);
    float t = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      t = max2(t, max_of(v[u]));
      v[u].keep();
    }
    if ((t - m) * c > 32.f) {
      s *= exp2_((m - t) * c);
      m = t;
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float f0 = exp2_((of(v[u].get(e)) - m) * c), f1 = exp2_((of(v[u].get(e + 1)) - m) * c);
        s0 += f0;
        s1 += f1;
      }
    s += s0 + s1;
  }
}

// The block's.  A sum that is no number is taken again without the NaN (of an
// infinite logit, which is none that the rows may hold, it stays one).
template <class T, int U>
__device__ __forceinline__ float2 sum_part(const typename T::raw* row, int lead, int c0, int v0, int v1, float c, float* shf) {
  float m, s;
  sum_thread<T, U, false>(row, lead, c0, v0, v1, c, m, s);
  float top = block_reduce<NT, Max>(m, shf), sum = block_reduce<NT, Sum>(s * exp2_((m - top) * c), shf);
  if (sum != sum) {                        // (for the block as a whole)
    numbers_win();
    sum_thread<T, U, true>(row, lead, c0, v0, v1, c, m, s);
    top = block_reduce<NT, Max>(m, shf);
    sum = block_reduce<NT, Sum>(s * exp2_((m - top) * c), shf);
  }
  return make_float2(top, sum);
}

// A row's softmax in 32 bits: exp2((x - m) c) / s.
struct Soft {
  float m;
  double s;
  __device__ __forceinline__ double of(float x, double c) const {
    const double t = ((double)x - m) * c;
    return s > 0 && t > -DEPTH ? exp2_64(t) / s : 0;
  }
};

// A row's chunks, one after another.
__device__ __forceinline__ Soft join_parts(const float2* part, int splits, double c) {
  Soft o{LOWEST, 0};
#pragma unroll 8
  for (int i = 0; i < splits; ++i) o.m = fmaxf(o.m, part[i].x);
#pragma unroll 4
  for (int i = 0; i < splits; ++i) o.s += part[i].y * exp2_64(fmax(((double)part[i].x - o.m) * c, -DEPTH));
  return o;
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
__device__ __forceinline__ Soft target_soft(const VerifyParams& p, int64_t b, int i) {
  return join_parts(p.part + (b * (p.drafts + 1) + i) * p.splits, p.splits, p.c);
}
__device__ __forceinline__ Soft draft_soft(const VerifyParams& p, int64_t b, int i) {
  return join_parts(p.part + (p.batch * (p.drafts + 1) + b * p.drafts + i) * p.splits, p.splits, p.c);
}

// Whether token i of sequence b is accepted: by its rows' sums in 32 bits (ps, qs
// give them); CLOSE where these leave it open.
enum Verdict { REFUSED, ACCEPTED, CLOSE };
template <class T, class P, class Q>
__device__ __forceinline__ Verdict accepts(const VerifyParams& p, int64_t b, int i, int64_t id, float u, P ps, Q qs) {
  if (id < 0 || id >= p.target.vocab) return REFUSED;
  const double px = ps().of(T::get(target_row<T>(p, b, i)[id]), p.c);
  const double qx = p.draft.data ? qs().of(T::get(draft_row<T>(p, b, i)[id]), p.c) : 1.0;
  const double line = u * qx;
  if (fabs(px - line) <= p.margin * px && px > 0) return CLOSE;
  return line < px ? ACCEPTED : REFUSED;
}

// The sum of exp2((x - m) c) of a row in 64 bits, by the block.
template <class T>
__device__ __forceinline__ double sum_row(const typename T::raw* row, int vocab, float m, double c, double* shd) {
  constexpr int E = Vec<T>::E;
  const int lead = lead_of<T>(row);
  const float floor = floor_of(m, c);
  double s = 0;
  for (int at = threadIdx.x * E; at < lead + vocab; at += NT * E) {
    Vec<T> v;
    v.load(row - lead, at, lead, lead + vocab, T::put(-INFINITY));
#pragma nounroll
    for (int e = 0; e < E; e += 4) {
      double t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = E == 4 || e == 0 ? v.get(i) : v.get(E == 4 ? i : i + 4);
        t[i] = x >= floor ? ((double)x - m) * c : -DEPTH;
      }
      exp2_64(t);
      s += (t[0] + t[1]) + (t[2] + t[3]);
    }
  }
  return block_reduce<NT, Sum>(s, shd);
}

// The same by sums in 64 bits, by the block.
template <class T>
__device__ __forceinline__ bool accepts_exactly(const VerifyParams& p, int64_t b, int i, double* shd) {
  const int id = (int)any_id(p.ids, b * p.drafts + i, p.ids_bytes);
  double ratio = p.accept_u[b * p.drafts + i];             // u q / p
#pragma nounroll
  for (int side = 0; side < (p.draft.data ? 2 : 1); ++side) {
    const typename T::raw* x = side ? draft_row<T>(p, b, i) : target_row<T>(p, b, i);
    const float m = (side ? draft_soft(p, b, i) : target_soft(p, b, i)).m;
    const double e = exp2_64(fmax(((double)T::get(x[id]) - m) * p.c, -DEPTH)), s = sum_row<T>(x, p.target.vocab, m, p.c, shd);
    ratio = side ? ratio * (e / s) : ratio / (e / s);
  }
  return ratio < 1;
}

// Chunks' sums: of every row that counts, or in rounds of those of one place,
// where every block first sees whether the token ahead of it was accepted.
template <class T, int U, bool ROUNDS>
__global__ __launch_bounds__(NT) void lt_verify_sums(VerifyParams p) {
  __shared__ float shf[NT / 64];
  const int64_t blk = p.block0 + blockIdx.x, row = blk / p.splits;
  const int split = (int)(blk - row * p.splits);
  const int64_t targets = ROUNDS ? p.batch : p.batch * (p.drafts + 1);
  const bool target = row < targets;
  const int64_t of = target ? row : row - targets, places = ROUNDS ? 1 : target ? p.drafts + 1 : p.drafts;
  const int64_t b = of / places;
  const int i = ROUNDS ? p.place : (int)(of - b * places), n = length_of(p, b);
  if (target ? i > n : i >= n) return;
  if constexpr (ROUNDS) {
    const bool writes = target && split == 0 && threadIdx.x == 0;
    __shared__ double shd[NT / 64];
    if (i == 0) {
      if (writes) p.stopped[b] = -1;
    } else {
      // (a block of this launch may write it, but only what this one finds too)
      const int at = p.stopped[b];
      if (at >= 0 && at < i - 1) return;
      const Verdict v = accepts<T>(p, b, i - 1, any_id(p.ids, b * p.drafts + i - 1, p.ids_bytes), p.accept_u[b * p.drafts + i - 1],
                                   [&] { return target_soft(p, b, i - 1); }, [&] { return draft_soft(p, b, i - 1); });
      if (v == REFUSED || (v == CLOSE && !accepts_exactly<T>(p, b, i - 1, shd))) {
        if (writes) p.stopped[b] = i - 1;
        return;
      }
    }
  }
  const typename T::raw* x = target ? target_row<T>(p, b, i) : draft_row<T>(p, b, i);
  const int lead = lead_of<T>(x), c0 = split * p.chunk, v1 = min(lead + p.target.vocab, c0 + p.chunk);
  const float2 o = sum_part<T, U>(x, lead, c0, max(lead, c0), v1, (float)p.c, shf);
  if (threadIdx.x == 0) p.part[((target ? b * (p.drafts + 1) : p.batch * (p.drafts + 1) + b * p.drafts) + i) * p.splits + split] = o;
}

// The place where sequence b stops, and the sums of its rows there.  (One launch
// for all: a thread a place, which reads ahead of the sequence's length what may
// be behind it.)
struct StopShared {
  int a, close;
  Soft p, q;
};
template <class T>
__device__ __forceinline__ int find_stop(const VerifyParams& p, int64_t b, StopShared& sh, double* shd, Soft& ps, Soft& qs) {
  const int tid = threadIdx.x;
  int a;
  if (p.rounds) {
    a = p.stopped[b];
    if (a < 0) a = length_of(p, b);
  } else {
    Soft tp, tq;
    int64_t id = -1;
    float u = 0;
    if (tid <= p.drafts) tp = target_soft(p, b, tid);
    if (tid < p.drafts) {
      id = any_id(p.ids, b * p.drafts + tid, p.ids_bytes);
      u = p.accept_u[b * p.drafts + tid];
      if (p.draft.data) tq = draft_soft(p, b, tid);
    }
    const int n = length_of(p, b);
    const Verdict v = tid < n ? accepts<T>(p, b, tid, id, u, [&] { return tp; }, [&] { return tq; }) : ACCEPTED;
    for (int from = 0;;) {
      if (tid == 0) sh.a = sh.close = n;
      __syncthreads();
      if (v == REFUSED && tid >= from) atomicMin(&sh.a, tid);
      if (v == CLOSE && tid >= from) atomicMin(&sh.close, tid);
      __syncthreads();
      a = sh.a;
      const int close = sh.close;
      __syncthreads();
      if (close >= a) break;               // (both n: none)
      if (!accepts_exactly<T>(p, b, close, shd)) {
        a = close;
        break;
      }
      from = close + 1;
    }
    if (a < NT) {
      if (tid == a) sh.p = tp, sh.q = tq;
      __syncthreads();
      ps = sh.p;
      qs = sh.q;
      return a;
    }
  }
  ps = target_soft(p, b, a);
  if (p.draft.data && a < p.drafts) qs = draft_soft(p, b, a);
  return a;
}

// What the next token is drawn by: e_p, or max(e_p - ratio e_q, 0), e_p and e_q
// the exponentials of the target's and the drafter's logits and ratio the
// quotient of their sums -- a multiple of max(p - q, 0); without a drafter's
// row, e_p of all but the token that was not accepted.
template <class T>
struct Stop {
  const typename T::raw *x = nullptr, *y = nullptr;
  float pm = LOWEST, qm = LOWEST, pfloor = LOWEST, qfloor = LOWEST;
  int id = -1;
  double ratio = 0;
  __device__ __forceinline__ void floors(double c) {
    pfloor = floor_of(pm, c);
    qfloor = floor_of(qm, c);
  }
  __device__ __forceinline__ double ep(float f, double c) const { return f >= pfloor ? soft_exp(f, pfloor, pm, c) : 0; }
  __device__ __forceinline__ double eq(float f, double c) const { return f >= qfloor ? soft_exp(f, qfloor, qm, c) : 0; }
  __device__ __forceinline__ double weight(int v, double c) const {
    if (v == id) return 0;
    const double w = ep(T::get(x[v]), c);
    return y ? fmax(w - ratio * eq(T::get(y[v]), c), 0.0) : w;
  }
};

template <class T>
__device__ __forceinline__ Stop<T> stop_at(const VerifyParams& p, int64_t b, int a) {
  Stop<T> st;
  st.x = target_row<T>(p, b, a);
  if (a < length_of(p, b)) {
    if (p.draft.data) {
      st.y = draft_row<T>(p, b, a);
    } else {
      const int64_t id = any_id(p.ids, b * p.drafts + a, p.ids_bytes);
      st.id = id >= 0 && id < p.target.vocab ? (int)id : -1;
    }
  }
  return st;
}

// One pass in 64 bits over the rows that the token is drawn from: the sums of
// e_p and e_q of all, and of 64 vectors each where e_p > ratio e_q, ratio as the
// sums in 32 bits give it.  (With the exact ratio, known when all is summed, a
// segment's weight is then e_p - ratio e_q of its two sums: a token that the
// ratio's last bits would put on the other side has no weight to speak of.)
template <class T>
__global__ __launch_bounds__(NT) void lt_verify_weigh(VerifyParams p) {
  constexpr int E = Vec<T>::E;
  __shared__ StopShared sh;
  __shared__ double shd[NT / 64];
  const int64_t blk = p.block0 + blockIdx.x, b = blk / p.weigh_splits;
  const int split = (int)(blk - b * p.weigh_splits), c0 = split * p.weigh_chunk;
  Soft ps{LOWEST, 0}, qs{LOWEST, 0};
  const int a = find_stop<T>(p, b, sh, shd, ps, qs);
  Stop<T> st = stop_at<T>(p, b, a);
  st.pm = ps.m;
  if (st.y) {
    st.qm = qs.m;
    st.ratio = qs.s > 0 ? ps.s / qs.s : 0;
  }
  st.floors(p.c);
  if (split == 0 && threadIdx.x == 0) p.stop[b] = StopNote{st.pm, st.qm, a, 0};
  const int lead = lead_of<T>(st.x), end = lead + p.target.vocab, v1 = min(c0 + p.weigh_chunk, end);
  const typename T::raw* const x = st.x - lead;
  const typename T::raw* const y = st.y ? st.y - lead : nullptr;       // (at any address)
  double sp = 0, sq = 0;
  for (int base = c0; base < v1; base += NT * E) {
    const int at = base + threadIdx.x * E;
    Vec<T> vx, vy;
    vx.load(x, at, lead, end, T::put(-INFINITY));
    if (y) vy.load(y, at, lead, end, T::put(-INFINITY));
    double wp = 0, wq = 0;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      double t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = ((double)max2(vx.get(e + i), st.pfloor) - st.pm) * p.c;
      exp2_64(t);
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = vx.get(e + i) >= st.pfloor ? t[i] : 0;
      sp += (t[0] + t[1]) + (t[2] + t[3]);
      if (y) {
        double q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = ((double)max2(vy.get(e + i), st.qfloor) - st.qm) * p.c;
        exp2_64(q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          q[i] = vy.get(e + i) >= st.qfloor ? q[i] : 0;
          sq += q[i];
          const bool more = t[i] > st.ratio * q[i];
          wp += more ? t[i] : 0;
          wq += more ? q[i] : 0;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) wp += at + e + i - lead == st.id ? 0 : t[i];
      }
    }
    wp = wave_reduce<Sum>(wp, 0.0);
    if (y) wq = wave_reduce<Sum>(wq, 0.0);
    if ((threadIdx.x & 63) == 0 && at < v1) p.weight[b * p.segments + at / (64 * E)] = make_double2(wp, wq);
  }
  sp = block_reduce<NT, Sum>(sp, shd);
  if (y) sq = block_reduce<NT, Sum>(sq, shd);
  if (threadIdx.x == 0) p.sums[blk] = make_double2(sp, sq);
}

struct Two {
  double x, y;
  __device__ __forceinline__ Two operator+(Two o) const { return {x + o.x, y + o.y}; }
};
template <> __device__ __forceinline__ Two neutral<Sum, Two>() { return {0, 0}; }

// The token: the first whose running sum of weights passes u of the whole, else
// the last with a weight; where all weights are 0 (p and q alike), drawn by p.
template <class T>
__global__ __launch_bounds__(NT) void lt_verify_draw(VerifyParams p) {
  constexpr int SEG = 64 * Vec<T>::E;
  __shared__ double shd[NT / 64];
  __shared__ Two sh2[NT / 64];
  __shared__ int first, last;
  constexpr int Q = 4;                     // segments of a thread
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t b = p.block0 + blockIdx.x;
  // what can be read at once: a load that waits for another takes a microsecond
  const double2* const weights = p.weight + b * p.segments;
  const StopNote note = p.stop[b];
  const double u = p.sample_u[b];
  const int64_t drafted = tid < p.drafts ? any_id(p.ids, b * p.drafts + tid, p.ids_bytes) : -1;
  double2 own[Q];
#pragma unroll
  for (int j = 0; j < Q; ++j) own[j] = tid * Q + j < p.segments ? weights[tid * Q + j] : make_double2(0, 0);
  Two sums{0, 0};
  for (int i = tid; i < p.weigh_splits; i += NT) {
    const double2 s = p.sums[b * p.weigh_splits + i];
    sums = sums + Two{s.x, s.y};
  }
  Stop<T> st = stop_at<T>(p, b, note.a);
  st.pm = note.pm;
  st.qm = note.qm;
  st.floors(p.c);
  const int lead = lead_of<T>(st.x), end = lead + p.target.vocab, segments = (end + SEG - 1) / SEG;
  sums = block_reduce<NT, Sum>(sums, sh2);
  const double sp = sums.x;
  if (st.y) st.ratio = sums.y > 0 ? sp / sums.y : 0;
  auto segment_of = [&](double2 w) { return st.y ? fmax(w.x - st.ratio * w.y, 0.0) : w.x; };
  // Of Q neighbours' weights of a thread, the first of which is number i: the first
  // whose running sum (from `before` on) passes the line.  -- found: 0x7fffffff or
  // that; before: the sum of all.  A thread's own in `mine`, its last with a weight
  // in `my_last`, with the sum ahead of each.
  int mine = -1, my_last = -1;
  double ahead = 0, last_ahead = 0;
  auto begin = [&]() {
    if (tid == 0) first = 0x7fffffff, last = -1;
    mine = my_last = -1;
  };
  auto pass = [&](auto& w, int i, auto line_of, double& before) {
    constexpr int N = sizeof(w) / sizeof(double);
    double sum = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) sum += w[j];
    double cum = wave_scan<Sum>(sum, 0.0);
    if (lane == 63) shd[wave] = cum;
    __syncthreads();
    double all = before;
    cum += before - sum;
#pragma unroll
    for (int k = 0; k < NT / 64; ++k) {
      if (k < wave) cum += shd[k];
      all += shd[k];
    }
    const double line = line_of(all);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (w[j] > 0) {
        if (mine < 0 && cum + w[j] > line) mine = i + j, ahead = cum;
        my_last = i + j, last_ahead = cum;
      }
      cum += w[j];
    }
    if (mine >= 0) atomicMin(&first, mine);
    __syncthreads();
    before = all;
    return first;
  };
  // That one, else the last with a weight, else -1; before: the sum ahead of it.
  auto settle = [&](double& before) {
    __syncthreads();
    int at = first;
    if (at == 0x7fffffff) {
      atomicMax(&last, my_last);
      __syncthreads();
      at = last;
      mine = my_last;
      ahead = last_ahead;
    }
    if (at >= 0 && mine == at) shd[0] = ahead;
    __syncthreads();
    before = shd[0];
    __syncthreads();
    return at;
  };
  // The same over [from, to), N neighbours of a thread at a time.
  auto cross = [&](auto n, int from, int to, double line, double& before, auto weight) {
    constexpr int N = decltype(n)::value;
    begin();
    for (int i0 = from; i0 < to; i0 += NT * N) {
      double w[N];
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] = i0 + tid * N + j < to ? weight(i0 + tid * N + j) : 0.0;
      if (pass(w, i0 + tid * N, [&](double) { return line; }, before) != 0x7fffffff) break;
    }
    return settle(before);
  };
  using std::integral_constant;
  constexpr integral_constant<int, Q> MANY;
  constexpr integral_constant<int, SEG / NT> STEP;
  auto of_token = [&](int v) { return st.weight(v, p.c); };
  double line = 0, before = 0;
  int at, token = -1;
  if (segments <= NT * Q) {
    double w[Q];
#pragma unroll
    for (int j = 0; j < Q; ++j) w[j] = tid * Q + j < segments ? segment_of(own[j]) : 0;
    begin();
    pass(w, tid * Q, [&](double all) { return line = u * all; }, before);
    at = settle(before);
  } else {
    double total = 0;
    auto segment = [&](int s) { return segment_of(weights[s]); };
    for (int s = tid; s < segments; s += NT) total += segment(s);
    line = u * block_reduce<NT, Sum>(total, shd);
    at = cross(MANY, 0, segments, line, before, segment);
  }
  if (at >= 0) {
    token = cross(STEP, max(0, at * SEG - lead), min(p.target.vocab, (at + 1) * SEG - lead), line, before, of_token);
    if (token < 0) {
      before = 0;                          // (a segment of rounding errors)
      token = cross(STEP, 0, p.target.vocab, line, before, of_token);
    }
  }
  if (token < 0 && sp > 0) {
    st.y = nullptr;
    st.id = -1;
    before = 0;
    token = cross(STEP, 0, p.target.vocab, u * sp, before, of_token);
  }
  if (tid == 0) p.accepted[b] = note.a;
  for (int i = tid; i <= p.drafts; i += NT)
    p.tokens[b * (p.drafts + 1) + i] = i < note.a ? drafted : i == note.a ? token : -1;
}

// ---- host ------------------------------------------------------------------
// Rounds read no row behind the one where a sequence stops; each costs a
// launch's time and waits for its slowest block.  They pay where a place's rows
// are large and the drafts are many; with lengths, of which about half counts,
// twice as many.  (131072 bf16, us, all at once the second: 512 x 7 drafts 430,
// 488; 350 x 7 336, 355; 512 x 4 350, 354; 260 x 7 284, 282; 512 x 2 274, 263;
// 64 x 5 138, 69; up to 7 each 512 375, 364.)
constexpr int64_t ROUND_BYTES = (int64_t)128 << 20, ROUNDS_BYTES = (int64_t)1 << 30;

int64_t chunks(int64_t numbers, int64_t step, int64_t rows, int64_t blocks) {
  int64_t n = (numbers + step - 1) / step;
  n = n < blocks / rows ? n : blocks / rows;
  return n > 1 ? n : 1;
}

void plan(VerifyParams& p, int dtype) {
  const int e = dtype == LT_F32 ? 4 : 8, step = NT * 4 * e, vectors = NT * e;
  const int64_t numbers = (int64_t)p.target.vocab + LEAD, kinds = p.draft.data ? 2 : 1;
  const int64_t place = p.batch * kinds * p.target.vocab * dtype_bytes(dtype);
  p.rounds = place >= ROUND_BYTES && place * p.drafts >= (p.lengths ? 2 : 1) * ROUNDS_BYTES;
  p.segments = (int32_t)((numbers + 64 * e - 1) / (64 * e));
  // blocks enough that those of rows that do not count leave the card full; in
  // rounds fewer, of which each first finds what was accepted (512 x 7 drafts: 429
  // us of 4096 blocks, 445 of 8192; 400 x 3 of 50261 float32 179 and 195)
  int64_t n = p.rounds ? chunks(numbers, step, p.batch * kinds, 4096) : chunks(numbers, step, p.batch * kinds * (p.drafts + 1), 8192);
  p.chunk = (int32_t)((numbers + n * step - 1) / (n * step) * step);
  p.splits = (int32_t)((numbers + p.chunk - 1) / p.chunk);
  // A bound of a sum's relative error, in roundings of 2^-24: a thread's additions
  // one after another (18 of a step, the steps), 9 to join the block's; its powers
  // of 2 (each within 2) of the term, once where the reference moves and to join,
  // and the two products of these: 8.  An exponent's three roundings (difference,
  // constant, product) are each up to its size times ln 2: the term's and those that
  // carry it to the block's reference add up to at most its depth below the row's
  // largest logit, of a mean of log2(vocab) at most, and 64, as a reference may lag
  // by 32.  (The chunks are joined in 64 bits.)  Twice that for the two that are
  // compared, and a thousandth for the products of errors.
  const double sum = 18 + p.chunk / step + 9 + 8 + 3 * LN2 * (64 + log2((double)p.target.vocab));
  p.margin = 2.002 * sum * 0x1p-24;
  n = chunks(numbers, vectors, p.batch, 1024);
  p.weigh_chunk = (int32_t)((numbers + n * vectors - 1) / (n * vectors) * vectors);
  p.weigh_splits = (int32_t)((numbers + p.weigh_chunk - 1) / p.weigh_chunk);
}

// The workspace's arrays, from `at` on; its bytes.
int64_t lay_out(VerifyParams& p, char* at) {
  int64_t n = 0;
  auto take = [&](int64_t bytes) {
    char* const q = at + n;
    n += (bytes + 15) / 16 * 16;
    return q;
  };
  p.weight = (double2*)take(p.batch * p.segments * (int64_t)sizeof(double2));
  p.sums = (double2*)take(p.batch * p.weigh_splits * (int64_t)sizeof(double2));
  p.part = (float2*)take(p.batch * (2 * p.drafts + 1) * p.splits * (int64_t)sizeof(float2));
  p.stop = (StopNote*)take(p.batch * (int64_t)sizeof(StopNote));
  p.stopped = (int32_t*)take(p.batch * (int64_t)sizeof(int32_t));
  return n;
}

template <class T>
lt_status launch_verify(VerifyParams& p, void* stream) {
  const char* what = "lt_verify_draft";
  lt_status st = LT_OK;
  if (p.rounds) {
    for (p.place = 0; p.place <= p.drafts && st == LT_OK; ++p.place) {
      const int64_t rows = p.batch * (p.draft.data && p.place < p.drafts ? 2 : 1);
      st = launch(lt_verify_sums<T, 4, true>, rows * p.splits, NT, p, stream, what);
    }
  } else {
    const int64_t rows = p.batch * (p.drafts + 1 + (p.draft.data ? p.drafts : 0));
    st = launch(lt_verify_sums<T, 4, false>, rows * p.splits, NT, p, stream, what);
  }
  if (st == LT_OK) st = launch(lt_verify_weigh<T>, p.batch * p.weigh_splits, NT, p, stream, what);
  return st != LT_OK ? st : launch(lt_verify_draw<T>, p.batch, NT, p, stream, what);
}

lt_status check(const lt_draft* d) {
  lt_status st;
  if (!d) BAD("draft: NULL");
  if (!rows_ok(d->target, "target", &st)) return st;
  if (d->batch < 0 || d->drafts < 0 || d->drafts > LT_MAX_DRAFTS)
    BAD("batch %lld, drafts %d (0 .. %d)", (long long)d->batch, d->drafts, LT_MAX_DRAFTS);
  if (d->target->rows != d->batch * (d->drafts + 1))
    BAD("target: %lld rows, batch * (drafts + 1) = %lld", (long long)d->target->rows, (long long)(d->batch * (d->drafts + 1)));
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
  VerifyParams p = verify_params(d);
  return lay_out(p, nullptr);
}

lt_status lt_verify_draft(const lt_draft* d, double temperature, int64_t* tokens, int64_t* accepted, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  const lt_status st = check(d);
  if (st != LT_OK) return st;
  if (!temperature_ok(temperature)) BAD("temperature %g (1e-6 .. 1e6)", temperature);
  if (d->batch == 0) return LT_OK;
  if (!tokens || !accepted || !d->sample_u || (d->drafts > 0 && (!d->ids || !d->accept_u))) BAD("NULL argument");
  VerifyParams p = verify_params(d);
  const int64_t need = lay_out(p, (char*)workspace);
  if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)
    BAD("workspace: %lld bytes, 16 B aligned, are needed", (long long)need);
  p.c = LOG2E / temperature;
  p.tokens = tokens;
  p.accepted = accepted;
  ON_DEVICE(d->target->device);
  return d->target->dtype == LT_F32   ? launch_verify<F32>(p, stream)
         : d->target->dtype == LT_F16 ? launch_verify<F16>(p, stream)
                                      : launch_verify<BF16>(p, stream);
}

}  // extern "C"
