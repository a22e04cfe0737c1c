// lt_top.hip -- the k best logits of a row with its log-sum-exp
// (include/lattice_logits.h lt_top_logits).
#include <dlfcn.h>
#include <stddef.h>

#include "lt_logits.h"

namespace {

constexpr int JOIN = 1024;                 // keys of a row's chunks, at most

struct TopParams {
  Rows x;
  int64_t rows;
  int64_t block0;         // of this launch
  int32_t k;
  int32_t splits;         // blocks of a row
  int32_t chunk;          // of a row's numbers, to a block (a multiple of its step)
  float c;                // log2(e) / temperature
  double inv_t;           // 1 / temperature
  void* values;
  int64_t* ids;
  float* lse;
  uint64_t* part_keys;    // splits > 1: [rows][splits][k], best first, 0 behind a short list
  float2* part_sums;      // [rows][splits]: reference and sum
};

// The log-sum-exp of a row whose exp2((x - m) c) sum up to s.
__device__ __forceinline__ float log_sum(float m, float s, double inv_t) {
  return m == INFINITY ? m : (float)(m * inv_t + log2_(s) * LN2);
}

// The logit of a key, row[id]: read again where the key does not tell it, a NaN
// (in a row whose sum is none: held as -inf) and a -0 (held as 0).
template <class T>
__device__ __forceinline__ typename T::raw logit_of(uint64_t key, float sum, const typename T::raw* row) {
  const uint32_t order = (uint32_t)(key >> 32);
  return sum != sum || order == order_of(0.f) ? row[~(uint32_t)key] : T::put(of_order(order));
}

// The key of lane ^ X: by the data-parallel primitives where they can, else by
// the LDS crossbar.
template <int X>
__device__ __forceinline__ uint64_t from_lane_xor(uint64_t v) {
  constexpr int CTRL = X == 1 ? 0xb1 : X == 2 ? 0x4e : X == 3 ? 0x1b : X == 7 ? 0x141 : X == 8 ? 0x128 : X == 15 ? 0x140 : 0;
  if constexpr (CTRL) {
    return dpp<CTRL, 0xf>(v, v);
  } else if constexpr (X < 32) {
    const uint32_t lo = __builtin_amdgcn_ds_swizzle((int)(uint32_t)v, X << 10 | 0x1f);
    const uint32_t hi = __builtin_amdgcn_ds_swizzle((int)(uint32_t)(v >> 32), X << 10 | 0x1f);
    return (uint64_t)hi << 32 | lo;
  } else {
    return __shfl_xor(v, X, 64);
  }
}
// The larger of the two keys to the lane whose bit BIT is 0.
template <int X, int BIT>
__device__ __forceinline__ void exchange(uint64_t& key) {
  const uint64_t other = from_lane_xor<X>(key);
  key = (key > other) == ((threadIdx.x & BIT) == 0) ? key : other;
}

// A wave's keys, n of them (else 0), largest in lane 0: a bitonic sort, every
// merge's first exchange with the mirrored lane, so that all go the same way.
// (n is the same for all; lanes behind the power of two that holds it are not
// sorted.)
__device__ __forceinline__ uint64_t sort_wave(uint64_t key, int n) {
  exchange<1, 1>(key);
  exchange<3, 2>(key), exchange<1, 1>(key);
  exchange<7, 4>(key), exchange<2, 2>(key), exchange<1, 1>(key);
  if (n <= 8) return key;
  exchange<15, 8>(key), exchange<4, 4>(key), exchange<2, 2>(key), exchange<1, 1>(key);
  if (n <= 16) return key;
  exchange<31, 16>(key), exchange<8, 8>(key), exchange<4, 4>(key), exchange<2, 2>(key), exchange<1, 1>(key);
  if (n <= 32) return key;
  exchange<63, 32>(key), exchange<16, 16>(key), exchange<8, 8>(key), exchange<4, 4>(key), exchange<2, 2>(key), exchange<1, 1>(key);
  return key;
}

// The best min(n, k) of the keys buf[0 .. n), n <= C, in order: sorted 64 at a
// time, then each by its rank, its place in its own 64 and how many of every
// other 64 are larger (a search of seven steps).
template <int NT, int C>
__device__ __forceinline__ void sort_keys(uint64_t* buf, int n, int k) {
  const int tid = thread_of<NT>(), lane = tid & 63;
  uint64_t key[C / NT];
#pragma unroll
  for (int i = 0; i < C / NT; ++i) {
    key[i] = 0;
    if (i * NT + (tid & ~63) < n) {
      key[i] = sort_wave(i * NT + tid < n ? buf[i * NT + tid] : 0, n);
      if (n > 64 || NT == 64) buf[i * NT + tid] = key[i];
    }
  }
  sync<NT>();
  int rank[C / NT];
#pragma unroll
  for (int i = 0; i < C / NT; ++i) {
    rank[i] = lane;
    if (n > 64 && i * NT + (tid & ~63) < n)
#pragma unroll 2
      for (int l = 0; l < n; l += 64) {
        const uint64_t* o = buf + l;
        int at = 0;
#pragma unroll
        for (int step = 32; step; step /= 2) at += o[at + step - 1] > key[i] ? step : 0;
        at += o[at] > key[i];
        rank[i] += l == i * NT + (tid & ~63) ? 0 : at;
      }
  }
  sync<NT>();
#pragma unroll
  for (int i = 0; i < C / NT; ++i)
    if (key[i] && rank[i] < k) buf[rank[i]] = key[i];
  sync<NT>();
}

// Keeps the k largest of the keys buf[0 .. n), k < n <= C, in any order, and
// returns a key that they reach and the others do not: the k-th is found eight
// bits at a time, from the leading bit in which the keys differ, by counting the
// keys of every value of the eight.  hist: 256 counts, 16 B aligned,
// cnt: one more, sh: NT / 64 keys.
template <int NT, int C>
__device__ __forceinline__ uint64_t cut_keys(uint64_t* buf, int n, int k, int* hist, int* cnt, uint64_t* sh) {
  const int tid = thread_of<NT>(), lane = tid & 63;
  uint64_t key[C / NT], hi = 0, lo = ~0ull;
#pragma unroll
  for (int i = 0; i < C / NT; ++i) {
    key[i] = i * NT + tid < n ? buf[i * NT + tid] : 0;
    hi = key[i] > hi ? key[i] : hi;
    if (key[i]) lo = key[i] < lo ? key[i] : lo;
  }
  hi = block_reduce<NT, Max>(hi, sh);
  lo = ~block_reduce<NT, Max>(~lo, sh);
  uint64_t at_least = lo;                 // the k-th key's leading bits, as a key
  int need = k;
  uint64_t width = ~0ull;                 // the keys still in question: less than this above it
  for (int shift = max(0, 56 - __clzll(hi - lo)); ; shift = max(0, shift - 8)) {
    for (int i = tid; i < 256; i += NT) hist[i] = 0;
    if (tid == 0) *cnt = 0;
    sync<NT>();
#pragma unroll
    for (int i = 0; i < C / NT; ++i) {
      const uint64_t over = key[i] - at_least;
      if (key[i] >= at_least && over < width) atomicAdd(&hist[over >> shift], 1);
    }
    sync<NT>();
    const int4 h = ((const int4*)hist)[lane];
    int above = h.x + h.y + h.z + h.w;
    const int upto = wave_scan<Sum>(above, 0);
    above += lane_value(upto, 63) - upto;         // keys from this lane's four values up
    const int l = 63 - __clzll(__ballot(above >= need));
    int d = l * 4, left = lane_value(above, l);      // keys of value d and up
    const int c0 = lane_value(h.x, l), c1 = lane_value(h.y, l), c2 = lane_value(h.z, l), c3 = lane_value(h.w, l);
    int here = c0;
    if (left - here >= need) left -= here, ++d, here = c1;
    if (d == l * 4 + 1 && left - here >= need) left -= here, ++d, here = c2;
    if (d == l * 4 + 2 && left - here >= need) left -= here, ++d, here = c3;
    at_least += (uint64_t)d << shift;
    need -= left - here;
    width = 1ull << shift;
    sync<NT>();
    if (here == need || shift == 0) break;
  }
#pragma unroll
  for (int i = 0; i < C / NT; ++i)
    if (key[i] >= at_least) buf[atomicAdd(cnt, 1)] = key[i];
  sync<NT>();
  return at_least;
}

// One pass over a row (or a chunk of it).  A step takes U vectors of 16 bytes
// a thread.  From the first step's largest logit of every thread comes a
// bound tau that at least k logits reach; a vector with a logit above it goes
// on a list in LDS (its number: a few instructions of a wave, where sorting
// out single logits here took half of the time).  When the list is long, and
// at the end, the vectors' logits above tau become keys, the k largest of
// which are kept and raise tau.
// - Equal logits: those at tau itself are left out; if fewer than k lie above
//   it, the first of them fill up (a scan that ends when enough are found),
//   which also serves rows masked with -inf.
// - What overflows the list or the keys (logits that rise along the row) is
//   taken again, one logit of a thread at a time, cutting the keys to k when
//   they are full.
// (keep() has the logits unpacked anew for each use: held as floats between
// the uses they took 118 registers and half the waves.)
// 4096 x 131072 bf16, k 64: 213 us, 5.1 TB/s, which is the memory's; 509 x 50261
// float16, k 256: 32 us, where reading takes 11: two blocks a CU, whose steps and
// sorts wait for each other.
template <int NT, int C, int CL>
struct TopShared {
  uint64_t buf[C];
  uint64_t sh64[NT / 64];
  alignas(16) int hist[256];               // (read four at a time)
  uint32_t list[CL];
  float shf[NT / 64];
  uint32_t th[NT / 64];
  int reach[NT / 64];
  int cnt, cnt2, listed;
};

template <class T, int NT, int U, int C, int CL>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void lt_top_k(TopParams p) {
  using raw = typename T::raw;
  constexpr int E = Vec<T>::E, W = NT / 64, STEP = NT * U * E, GROUPS = NT == 64 ? 4 : 1;
  numbers_win();
  using Shared = TopShared<NT, C, CL>;
  static_assert(offsetof(Shared, hist) % 16 == 0 && sizeof(Shared) % 16 == 0, "each wave's counts at 16 B");
  __shared__ Shared shared[GROUPS];
  Shared& sh = shared[group_of<NT>()];
  uint64_t* const buf = sh.buf;
  const int tid = thread_of<NT>(), lane = tid & 63, wave = tid >> 6;
  const int64_t blk = (p.block0 + blockIdx.x) * GROUPS + group_of<NT>();
  if (blk >= p.rows * p.splits) return;  // (a wave as a whole)
  const int64_t r = p.splits == 1 ? blk : blk / p.splits;
  const int split = p.splits == 1 ? 0 : (int)(blk % p.splits);
  const raw* const row = (const raw*)p.x.data + p.x.at(r);
  const int lead = lead_of<T>(row);
  const raw* const x = row - lead;
  const int c0 = split * p.chunk;        // the block's: [v0, v1) from c0 on
  const int v0 = max(lead, c0), v1 = min(lead + p.x.vocab, c0 + p.chunk);
  const int k = max(0, min(p.k, v1 - v0));
  const int per_wave = W == 1 ? k + 2 + k / 16 : (k + W - 1) / W + 1;
  float m = LOWEST, s = 0.f, tau = -INFINITY;
  int n = 0;                             // keys
  if (tid == 0) sh.cnt = sh.listed = 0;
  sync<NT>();

  // Above tau; or equal to it, and ahead of the last that a cut kept (in a
  // list, whose vectors lie in any order: of later steps none is ahead).
  uint32_t tie = 0xffffffffu;
  auto counts = [&](float f, int at) {
    return at >= v0 && at < v1 && (f > tau || (f == tau && ~(uint32_t)(at - lead) > tie));
  };
  auto cut = [&]() {
    const uint64_t least = cut_keys<NT, C>(buf, n, k, sh.hist, &sh.cnt2, sh.sh64);
    // (The order next below that of 0 is no logit's: it reads as -0, which compares
    // as 0.  A cut there keeps every 0 so far, and one of a lower index to come.)
    const bool zero = (uint32_t)(least >> 32) == order_of(0.f) - 1;
    tau = zero ? 0.f : of_order((uint32_t)(least >> 32));
    tie = zero ? 0 : max((uint32_t)least, 1u) - 1;
    n = k;
  };

  // The logits of nv vectors -- list[i], or first + i -- that count become keys.
  auto expand = [&](const uint32_t* of, int first, int nv) {
#pragma nounroll
    for (int i0 = 0; i0 < nv; i0 += NT) {
      const int i = i0 + tid;
      const int at = i < nv ? c0 + (of ? (int)of[i] : first + i) * E : v1;
      Vec<T> v;
      v.load(x, at, v0, v1, T::put(-INFINITY));
      int mine = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) mine += counts(v.get(e), at + e);
      if (__any(mine)) {
        const int upto = wave_scan<Sum>(mine, 0);
        int pos = 0;
        if (lane == 63) pos = atomicAdd(&sh.cnt, upto);
        pos = __builtin_amdgcn_readlane(pos, 63) + upto - mine;
        v.keep();
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float f = v.get(e);
          if (counts(f, at + e)) {
            if (pos < C) buf[pos] = order_key(f, (uint32_t)(at + e - lead));
            ++pos;
          }
        }
      }
      sync<NT>();
      const int was = n;
      n = sh.cnt;
      sync<NT>();
      if (n > C) {
        n = was;
#pragma nounroll
        for (int e = 0; e < E; ++e) {
          if (n > C - NT) cut();           // (room for a logit of every thread)
          if (tid == 0) sh.cnt = n;
          sync<NT>();
          const float f = at + e >= v0 && at + e < v1 ? T::get(x[at + e]) : -INFINITY;
          if (counts(f, at + e)) buf[atomicAdd(&sh.cnt, 1)] = order_key(f, (uint32_t)(at + e - lead));
          sync<NT>();
          n = sh.cnt;
          sync<NT>();
        }
      }
    }
  };

  int have = 0;                          // vectors on the list
  for (int base = c0; base < v1; base += STEP) {
    Vec<T> v[U];
    float vm[U];
    load_step<T, NT, U>(v, x, base, tid, v0, v1);
    float t = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      vm[u] = max_of(v[u]);
      t = max2(t, vm[u]);
      v[u].keep();
    }
    if ((t - m) * p.c > 32.f) {
      s *= exp2_((m - t) * p.c);
      m = t;
    }
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        s0 += exp2_((v[u].get(e) - m) * p.c);
        s1 += exp2_((v[u].get(e + 1) - m) * p.c);
      }
    s += s0 + s1;
    if (base == c0) {
      // the per_wave-th largest of a wave's threads (from its leading 18 bits
      // down), and of the waves' the largest that k threads of the block are
      // above (the least where ties leave none: k threads reach that)
      const uint32_t o = order_of(t);
      uint32_t th = 0;
      for (int bit = 31; bit >= 14; --bit) {
        const uint32_t cand = th | 1u << bit;
        if (__popcll(__ballot(o >= cand)) >= per_wave) th = cand;
      }
      if (W > 1) {
        if (lane == 0) {
          sh.th[wave] = th;
          sh.reach[wave] = 0;
        }
        sync<NT>();
        const uint32_t theirs = lane < W ? sh.th[lane] : 0;
        int reach = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int c = __popcll(__ballot(o > (uint32_t)__builtin_amdgcn_readlane(theirs, w)));
          reach = lane == w ? c : reach;
        }
        if (lane < W) atomicAdd(&sh.reach[lane], reach);
        sync<NT>();
        th = wave_reduce<Max>(lane < W && sh.reach[lane] >= k ? theirs : 0u, 0u);
        if (!th) th = ~wave_reduce<Max>(lane < W ? ~theirs : 0u, 0u);
      }
      tau = th <= order_of(-INFINITY) ? -INFINITY : of_order(th);
    }
    if (__any(t > tau)) {
      uint64_t b[U];
      int all = 0, pos = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        b[u] = __ballot(vm[u] > tau);
        all += __popcll(b[u]);
      }
      if (lane == 0) pos = atomicAdd(&sh.listed, all);
      pos = __builtin_amdgcn_readfirstlane(pos);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = pos + __builtin_amdgcn_mbcnt_hi((uint32_t)(b[u] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b[u], 0));
        if (vm[u] > tau && at < CL) sh.list[at] = (uint32_t)((base - c0) / E + u * NT + tid);
        pos += __popcll(b[u]);
      }
    }
    sync<NT>();
    const int was = have;
    have = sh.listed;
    sync<NT>();                          // (a push of the next step may run ahead of the slowest read of `listed`)
    const bool last = base + STEP >= v1, over = have > CL;
    if (last || over || n + have > k + k / 2 + 192) {
#pragma nounroll
      for (int pass = 0; pass <= (int)over; ++pass)
        expand(pass ? nullptr : sh.list, (base - c0) / E, pass ? min(NT * U, (v1 - base + E - 1) / E) : over ? was : have);
      // the best k so far: fewer of the logits to come lie above the last of them
      if (n > k && (!last || n > 512)) cut();
      tie = 0xffffffffu;
      have = 0;
      if (tid == 0) {
        sh.cnt = n;
        sh.listed = 0;
      }
      sync<NT>();
    }
  }
  const float top = block_reduce<NT, Max>(m, sh.shf);
  const float sum = block_reduce<NT, Sum>(s * exp2_((m - top) * p.c), sh.shf);
  // (a NaN as -inf, which nothing else is less than)
  auto equals = [&](float f, int at) { return at >= v0 && at < v1 && (tau == -INFINITY ? !(f > tau) : f == tau); };
  for (int base = c0; n < k && base < v1; base += NT * E) {
    // the first logits that equal tau: in order, a vector a thread (never
    // short of k: at least k logits reach tau)
    const int at = base + tid * E;
    Vec<T> v;
    v.load(x, at, v0, v1, T::put(-INFINITY));
    int mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine += equals(v.get(e), at + e);
    const int upto = wave_scan<Sum>(mine, 0);
    if (lane == 63) sh.reach[wave] = upto;
    sync<NT>();
    int pos = n + upto - mine, all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int c = sh.reach[w];
      if (w < wave) pos += c;
      all += c;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (equals(v.get(e), at + e)) {
        if (pos < k) buf[pos] = order_key(tau, (uint32_t)(at + e - lead));
        ++pos;
      }
    n = min(k, n + all);
    sync<NT>();
  }
  sort_keys<NT, C>(buf, n, k);
  if (p.splits == 1) {
    if (tid == 0) p.lse[r] = log_sum(top, sum, p.inv_t);
    for (int j = tid; j < k; j += NT) {
      p.ids[r * k + j] = ~(uint32_t)buf[j];
      ((raw*)p.values)[r * k + j] = logit_of<T>(buf[j], sum, row);
    }
  } else {
    if (tid == 0) p.part_sums[blk] = make_float2(top, sum);
    for (int j = tid; j < p.k; j += NT) p.part_keys[blk * p.k + j] = j < k ? buf[j] : 0;
  }
}

// The k best of a row's chunks' lists, and its sum.
template <class T>
__global__ __launch_bounds__(256) void lt_top_join(TopParams p) {
  constexpr int NT = 256, C = JOIN;
  __shared__ TopShared<NT, C, 1> sh;
  const int tid = threadIdx.x;
  const int64_t r = p.block0 + blockIdx.x;
  const int n = p.splits * p.k;
  for (int i = tid; i < n; i += NT) sh.buf[i] = p.part_keys[r * n + i];
  float m = LOWEST, s = 0.f;
  for (int i = 0; i < p.splits; ++i) m = max2(m, p.part_sums[r * p.splits + i].x);
  for (int i = 0; i < p.splits; ++i) {
    const float2 part = p.part_sums[r * p.splits + i];
    s += part.y * exp2_((part.x - m) * p.c);
  }
  __syncthreads();
  int left = n;
  if (n > 256) {
    cut_keys<NT, C>(sh.buf, n, p.k, sh.hist, &sh.cnt2, sh.sh64);
    left = p.k;
  }
  sort_keys<NT, C>(sh.buf, left, p.k);
  if (tid == 0) p.lse[r] = log_sum(m, s, p.inv_t);
  const typename T::raw* x = (const typename T::raw*)p.x.data + p.x.at(r);
  for (int j = tid; j < p.k; j += NT) {
    p.ids[r * p.k + j] = ~(uint32_t)sh.buf[j];
    ((typename T::raw*)p.values)[r * p.k + j] = logit_of<T>(sh.buf[j], s, x);
  }
}

// Rows of at most FEW logits and k <= K: a thread keeps its row's k best in
// registers, inserting each logit (64 rows of 41 logits, k 5: about 40
// instructions of a wave a row, where a wave a row takes 240; 131072 x 41
// float32: 16 us, 1.9 TB/s: two waves a SIMD, 9 us of instructions, the insertions
// foremost, and the rest waiting).
template <class T, int K>
__global__ __launch_bounds__(64) void lt_top_few(TopParams p) {
  using raw = typename T::raw;
  extern __shared__ float few[];           // [64][few_pitch(vocab)], then [64][k] results
  numbers_win();
  const int lane = threadIdx.x, vocab = p.x.vocab, pitch = few_pitch(vocab);
  const int64_t r0 = (p.block0 + blockIdx.x) * 64;
  const int rows = (int)min((int64_t)64, p.rows - r0);
  load_few<T>(p.x, r0, rows, few, pitch);
  __syncthreads();
  const float* x = few + min(lane, rows - 1) * pitch;
  uint32_t best[K];
  int id[K];
#pragma unroll
  for (int j = 0; j < K; ++j) best[j] = 0, id[j] = 0;
  float m = LOWEST;
  for (int v0 = 0; v0 < vocab; v0 += 4) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = x[v0 + i];
    m = max2(max3(m, f[0], f[1]), max2(f[2], f[3]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t o = v0 + i < vocab ? order_of(f[i]) : 0;
      // (behind an equal one, which came earlier)
#pragma unroll
      for (int j = K - 1; j >= 0; --j) {
        const bool here = o > best[j], ahead = j > 0 && o > best[j > 0 ? j - 1 : 0];
        best[j] = ahead ? best[j > 0 ? j - 1 : 0] : here ? o : best[j];
        id[j] = ahead ? id[j > 0 ? j - 1 : 0] : here ? v0 + i : id[j];
      }
    }
  }
  float s = 0.f;
  for (int v0 = 0; v0 < vocab; v0 += 4) {
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = exp2_((x[v0 + i] - m) * p.c);
    s += (e[0] + e[1]) + (e[2] + e[3]);
  }
  if (lane < rows) p.lse[r0 + lane] = log_sum(m, s, p.inv_t);
  // results by way of LDS, so that the rows' are written together
  raw* val = (raw*)(few + 64 * pitch);
  uint8_t* at = (uint8_t*)(val + 64 * p.k);
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (j < p.k) {
      val[lane * p.k + j] = T::put(x[id[j]]);
      at[lane * p.k + j] = (uint8_t)id[j];
    }
  __syncthreads();
  for (int i = lane; i < rows * p.k; i += 64) {
    ((raw*)p.values)[r0 * p.k + i] = val[i];
    p.ids[r0 * p.k + i] = at[i];
  }
}

// What is made of this inside a loop is made there each time: the numbers of all
// of a lane's logits, made ahead of the loop, took 40 registers.
__device__ __forceinline__ int renewed(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Rows that a wave holds in its registers, U vectors a lane.  The k-th largest
// is found from below by its bits, from the leading one down: of the lanes'
// largest logits, of the vectors' or of all logits, the fewest that are at least
// twice as many as k -- k logits reach what is found, and not many more.  Those
// become keys in LDS, which are sorted.  Its instructions bound it, but for long
// rows and a small k: 65536 x 2000 bf16, k 5: 60 us (4.4 TB/s), k 100: 138;
// 65536 x 200, k 5: 32 (a wave that sorts all of the row 108).
// Rows where more than C logits reach it (equal ones, mostly) or where it is
// -inf, and rows with a NaN: the bound is raised to the largest logit if k equal
// it, else by a search among all logits, which ends when few enough reach it or at
// the k-th itself; then only those above it become keys, and the first of those
// that equal it (65536 x 2000 bf16, k 5: 60 us, constant rows 172).
template <class T, class V, int U>
__global__ __launch_bounds__(256) void lt_top_wave(TopParams p) {
  using raw = typename T::raw;
  constexpr int E = V::E, C = 2 * MAXK;
  numbers_win();
  __shared__ __attribute__((aligned(16))) uint64_t keys[4][C];
  uint64_t* const buf = keys[group_of<64>()];
  const int lane = threadIdx.x & 63, vocab = p.x.vocab, k = p.k;
  const int64_t r = (p.block0 + blockIdx.x) * 4 + group_of<64>();
  if (r >= p.rows) return;                 // (a wave as a whole)
  const raw* const x = (const raw*)p.x.data + p.x.at(r);
  V v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = (u * 64 + lane) * E;
    if ((u + 1) * 64 * E <= vocab) v[u].load(x + at);
    else v[u].load(x, at, 0, vocab, T::put(-INFINITY));
  }
  float vm[U], m = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    vm[u] = max_of(v[u]);
    m = max2(m, vm[u]);
    v[u].keep();
  }
  m = max2(m, -INFINITY);                  // (of NaNs alone)
  const float top = max2(wave_reduce<Max>(m, -INFINITY), LOWEST);
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int e = 0; e < E; ++e) s[(u * E + e) & 1] += exp2_((v[u].get(e) - top) * p.c);
    v[u].keep();
  }
  const float sum = wave_reduce<Sum>(s[0] + s[1], 0.f);
  if (lane == 0) p.lse[r] = log_sum(top, sum, p.inv_t);
  int n = 0;
  uint64_t key = 0;
  uint32_t th = 0;
  // (18 bits: all of a 16-bit logit's)
  if (k * 2 <= min(64, (vocab + E - 1) / E)) {
    const uint32_t o = order_of(m);
#pragma unroll 2
    for (int bit = 31; bit >= 14; --bit) {
      const uint32_t cand = th | 1u << bit;
      if (__popcll(__ballot(o >= cand)) >= k) th = cand;
    }
  } else if (U > 1 && E > 1 && k * (2 * E) <= vocab) {
    uint32_t o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) o[u] = order_of(vm[u]);
#pragma nounroll
    for (int bit = 31; bit >= 14; --bit) {
      const uint32_t cand = th | 1u << bit;
      int c = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) c += __popcll(__ballot(o[u] >= cand));
      if (c >= k) th = cand;
    }
  } else {
#pragma nounroll
    for (int bit = 31; bit >= 14; --bit) {
      const float f = of_order(th | 1u << bit);
      int c = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        V w = v[u];
        // (64 logits of a lane take too many registers as floats: 16384 x 4000, k
        // 200 99 us, unpacked each time 86; 32 do not: 65536 x 2000, k 256 304, 331)
        if (U * E > 32) w.keep();
#pragma unroll
        for (int e = 0; e < E; ++e) c += __popcll(__ballot(w.get(e) >= f));
      }
      if (c < k) continue;
      th |= 1u << bit;
      if (c <= ((k + 63) & ~63)) break;
    }
  }
  float tau = of_order(th);
  if (th > order_of(-INFINITY)) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = v[u].get(e);
        const uint64_t b = __ballot(f >= tau);
        if (b) {
          const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
          if (f >= tau && at < C) buf[at] = order_key(f, (uint32_t)((u * 64 + lane) * E + e));
          n += __popcll(b);
        }
      }
  } else {
    n = C + 1;
  }
  if (n > C) {
    // Logits that reach f, which is above -inf (so does no NaN).
    auto reach = [&](float f) {
      int c = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        V w = v[u];
        w.keep();
#pragma unroll
        for (int e = 0; e < E; ++e) c += __popcll(__ballot(w.get(e) >= f));
      }
      return c;
    };
    th = order_of(LOWEST);
    int c = reach(LOWEST);
    if (c > C) {
      th = order_of(top);
      c = reach(top);
      if (c < k) {
        th = 0;
#pragma nounroll
        for (int bit = 31; bit >= 0; --bit) {
          const int d = reach(of_order(th | 1u << bit));
          if (d < k) continue;
          th |= 1u << bit;
          c = d;
          if (c <= C) break;
        }
      }
      th += c > C;
    }
    tau = of_order(th);
    // those that reach th, then, if these are less than k, the first of those next
    // below it (-inf, or a NaN in its place, below the lowest)
    const float next = of_order(th - 1);
    n = 0;
#pragma nounroll
    for (int below = 0; below < 2; ++below)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!below || n < k) {
          V w = v[u];
          w.keep();
          const int first = renewed((u * 64 + lane) * E);
          auto counts = [&](int e) {
            const float f = w.get(e);
            return below ? first + e < vocab && (next == -INFINITY ? !(f > next) : f == next) : f >= tau;
          };
          int mine = 0;
#pragma unroll
          for (int e = 0; e < E; ++e) mine += counts(e);
          const int upto = wave_scan<Sum>(mine, 0);
          int at = n + upto - mine;
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (counts(e)) {
              if (at < (below ? k : C)) buf[at] = order_key(below ? next : w.get(e), (uint32_t)(first + e));
              ++at;
            }
          n += lane_value(upto, 63);
          if (below) n = min(k, n);
        }
  }
  sync<64>();
  if (n > 64) sort_keys<64, C>(buf, n, k);
  else key = sort_wave(lane < n ? buf[lane] : 0, n);
  for (int j = lane; j < k; j += 64) {
    if (n > 64) key = buf[j];
    p.ids[r * k + j] = ~(uint32_t)key;
    ((raw*)p.values)[r * k + j] = logit_of<T>(key, sum, x);
  }
}

// Chunks of a row: one where the rows fill the card or a row is a few steps of
// a block; else a step or more each.  (64 x 131072 bf16, k 20: 27 us whole; in
// 8 chunks 10 us, and 4 us to join them in a launch of its own.)
void split_rows(TopParams& p, int dtype) {
  const int step = 512 * 4 * (dtype == LT_F32 ? 4 : 8);
  const int64_t numbers = (int64_t)p.x.vocab + LEAD;
  int64_t n = 1;
  if (p.x.vocab > 6 * step && p.rows < 256) {
    n = (numbers + step - 1) / step;
    n = n < 512 / p.rows ? n : 512 / p.rows;
    n = n < JOIN / p.k ? n : JOIN / p.k;
  }
  const int64_t steps = (numbers + n * step - 1) / (n * step);
  p.chunk = (int32_t)(n == 1 ? 0x7fffff80 : steps * step);
  p.splits = (int32_t)((numbers + p.chunk - 1) / p.chunk);     // at most n: JOIN keys hold
}

int64_t top_workspace(const TopParams& p) {
  return p.splits == 1 ? 0 : p.rows * p.splits * (int64_t)(p.k * sizeof(uint64_t) + sizeof(float2));
}

// (65536 rows of 100 logits, k 5: 28 us by single logits, 68 by vectors; of 300:
// 35 by a vector a lane, 39 by two.  16384 rows of 4000, k 100: 60 us, lt_top_k
// of 256 threads 105.)
template <class T>
auto wave_kernel(int vocab) -> void (*)(TopParams) {
  using V = Vec<T>;
  if (vocab <= 128) return lt_top_wave<T, One<T>, 2>;
  if (vocab <= 256) return lt_top_wave<T, One<T>, 4>;
  if (vocab <= 64 * V::E) return lt_top_wave<T, V, 1>;
  if (vocab <= 128 * V::E) return lt_top_wave<T, V, 2>;
  return vocab <= 256 * V::E ? lt_top_wave<T, V, 4> : lt_top_wave<T, V, 8>;
}

template <class T>
lt_status launch_top(TopParams& p, void* stream) {
  // Few logits a row, few of them wanted, and rows enough: a thread a row.
  // (131072 x 41 float32, k 5: 15 us, a wave a row 49; 16384 x 64, k 8: 16 and 12.
  // Registers for 1 logit 13 us, for 5 15, for 8 19.)
  if (p.x.vocab <= FEW && p.k <= 8 && p.rows >= 16384) {
    const int64_t blocks = (p.rows + 63) / 64;
    const int lds = 64 * (few_pitch(p.x.vocab) * 4 + p.k * (int)(sizeof(typename T::raw) + 1));
    if (p.k == 1) return launch(lt_top_few<T, 1>, blocks, 64, p, stream, "lt_top_logits", lds);
    if (p.k <= 5) return launch(lt_top_few<T, 5>, blocks, 64, p, stream, "lt_top_logits", lds);
    return launch(lt_top_few<T, 8>, blocks, 64, p, stream, "lt_top_logits", lds);
  }
  const int64_t fours = (p.rows + 3) / 4;
  // Rows that fit a wave's registers; few of them with many wanted are sorted
  // sooner by a block.  (bf16, us, 256 threads the second: 256 x 2000, k 60 13, 13;
  // k 200 18, 13; 2000 x 2000, k 200 20, 26; 256 x 1000, k 200 14, 14.  float32: 256 x
  // 2000, k 200 17, 13; 400 x 1100, k 150 16, 13; 500 x 2000, k 110 13, 13.)
  const bool few_rows = p.rows < 512 && p.k > 100 && p.k <= 252 && p.x.vocab > 1024;
  if (p.x.vocab <= 512 * Vec<T>::E && !few_rows)
    return launch(wave_kernel<T>(p.x.vocab), fours, 256, p, stream, "lt_top_logits");
  if (p.splits > 1) {
    const lt_status st = launch(lt_top_k<T, 512, 4, 1024, 1024>, p.rows * p.splits, 512, p, stream, "lt_top_logits");
    return st != LT_OK ? st : launch(lt_top_join<T>, p.rows, 256, p, stream, "lt_top_logits");
  }
  // Longer rows: a wave a row, 256 threads or 512.  Fewer threads wait for each
  // other less, more find enough to do in few rows and hold a k of their size.
  // (bf16, us: 16384 x 6000, k 5: 48, 96, -; k 32: 96, 97, -; 2048 x 6000, k 32:
  // 27, 18, -; 4096 x 16000, k 60: 76, 42, 61; k 200: -, 97, 68; 16384 x 8000, k
  // 200: -, 187, 241; 256 x 50000, k 60: 83, 24, 17.  float32: 16384 x 6000, k 5: 79,
  // 118, 183; k 32: 105, 123, 193; 2048 x 6000, k 32: 25, 20, 26; 4096 x 16000, k 60:
  // -, 66, 65; k 200: -, 95, 85; 16384 x 8000, k 200: -, 246, 223; 256 x 50000, k 60:
  // -, 27, 21.)  Beyond k 252 the first bound of 256 threads would need more of a
  // wave's threads than it has.
  if (p.k <= 32 && p.x.vocab <= 8192 && p.rows >= 2048)
    return launch(lt_top_k<T, 64, 4, 256, 128>, fours, 256, p, stream, "lt_top_logits");
  if (p.k > 252 || (p.k > 192 && p.x.vocab > 8192) || (p.rows < 512 && p.x.vocab > 8192))
    return launch(lt_top_k<T, 512, 4, 1024, 1024>, p.rows, 512, p, stream, "lt_top_logits");
  return launch(lt_top_k<T, 256, 4, 1024, 512>, p.rows, 256, p, stream, "lt_top_logits");
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

int64_t lt_top_logits_workspace(const lt_rows* x, int32_t k) {
  if (!x || x->rows < 1 || x->vocab < 1 || x->vocab > LT_MAX_VOCAB || k < 1 || k > MAXK) return 0;
  TopParams p{};
  p.x = rows_of(x);
  p.rows = x->rows;
  p.k = k;
  split_rows(p, x->dtype);
  return top_workspace(p);
}

lt_status lt_top_logits(const lt_rows* x, int32_t k, double temperature, void* values, int64_t* ids, float* lse,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  lt_status st;
  if (!rows_ok(x, "logits", &st)) return st;
  if (k < 1 || k > MAXK || k > x->vocab) BAD("k %d (1 .. min(vocab, %d))", k, MAXK);
  if (!temperature_ok(temperature)) BAD("temperature %g (1e-6 .. 1e6)", temperature);
  if (x->rows == 0) return LT_OK;
  if (!values || !ids || !lse) BAD("output: NULL");
  TopParams p{};
  p.x = rows_of(x);
  p.rows = x->rows;
  p.k = k;
  p.c = (float)(LOG2E / temperature);
  p.inv_t = 1 / temperature;
  p.values = values;
  p.ids = ids;
  p.lse = lse;
  split_rows(p, x->dtype);
  const int64_t need = top_workspace(p);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    BAD("workspace: %lld bytes, 16 B aligned, are needed", (long long)need);
  p.part_keys = (uint64_t*)workspace;
  p.part_sums = (float2*)((char*)workspace + p.rows * p.splits * (int64_t)p.k * sizeof(uint64_t));
  ON_DEVICE(x->device);
  return x->dtype == LT_F32 ? launch_top<F32>(p, stream) : x->dtype == LT_F16 ? launch_top<F16>(p, stream) : launch_top<BF16>(p, stream);
}

}  // extern "C"
