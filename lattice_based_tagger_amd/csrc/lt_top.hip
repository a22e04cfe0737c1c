// lt_top.hip -- the k best logits of a row with its log-sum-exp
// (include/lattice_logits.h lt_top_logits).
#include <dlfcn.h>

#include "lt_logits.h"

namespace {

struct TopParams {
  Rows x;
  int64_t rows;
  int32_t k;
  int32_t splits;         // blocks of a row
  int32_t chunk;          // logits of a block (a multiple of 8), the last one's fewer
  float c;                // log2(e) / temperature
  void* values;
  int64_t* ids;
  float* lse;
  uint64_t* part_keys;    // splits > 1: [rows][splits][k], best first, 0 behind a short list
  float2* part_sums;      // [rows][splits]: reference and sum
};

// The sum behind a log-sum-exp: that of exp2((x - m) c), m any logit at most 32
// (in the exponent) below the largest seen.
__device__ __forceinline__ float log_sum(float m, float s, float c) {
  return m == INFINITY ? m : (float)((double)m * (c * 0.6931471805599453) + log((double)s));
}

// The keys of buf[0 .. n), n <= C, each by its rank (the number of larger
// ones): afterwards buf[0 .. min(n, k)) holds the best in order.
template <int NT, int C>
__device__ __forceinline__ void rank_keys(uint64_t* buf, int n, int k) {
  uint64_t key[C / NT];
  int rank[C / NT];
#pragma unroll
  for (int i = 0; i < C / NT; ++i) {
    const int at = i * NT + threadIdx.x;
    rank[i] = at < n ? 0 : k;
    key[i] = at < n ? buf[at] : ~0ull;
    if (i * NT + (int)(threadIdx.x & ~63u) < n)
      for (int j = 0; j < n; ++j) rank[i] += buf[j] > key[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < C / NT; ++i)
    if (rank[i] < k) buf[rank[i]] = key[i];
  __syncthreads();
}

// The k best of x[v0 .. v1) one after another, k passes: rows with a NaN.
template <class T, int NT>
__device__ void best_by_passes(const typename T::raw* x, int v0, int v1, int k, uint64_t* out, uint64_t* sh) {
  uint64_t below = ~0ull;
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    for (int v = v0 + threadIdx.x; v < v1; v += NT) {
      const uint64_t key = order_key(T::get(x[v]), (uint32_t)v);
      if (key < below && key > best) best = key;
    }
    below = block_reduce<NT, Max>(best, sh);
    if (threadIdx.x == 0) out[j] = below;
  }
  __syncthreads();
}

// One pass over a row (or a chunk of it).  A step takes U vectors of 16 bytes
// a thread.  From the first step's largest logit of every thread comes a
// bound tau that at least k logits reach; what is above it goes into an LDS
// buffer, a few more than k of a row's logits, which are then ranked.
// - Equal logits: those at tau itself are left out; if fewer than k lie above
//   it, the first of them fill up (a scan that ends when enough are found),
//   which also serves rows masked with -inf.
// - A step that overflows the buffer (logits that rise along the row) is
//   taken again from the registers, one logit of a thread at a time, ranking
//   when the buffer is full, which raises tau to the k-th best so far.
template <class T, int NT, int U, int C>
__global__ __launch_bounds__(NT) void lt_top_k(TopParams p) {
  using raw = typename T::raw;
  constexpr int E = Vec<T>::E, W = NT / 64, STEP = NT * U * E;
  __shared__ __attribute__((aligned(16))) uint64_t buf[C];
  __shared__ uint64_t sh64[W];
  __shared__ float shf[W];
  __shared__ int cnt;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per_wave = (p.k + W - 1) / W + 1;
  for (int64_t blk = blockIdx.x; blk < p.rows * p.splits; blk += gridDim.x) {
    const int64_t r = p.splits == 1 ? blk : blk / p.splits;
    const int split = p.splits == 1 ? 0 : (int)(blk % p.splits);
    const raw* x = (const raw*)p.x.data + p.x.at(r);
    const int v0 = split * p.chunk, v1 = min(p.x.vocab, v0 + p.chunk);
    const int k = min(p.k, v1 - v0);
    float m = LOWEST, s = 0.f, tau = -INFINITY;
    if (tid == 0) cnt = 0;
    __syncthreads();
    int before = 0;                        // the buffer's entries ahead of this step
    for (int base = v0; base < v1; base += STEP) {
      Vec<T> v[U];
      float vm[U];
      if (base + STEP <= v1) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u].load(x + base + (u * NT + tid) * E);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = base + (u * NT + tid) * E;
          if (at + E <= v1) v[u].load(x + at);
          else v[u].load_part(x + at, max(0, v1 - at), T::put(-INFINITY));
        }
      }
      float t = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        vm[u] = max_of(v[u]);
        t = max2(t, vm[u]);
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
      if (base == v0) {
        // the per_wave-th largest of a wave's threads (from its leading 18
        // bits down): over all waves at least k logits reach the least of them
        const uint32_t o = order_of(t);
        uint32_t th = 0;
        for (int bit = 31; bit >= 14; --bit) {
          const uint32_t cand = th | 1u << bit;
          if (__popcll(__ballot(o >= cand)) >= per_wave) th = cand;
        }
        tau = th <= order_of(-INFINITY) ? -INFINITY : of_order(th);
        if (W > 1) {
          if (lane == 0) shf[wave] = tau;
          __syncthreads();
          for (int w = 0; w < W; ++w) tau = fminf(tau, shf[w]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (vm[u] > tau) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float f = v[u].get(e);
            if (f > tau) {
              const int at = atomicAdd(&cnt, 1);
              if (at < C) buf[at] = order_key(f, (uint32_t)(base + (u * NT + tid) * E + e));
            }
          }
        }
      __syncthreads();
      int n = cnt;
      if (n > C) {
        uint64_t above = (uint64_t)order_of(tau) << 32 | 0xffffffffu;
        __syncthreads();
        if (tid == 0) cnt = before;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u)
          for (int e = 0; e < E; ++e) {
            float f = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) f = i == e ? v[u].get(i) : f;
            const int at = base + (u * NT + tid) * E + e;
            const uint64_t key = order_key(f, (uint32_t)at);
            if (at < v1 && key > above) buf[atomicAdd(&cnt, 1)] = key;
            __syncthreads();
            n = cnt;
            __syncthreads();
            if (n > C - NT) {
              rank_keys<NT, C>(buf, n, k);
              above = buf[k - 1];
              tau = of_order((uint32_t)(above >> 32));
              n = k;
              if (tid == 0) cnt = k;
              __syncthreads();
            }
          }
      }
      before = n;
      // (a later step's first push may run ahead of this step's slowest read)
      if (base + STEP < v1) __syncthreads();
    }
    const float top = block_reduce<NT, Max>(m, shf);
    const float sum = block_reduce<NT, Sum>(s * exp2_((m - top) * p.c), shf);
    int n = before;
    if (sum != sum) {
      best_by_passes<T, NT>(x, v0, v1, k, buf, sh64);
    } else {
      for (int base = v0; n < k; base += NT) {
        // the first logits that equal tau: in order, a thread a logit
        const int at = base + tid;
        const bool hit = at < v1 && T::get(x[min(at, v1 - 1)]) == tau;
        const uint64_t b = __ballot(hit);
        if (lane == 0) sh64[wave] = b;
        __syncthreads();
        int pos = n + __popcll(b & ((1ull << lane) - 1)), all = 0;
        for (int w = 0; w < W; ++w) {
          const int c = __popcll(sh64[w]);
          if (w < wave) pos += c;
          all += c;
        }
        if (hit && pos < k) buf[pos] = order_key(tau, (uint32_t)at);
        n = min(k, n + all);
        __syncthreads();
        if (base + NT >= v1) break;        // (never short of k: at least k logits reach tau)
      }
      rank_keys<NT, C>(buf, n, k);
    }
    if (p.splits == 1) {
      if (tid == 0) p.lse[r] = log_sum(top, sum, p.c);
      for (int j = tid; j < k; j += NT) {
        const uint32_t id = ~(uint32_t)buf[j];
        p.ids[r * k + j] = id;
        // (the key holds a NaN as -inf)
        ((raw*)p.values)[r * k + j] = sum != sum ? x[id] : T::put(of_order((uint32_t)(buf[j] >> 32)));
      }
    } else {
      if (tid == 0) p.part_sums[blk] = make_float2(top, sum);
      for (int j = tid; j < p.k; j += NT) p.part_keys[blk * p.k + j] = j < k ? buf[j] : 0;
    }
    __syncthreads();
  }
}

template <class T>
lt_status launch_top(TopParams& p, void* stream) {
  const int64_t rows = p.rows < MAX_BLOCKS ? p.rows : MAX_BLOCKS;
  p.splits = 1;
  p.chunk = (p.x.vocab + 7) / 8 * 8;
  if (p.k > 192 ? p.x.vocab > 2048 : p.x.vocab > 16384)
    return launch(lt_top_k<T, 1024, 4, 2048>, rows, 1024, p, stream, "lt_top_logits");
  if (p.k > 62 || p.x.vocab > 2048) return launch(lt_top_k<T, 256, 4, 2048>, rows, 256, p, stream, "lt_top_logits");
  return launch(lt_top_k<T, 64, 4, 512>, rows, 64, p, stream, "lt_top_logits");
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
  return x->dtype == LT_F32 ? launch_top<F32>(p, stream) : x->dtype == LT_F16 ? launch_top<F16>(p, stream) : launch_top<BF16>(p, stream);
}

}  // extern "C"
