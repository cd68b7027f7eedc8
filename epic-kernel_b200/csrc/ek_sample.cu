// Token sampling: temperature, top-k, top-p and min-p, then one draw per row.
//
// All filters keep a prefix of the order (logit descending, index ascending),
// so a cut is a pair: the key of the last kept logit, and how many of its ties
// stay. Weights are exp((l - max) / T) in double, rounded to fixed point (at
// least 43 bits below the largest), so every sum is exact, in any order of the
// atomics, and a launch repeats bit for bit. Single precision would not do: a
// flat row has 10^5 borders that are 10^-5 apart, and each border's error
// moves some tokens.
//
// Finding a cut. Counts of the logits in 1024 (or 512) equal bins between the maximum
// and the lowest logit with a weight put a top-k cut into one bin, and, each
// count times the weight of the bin's centre, a top-p cut into one or two. One
// pass then adds up all weights exactly (which shows whether those bins hold
// the cut; if not, all logits are searched) and lists the logits of those bins,
// which go into histograms over their order-preserving integer keys until a
// bin is one value. When few tokens are left, up to 512, they are listed
// instead, and one block ranks them. For top-k <= 512
// the bins are filled with the largest logit of each thread only (with all of a
// short row): at least k logits lie at or above the bin where k are reached. bf16
// logits take few values: without top-k their weights come from a table of
// values, and for top-p a count per value gives the cut in one pass (64 rows of
// 128256 logits with top-p 0.95: 66 us before the table, 44 with it).
//
// A row is spread over a cluster of 1 to 8 blocks that hold it in shared
// memory, so it is read from HBM once; the blocks exchange maxima, histograms
// and sums through distributed shared memory. With more rows than such
// clusters fit at once, one block per row reads it again in each pass (mostly
// from L2), and with min-p alone it lists the kept tokens in the first pass,
// against the maximum so far. Bound: for many rows the bytes of the logits;
// for few the latency of the load and of the barriers; with a deep top-p cut
// the weights of fp32 logits (about 14 double operations each, twice) or, in
// bf16, the shared-memory atomics and lookups of the table.
// Kernel times: one row of 128256 bf16 logits with top-k 50 and top-p 0.9
// 11.5 us; 17 rows of 32003 fp32 logits 12.6; 64 rows of 128256 bf16 logits
// with top-p 0.95 43.5; 256 rows of 128256 fp32 logits with min-p 41 (3.2
// TB/s: 256 rows on 148 SMs leave 40 SMs with one row instead of two).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "ek_host.h"

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;
constexpr int kMaxElements = 65536;    // of a slice held in shared memory
constexpr int kMaxBytes = 176 * 1024;  // of logits per block
constexpr int kBatch = 4;
constexpr int kList = 512;   // tokens that one block ranks
// So many by counting, more by sorting (one row of 2000 fp32 logits: top-k 64 takes 7.9 and 9.7 us, 160 10.4 and 11.0,
// 256 18.1 and 12.4).
constexpr int kCount = 160;
constexpr int kRoom = 1024;  // a block's list; also room for all of one of 512 ranges of the index
constexpr int kRaw = 4096;   // logits listed against a maximum that still grows
// Table of bf16 values, 2^-9 <= |l| < 2^7, by falling value: 2048 positive, 2048 negative.
constexpr int kValues = 4096;
constexpr int kTableBytes = kValues * (sizeof(unsigned) + sizeof(unsigned long long));  // counts, weights
constexpr int kMaxVocab = kMaxCluster * kMaxBytes / 4;
using u64 = unsigned long long;

// Weights (up to 2^46) are added up in 32-bit limbs, the last with what is left: 16 bits each when a block sees a slice,
// 13 when it sees a whole row, so that no sum of equal weights reaches 2^32.
template <bool RESIDENT>
struct Limbs {
  static constexpr int N = RESIDENT ? 3 : 4, BITS = RESIDENT ? 16 : 13, MOST = RESIDENT ? kMaxElements : kMaxVocab;
  static_assert(((1ull << BITS) - 1) * MOST < 1ull << 32 && (1ull << (46 - BITS * (N - 1))) * MOST < 1ull << 32, "limbs");
};

struct SampleParams {
  const void* logits;
  long long row_stride;
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  long long* tokens;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all, vocab, weight_bits;
  int slice;  // elements per block, a multiple of 16
  int table;  // bytes of the slice when a table of values follows it, else 0
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// The largest and the smallest of 16 bytes of logits. NaN counts as not there (16 of NaN give NaN, which fmaxf ignores).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float most_of(const float (&x)[4]) { return max3(fmaxf(x[0], x[1]), x[2], x[3]); }
__device__ __forceinline__ float least_of(const float (&x)[4]) { return min3(fminf(x[0], x[1]), x[2], x[3]); }
__device__ __forceinline__ float most_of(const __nv_bfloat16 (&x)[8]) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(x);
  const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float least_of(const __nv_bfloat16 (&x)[8]) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(x);
  const __nv_bfloat162 m = __hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3]));
  return fminf(__low2float(m), __high2float(m));
}

// Order-preserving key of a logit that is not NaN; -0 counts as +0.
template <typename T>
__device__ __forceinline__ unsigned key_of(float l) {
  unsigned u = __float_as_uint(l + 0.f);
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  return sizeof(T) == 2 ? u >> 16 : u;
}
template <typename T>
__device__ __forceinline__ float value_of(unsigned key) {
  if (sizeof(T) == 2) key = key & 0x8000u ? key << 16 : key << 16 | 0xffffu;
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// Fixed-point weight 2^bits exp((l - top) / T).
//
// 2^(x / 32) with x = 32 log2(e) (l - top) / T split into a whole part n and a
// rest |r| <= 1/2: 2^(n div 32) * 2^((n mod 32) / 32) * e^(r ln 2 / 32). The
// last factor is its Taylor polynomial to the fifth power; |r ln 2 / 32| <=
// 0.0109 leaves an error below 0.0109^6 / 720 = 2.4e-15. The middle one is a
// table. Both roundings to whole numbers are additions of 1.5 * 2^52.
// An infinite maximum (then only infinite logits are weighed) counts as the largest finite number.
// Logits below `low` (and NaN) weigh 0: their weight is less than half a unit, and further down n div 32 is not the
// exponent of a number any more.
struct Weight {
  double top, c;       // c = 32 log2(e) / T
  const double* table; // 2^(j / 32), shared memory
  int bits;
  float low;

  __device__ __forceinline__ u64 operator()(float l) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    const double x = ((double)fminf(l, 3.402823466e38f) - top) * c;
    const double shifted = x + kRound;
    const int n = __double2loint(shifted);
    const double r = x - (shifted - kRound);
    constexpr double h = 0.021660849392498290;  // ln 2 / 32
    double p = h * h * h * h * h / 120.0;
    p = fma(p, r, h * h * h * h / 24.0);
    p = fma(p, r, h * h * h / 6.0);
    p = fma(p, r, h * h / 2.0);
    p = fma(p, r, h);
    p = fma(p, r, 1.0);
    p *= table[n & 31];
    p = __hiloint2double(__double2hiint(p) + ((n >> 5) + bits) * (1 << 20), __double2loint(p));
    const double whole = p + 4503599627370496.0;  // 2^52: the low bits are the rounded p
    return l >= low ? (u64)__double_as_longlong(whole) & 0xfffffffffffffull : 0;
  }
};

template <int kThreads, int kLimbs>
struct Shared {
  static constexpr int kWarps = kThreads / 32, kBins = kThreads;
  unsigned hist[2][kLimbs][kBins];  // counts, or the limbs of weights
  double table[32];
  double c, min_offset;        // 32 log2(e) / T; T ln(min_p)
  u64 scan[kWarps];
  float top[kMaxCluster], low[kMaxCluster];  // maxima and minima of the blocks
  u64 warp_weight[kMaxCluster * kWarps];     // per warp of the cluster: weight above the cut, ties
  unsigned warp_ties[kMaxCluster * kWarps];
  u64 block_above[kMaxCluster], block_total[kMaxCluster];
  u64 total[2], found_before;
  int found_bin, last_bin;
  int first[kMaxCluster];
  unsigned running_top;        // key of the largest logit so far
  int listed;                  // logits appended by this block; beyond kRaw (kRoom) they did not fit
  u64 extra[kWarps];           // listed logits above the cut, by the warp that owns their index: weight and ties
  unsigned extra_ties[kWarps];
  u64 list[kRoom];             // ~key << 32 | index
  u64 list_weight[kList];
};

// ceil(a / b) for quotients below 2^20: one float division, off by at most one, put right.
__device__ __forceinline__ u64 quotient_up(u64 a, u64 b) {
  u64 q = (u64)(unsigned)__fdividef((float)a, (float)b);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (q > 0 && (q - 1) * b >= a) --q;
    if (q * b < a) ++q;
  }
  return q;
}

// Inclusive scan over the block's threads.
template <int kThreads, int kLimbs>
__device__ u64 block_scan(u64 v, Shared<kThreads, kLimbs>& sh) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const u64 o = __shfl_up_sync(~0u, v, m);
    if (lane >= m) v += o;
  }
  if (lane == 31) sh.scan[warp] = v;
  __syncthreads();
  u64 t = lane < kWarps ? sh.scan[lane] : 0;
#pragma unroll
  for (int m = 1; m < kWarps; m <<= 1) {
    const u64 o = __shfl_up_sync(~0u, t, m);
    if (lane >= m) t += o;
  }
  const u64 earlier = __shfl_sync(~0u, t, (warp + 31) % 32);
  return warp ? v + earlier : v;
}

// Place of a bf16 value (its 16 bits) in the table; outside [0, kValues) halves for tiny values (callers check).
__device__ __forceinline__ int place_of(unsigned bits) {
  const int m = (int)(bits & 0x7fffu) - 0x3b00;
  return bits & 0x8000u ? kValues / 2 + m : kValues / 2 - 1 - m;
}
__device__ __forceinline__ bool tabled(unsigned bits) { return (bits & 0x7fffu) >= 0x3b00u; }  // (callers: below 2^7)
__device__ __forceinline__ float value_at(int place) {
  const int half = kValues / 2;
  const unsigned bits = place < half ? 0x3b00u + (half - 1 - place) : 0x8000u | (0x3b00u + place - half);
  return __uint_as_float(bits << 16);
}

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
};

// RESIDENT: a cluster holds the row in shared memory. Otherwise one block reads the row again in each pass.
template <typename T, bool RESIDENT, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_rows(const SampleParams p) {
  constexpr int kWarps = kThreads / 32, kBins = kThreads;
  constexpr int kBinBits = kThreads == 1024 ? 10 : 9;
  using V16 = Vec<T>;
  constexpr int N = V16::N;
  extern __shared__ uint4 dynamic[];
  T* slice = reinterpret_cast<T*>(dynamic);
  u64* raw_list = reinterpret_cast<u64*>(dynamic);  // without a resident slice
  using L = Limbs<RESIDENT>;
  __shared__ Shared<kThreads, L::N> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = RESIDENT ? cluster.num_blocks() : 1, rank = RESIDENT ? cluster.block_rank() : 0;
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int first = min(p.vocab, rank * p.slice), count = min(p.vocab - first, p.slice);
  const T* row = static_cast<const T*>(p.logits) + b * p.row_stride + first;
  auto sync = [&] {
    if (C > 1) cluster.sync();
    else __syncthreads();
  };
  if (C > 1) cluster.barrier_arrive();  // peers' shared memory may be written once all have started
  auto peer = [&](auto* at, int r) { return C > 1 ? cluster.map_shared_rank(at, r) : at; };

  const float inf = INFINITY;
  const int vectors = (count + N - 1) / N, whole = count / N;
  const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
  // vector i of the slice from memory, -inf past the end
  auto fetch = [&](int i) {
    V16 v;
    if (aligned && i < whole) {
      *reinterpret_cast<uint4*>(&v) = __ldg(reinterpret_cast<const uint4*>(row) + i);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v.x[e] = i * N + e < count ? row[i * N + e] : (T)-inf;
    }
    return v;
  };
  auto vec = [&](int i) {
    if (!RESIDENT) return fetch(i);
    const uint4 raw = reinterpret_cast<const uint4*>(slice)[i];
    return *reinterpret_cast<const V16*>(&raw);
  };
  // f(index in the slice, logit) for this thread's share; small bodies, so that a pass stays in the instruction cache
  auto for_each = [&](auto f) {
    if (RESIDENT) {
#pragma unroll 4
      for (int i = tid; i < count; i += kThreads) f(i, as_float(slice[i]));
    } else {
      V16 v, next, later;
      if (tid < vectors) next = fetch(tid);
      if (tid + kThreads < vectors) later = fetch(tid + kThreads);
#pragma unroll 1
      for (int i = tid; i < vectors; i += kThreads) {
        v = next, next = later;
        if (i + 2 * kThreads < vectors) later = fetch(i + 2 * kThreads);
#pragma unroll
        for (int e = 0; e < N; ++e) f(i * N + e, as_float(v.x[e]));
      }
    }
  };

  // the same, a contiguous range per warp: sums of warps run by index
  const int per_warp = (vectors + kWarps - 1) / kWarps;
  const int v0 = min(vectors, warp * per_warp), v1 = min(vectors, v0 + per_warp);
  // (four logits at a time, -inf past the end: their weights are independent chains of double operations)
  auto for_each_by_warp = [&](auto f) {
    const int end = min(count, v1 * N);
#pragma unroll 1
    for (int i = v0 * N + lane; i < end; i += 32 * kBatch) {
      float l[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int at = i + 32 * u;
        l[u] = at < end ? as_float(RESIDENT ? slice[at] : __ldg(row + at)) : -inf;
      }
      f(i, l);
    }
  };

  const float given = p.temperature ? p.temperature[b] : p.temperature_all;
  const bool flat = given == INFINITY;  // all weights are 1: as the largest finite temperature, but for min-p
  const float temp = flat ? 3.402823466e38f : given;
  const int k = p.top_k ? p.top_k[b] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float min_p = flat ? 0.f : p.min_p ? p.min_p[b] : p.min_p_all;
  const bool use_k = k > 0 && k < p.vocab, use_p = top_p < 1.f;
  // list the kept tokens while the row is read
  const bool online = !RESIDENT && min_p > 0.f && !use_k && !use_p && temp > 0.f;
  if (tid == 0) sh.listed = 0, sh.running_top = 0;
  if (online) {
    if (tid == 0) sh.min_offset = (double)temp * log((double)fminf(min_p, 1.f));
    __syncthreads();
  }
  // a little below T ln(min_p), for comparisons in single precision
  const float reach = online ? __double2float_rd(sh.min_offset * 1.000001) : 0.f;

  // ---- the maximum and the minimum above -inf; NaN fails every comparison, here and below
  float top = -inf, low = online ? -inf : inf;  // (the minimum only narrows the histograms)
  auto take = [&](float l) { top = fmaxf(top, l), low = l > -inf ? fminf(low, l) : low; };
  if (RESIDENT && !aligned) {  // element by element, so that a warp's loads are contiguous
    constexpr int U = 8;
    for (int i = tid; i < vectors * N; i += U * kThreads) {
      T w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = i + u * kThreads < count ? row[i + u * kThreads] : (T)-inf;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < vectors * N) take(as_float(w[u])), slice[i + u * kThreads] = w[u];
    }
  } else {
    constexpr int U = 4;
    V16 v[U], next[U];
    auto load = [&](V16 (&x)[U], int i) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < vectors) x[u] = fetch(i + u * kThreads);
    };
    if (!RESIDENT) load(next, tid);  // long slices: the next loads are under way while these are looked at
    for (int i = tid; i - lane < vectors; i += U * kThreads) {  // whole warps
      if (RESIDENT) {
        load(v, i);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
        load(next, i + U * kThreads);
      }
      float most[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < vectors) {
          most[u] = most_of(v[u].x);
          top = fmaxf(top, most[u]);
          if (!online) {
            float least = least_of(v[u].x);
            if (least == -inf) {
              least = inf;
#pragma unroll
              for (int e = 0; e < N; ++e) least = as_float(v[u].x[e]) > -inf ? fminf(least, as_float(v[u].x[e])) : least;
            }
            low = fminf(low, least);
          }
          if (RESIDENT) reinterpret_cast<uint4*>(slice)[i + u * kThreads] = *reinterpret_cast<uint4*>(&v[u]);
        }
      if (online) {
        // the largest logit seen by any warp bounds the final one from below
        unsigned key = __reduce_max_sync(~0u, top > -inf ? key_of<float>(top) : 0u);
        const unsigned seen = *reinterpret_cast<volatile unsigned*>(&sh.running_top);
        if (key > seen && lane == 0) atomicMax(&sh.running_top, key);
        key = max(key, seen);
        const float bar = key ? value_of<float>(key) + reach : inf;
        const float bar_down = bar < inf ? bar - fabsf(bar) * 0x1p-22f : inf;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i + u * kThreads >= vectors) continue;
          if (!(most[u] >= bar_down) || *reinterpret_cast<volatile int*>(&sh.listed) > kRaw) continue;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float l = as_float(v[u].x[e]);
            if (l >= bar_down && l > -inf) {
              const int at = atomicAdd(&sh.listed, 1);
              if (at < kRaw) raw_list[at] = (u64)~key_of<T>(l) << 32 | (unsigned)((i + u * kThreads) * N + e);
            }
          }
        }
      }
    }
  }
  const float mine_top = top;
  // the slow double functions once, on different warps
  if (warp == 1) sh.table[lane] = exp2((double)lane / 32.0);
  if (warp == 2 && lane == 0) sh.c = 46.166241308446828 / (double)temp;
  if (warp == 3 && lane == 0) sh.min_offset = min_p > 0.f ? (double)temp * log((double)fminf(min_p, 1.f)) : 0.0;
  for (int i = tid; i < L::N * kBins; i += kThreads) sh.hist[0][0][i] = 0;
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
    low = fminf(low, __shfl_xor_sync(~0u, low, m));
  }
  {
    float* wt = reinterpret_cast<float*>(sh.scan);
    if (lane == 0) wt[2 * warp] = top, wt[2 * warp + 1] = low;
    __syncthreads();
    if (C > 1) cluster.barrier_wait();
    if (warp == 0) {
      top = lane < kWarps ? wt[2 * lane] : -inf, low = lane < kWarps ? wt[2 * lane + 1] : inf;
#pragma unroll
      for (int m = 16; m; m >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
        low = fminf(low, __shfl_xor_sync(~0u, low, m));
      }
      if (lane < C) *peer(&sh.top[rank], lane) = top, *peer(&sh.low[rank], lane) = low;
    }
  }
  sync();
  top = sh.top[0], low = sh.low[0];
  for (int r = 1; r < C; ++r) top = fmaxf(top, sh.top[r]), low = fminf(low, sh.low[r]);

  if (!(temp > 0.f) || top == -inf) {  // the first of the largest; nothing above -inf gives 0
    int at = 0x7fffffff;
    if (top > -inf)
      for_each([&](int i, float l) { at = l == top ? min(at, first + i) : at; });
    at = __reduce_min_sync(~0u, at);
    int* wi = reinterpret_cast<int*>(sh.scan);
    __syncthreads();
    if (lane == 0) wi[warp] = at;
    __syncthreads();
    if (warp == 0) {
      at = __reduce_min_sync(~0u, lane < kWarps ? wi[lane] : 0x7fffffff);
      if (lane == 0) *peer(&sh.first[rank], 0) = at;
    }
    sync();
    if (rank == 0 && tid == 0) {
      for (int r = 0; r < C; ++r) at = min(at, sh.first[r]);
      p.tokens[b] = top > -inf ? at : 0;
    }
    return;
  }
  // below `low` a weight rounds to 0 and the token can never be drawn
  low = fmaxf(low, __double2float_ru((double)top - (double)temp * (0.6931471805599453 * (p.weight_bits + 1))));
  const Weight weight{(double)fminf(top, 3.402823466e38f), sh.c, sh.table, p.weight_bits, low};
  const float u01 = p.uniforms[b];
  // the draw among a weight of `total`: the first token whose running weight exceeds this
  auto target = [&](u64 total) {
    const u64 t = (u64)((double)(u01 > 0.f ? fminf(u01, 1.f) : 0.f) * (double)total);
    return min(t, total - 1);
  };
  // weight that must be reached for top-p; the first token always stays
  auto share = [&](u64 total) { return max((u64)ceil((double)fmaxf(top_p, 0.f) * (double)total), 1ull); };

  // ---- cuts: keys above `cut` stay, and the first `ties` (by index) of those equal to it
  // (the first value of the logits' type at or above a border: a key of bf16 is cut off downwards for positive logits)
  auto first_key = [&](float l) { return key_of<T>(sizeof(T) == 2 ? __bfloat162float(__float2bfloat16_ru(l)) : l); };
  unsigned cut = first_key(low);
  u64 ties = ~0ull;
  if (min_p > 0.f) cut = max(cut, first_key(fminf(__double2float_ru((double)top + sh.min_offset), top)));

  // Finishes the row from the n <= kList listed tokens, which are all that may stay. `goal`: the weight for top-p, 0 if
  // it follows from the list.
  auto finish_sorted = [&](int n, u64 goal) {
    // `own` of threads 0 .. n - 1 in rising order (bitonic; exchanges within a warp by shuffles)
    auto sort = [&](u64 own) {
      for (int size = 2; size < 2 * n; size *= 2)
        for (int j = size / 2; j > 0; j /= 2) {
          u64 other;
          if (j < 32) {
            other = __shfl_xor_sync(~0u, own, j);
          } else {
            __syncthreads();
            if (tid < kList) sh.list[tid] = own;
            __syncthreads();
            other = tid < kList ? sh.list[tid ^ j] : ~0ull;
          }
          if ((own < other) == (((tid & j) != 0) == ((tid & size) == 0))) own = other;
        }
      return own;
    };
    __syncthreads();
    // by falling logit, then by rising index
    const u64 own = sort(tid < n ? sh.list[tid] : ~0ull);
    const unsigned key = ~(unsigned)(own >> 32);
    bool stay = tid < n && (!use_k || tid < k);
    const u64 w = stay ? weight(value_of<T>(key)) : 0;
    if (use_p) {
      const u64 upto = block_scan(w, sh);
      if (goal == 0) {
        if (tid == kThreads - 1) sh.found_before = upto;
        __syncthreads();
        goal = share(sh.found_before);
      }
      stay = stay && upto - w < goal;
    }
    stay = stay && key >= cut;
    // what stays, by rising index
    if (tid < kList) sh.list_weight[tid] = w;
    const u64 next = sort(stay ? own << 32 | (unsigned)tid : ~0ull);
    __syncthreads();
    const u64 its = next != ~0ull ? sh.list_weight[(unsigned)next] : 0, upto = block_scan(its, sh);
    if (tid == kThreads - 1) sh.found_before = upto;
    __syncthreads();
    const u64 t = target(sh.found_before);
    if (upto - its <= t && t < upto) p.tokens[b] = (long long)(next >> 32);
  };
  // The same by counting, for each token, those ahead of it.
  auto finish = [&](int n, u64 goal) {
    if (kThreads == 1024 || n > kCount) {  // 1024 threads lack the registers for both (64 rows, top-p: 48 us, not 44)
      finish_sorted(n, goal);
      return;
    }
    int parts = 1;  // neighbouring lanes that share a token
    while (parts < 32 && n * parts * 2 <= kThreads) parts *= 2;
    const int i = tid / parts, sub = tid % parts;
    const u64 own = i < n ? sh.list[i] : 0;
    const unsigned key = ~(unsigned)(own >> 32);
    const u64 w = i < n ? weight(value_of<T>(key)) : 0;
    if (i < n && sub == 0) sh.list_weight[i] = w;
    __syncthreads();
    int rank_of = 0;
    u64 before = 0;
    if (use_k || use_p) {
#pragma unroll 8
      for (int j = sub; j < n; j += parts) {
        const u64 x = sh.list_weight[j];
        const bool ahead = sh.list[j] < own;
        rank_of += ahead, before += ahead ? x : 0;
      }
    }
    for (int m = 1; m < parts; m <<= 1) {
      rank_of += __shfl_xor_sync(~0u, rank_of, m);
      before += __shfl_xor_sync(~0u, before, m);
    }
    bool stay = i < n && (!use_k || rank_of < k);
    if (use_p) {
      if (goal == 0) {
        const u64 sum = block_scan(stay && sub == 0 ? w : 0, sh);
        if (tid == kThreads - 1) sh.found_before = sum;
        __syncthreads();
        goal = share(sh.found_before);
      }
      stay = stay && before < goal;
    }
    stay = stay && key >= cut;
    __syncthreads();
    if (i < n && sub == 0) sh.list_weight[i] = stay ? w : 0;
    const u64 sum = block_scan(stay && sub == 0 ? w : 0, sh);
    if (tid == kThreads - 1) sh.found_before = sum;
    __syncthreads();
    if (!__any_sync(~0u, stay)) return;
    before = 0;
#pragma unroll 8
    for (int j = sub; j < n; j += parts) {
      const u64 x = sh.list_weight[j];
      before += (unsigned)sh.list[j] < (unsigned)own ? x : 0;
    }
    for (int m = 1; m < parts; m <<= 1) before += __shfl_xor_sync(~0u, before, m);
    if (stay && sub == 0) {
      const u64 t = target(sh.found_before);
      if (before <= t && t < before + w) p.tokens[b] = (long long)(unsigned)own;
    }
  };
  auto add_weight = [&](int buffer, int bin, u64 w) {
#pragma unroll
    for (int e = 0; e < L::N; ++e)
      atomicAdd(&sh.hist[buffer][e][bin], (unsigned)(w >> (L::BITS * e)) & (e + 1 < L::N ? (1u << L::BITS) - 1 : ~0u));
  };
  if (online && sh.listed <= kRaw) {
    // All kept tokens are listed. Their weights by ranges of the index, 512 of them; the range that holds the draw
    // is small enough to compare its tokens with each other.
    const int n = sh.listed, wide = (p.vocab + kBins - 1) / kBins;
    for (int i = tid; i < n; i += kThreads) {
      const u64 own = raw_list[i];
      const unsigned key = ~(unsigned)(own >> 32);
      if (key < cut) continue;  // ruled out by the final maximum
      const int at = (int)((unsigned)own / wide);
      const u64 w = weight(value_of<T>(key));
      add_weight(0, at, w);
    }
    __syncthreads();
    u64 mine = 0;
#pragma unroll
    for (int e = 0; e < L::N; ++e) mine += (u64)sh.hist[0][e][tid] << (L::BITS * e);
    const u64 sum = block_scan(mine, sh);
    if (tid == kThreads - 1) sh.found_before = sum;
    __syncthreads();
    const u64 goal = target(sh.found_before);
    __syncthreads();
    if (sum > goal && sum - mine <= goal) sh.found_bin = tid, sh.found_before = sum - mine;
    __syncthreads();
    const u64 before_range = sh.found_before;
    const unsigned from = sh.found_bin * wide;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const u64 own = raw_list[i];
      if ((unsigned)own - from < (unsigned)wide && ~(unsigned)(own >> 32) >= cut)
        sh.list[atomicAdd(&sh.listed, 1)] = own;
    }
    __syncthreads();
    for (int i = tid; i < sh.listed; i += kThreads) {
      const unsigned index = (unsigned)sh.list[i];
      u64 before = before_range;
      for (int j = 0; j < sh.listed; ++j)
        if ((unsigned)sh.list[j] < index) before += weight(value_of<T>(~(unsigned)(sh.list[j] >> 32)));
      const u64 w = weight(value_of<T>(~(unsigned)(sh.list[i] >> 32)));
      if (before <= goal && goal < before + w) p.tokens[b] = (long long)index;
    }
    return;
  }

  int buffer = 0;
  const float bins_per = top > low && top < inf ? fminf((float)(kBins - 1) / (top - low), 3e38f) : 0.f;
  // (top - l) * bins_per to the nearest whole number, by an addition of 1.5 * 2^23; within 0 .. kBins - 1 for
  // l >= low. An infinite maximum makes it NaN and the bin kBins - 1.
  auto bin_of = [&](float l) {
    return (int)(__float_as_uint(fmaf(top - l, bins_per, 12582912.f)) & (kBins - 1));
  };
  // An upper (-1/2) or lower (+1/2) bound of the logits of a bin, widened by the rounding of bin_of.
  auto edge_of = [&](int bin, float half) {
    const float margin = (top - low) * 0x1p-18f + fmaxf(fabsf(top), fabsf(low)) * 0x1p-20f;
    return top - ((float)bin + half) / bins_per - copysignf(margin, half);
  };
  // The cluster's sum of bin `tid` of the current histogram (one count, or the limbs); call after sync(). Turns
  // to the other buffer, which is free: its last readers were past it before that barrier.
  auto collect = [&](bool limbs) {
    constexpr int R = RESIDENT ? kMaxCluster : 1;
    unsigned h[L::N][R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < C) {
        const unsigned* other = peer(&sh.hist[buffer][0][0], r);
        h[0][r] = other[tid];
#pragma unroll
        for (int e = 1; e < L::N; ++e)
          if (limbs) h[e][r] = other[e * kBins + tid];
      }
    u64 sum = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < C) {
        sum += h[0][r];
#pragma unroll
        for (int e = 1; e < L::N; ++e) sum += limbs ? (u64)h[e][r] << (L::BITS * e) : 0;
      }
    buffer ^= 1;
    for (int i = tid; i < L::N * kBins; i += kThreads) sh.hist[buffer][0][i] = 0;
    return sum;
  };
  // All blocks' lists together in the first block's: their number, or -1 (nothing moved) if they are too many.
  auto join_lists = [&] {
    int sum = lane < C ? *peer(&sh.listed, lane) : 0, mine = lane < rank ? sum : 0;
    sum = __reduce_add_sync(~0u, sum), mine = __reduce_add_sync(~0u, mine);
    if (sum > kList) return -1;
    if (rank > 0)
      for (int i = tid; i < sh.listed; i += kThreads) *peer(&sh.list[mine + i], 0) = sh.list[i];
    sync();
    return sum;
  };
  auto append = [&](unsigned key, int index) {
    if (*reinterpret_cast<volatile int*>(&sh.listed) > kRoom) return;
    const int at = atomicAdd(&sh.listed, 1);
    if (at < kRoom) sh.list[at] = (u64)~key << 32 | (unsigned)index;
  };

  // Short rows (of one block) as a whole: one of 128 with top-p takes 7 us, one of 512 11; one of 513 18, but with top-k
  // 50 too, 8.
  if (p.vocab <= 128 || (p.vocab <= kList && use_p && !use_k)) {
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    for_each([&](int i, float l) {
      if (l >= low) append(key_of<T>(l), i);
    });
    __syncthreads();
    finish(sh.listed, 0);
    return;
  }
  if (use_k && k <= kList) {  // at least k logits lie in the bins down to that of the k-th largest thread maximum
    if (tid == 0) sh.listed = 0;
    if (vectors <= kThreads) {  // short rows have too few maxima: all logits (129 of them, k = 20: 8 us, not 33)
      for_each([&](int, float l) {
        if (l >= low) atomicAdd(&sh.hist[buffer][0][bin_of(l)], 1u);
      });
    } else if (mine_top >= low) {
      atomicAdd(&sh.hist[buffer][0][bin_of(mine_top)], 1u);
    }
    sync();
    const u64 count_here = collect(false);
    const u64 sum = block_scan(count_here, sh);
    if (tid == kThreads - 1) sh.found_bin = -1;
    __syncthreads();
    if (sum >= (u64)k && sum - count_here < (u64)k) sh.found_bin = tid;
    __syncthreads();
    const int last = sh.found_bin;
    if (last >= 0) {
      const float bar = last == kBins - 1 || bins_per == 0.f ? low : fmaxf(low, edge_of(last, 0.5f));
      if (RESIDENT) {  // 16 bytes at a time: most hold nothing above the bar
#pragma unroll 2
        for (int i = tid; i < vectors; i += kThreads) {
          const V16 v = vec(i);
          if (!(most_of(v.x) >= bar)) continue;
          unsigned hits = 0;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float l = as_float(v.x[e]);
            hits |= l >= bar && bin_of(l) <= last ? 1u << e : 0;
          }
          for (; hits; hits &= hits - 1) {
            const int j = i * N + __ffs(hits) - 1;
            append(key_of<T>(as_float(slice[j])), first + j);
          }
        }
      } else {
        for_each([&](int i, float l) {
          if (l >= bar && bin_of(l) <= last) append(key_of<T>(l), first + i);
        });
      }
      sync();
      const int n = join_lists();
      if (n >= 0) {
        if (rank == 0) finish(n, 0);
        return;
      }
    }
    sync();  // sh.listed and the lists may be used again
  }

  unsigned weighed_cut = 0;  // the cut of top-p, when `weighed` holds this thread's weights
  u64 weighed = 0;           // above weighed_high; the logits in question are those from there down
  float weighed_high = 0.f;
  bool listed = false;       // sh.list holds this block's logits in question
  unsigned k_cut = 0;  // top-k keeps keys above, and k_ties equal ones
  u64 k_ties = 0;
  // bf16 logits take few values: a table of their weights, and for top-p a count per value, which gives the cut at once
  bool by_value = false;
  unsigned* counts_at = reinterpret_cast<unsigned*>(reinterpret_cast<uint8_t*>(dynamic) + p.table);
  u64* weight_at = reinterpret_cast<u64*>(counts_at + kValues);
  const bool table = sizeof(T) == 2 && RESIDENT && p.table && !use_k && top < 128.f && low > -128.f;
  if (table && !use_p && !(min_p > 0.f)) {  // min-p leaves too few weights
    for (int i = tid; i < kValues; i += kThreads) {
      const float l = value_at(i);
      weight_at[i] = l <= top ? weight(l) : 0;
    }
    __syncthreads();
    by_value = true;
  } else if (table && use_p) {
    constexpr int PER = kValues / kThreads;
    for (int i = tid; i < kValues / 4; i += kThreads) reinterpret_cast<uint4*>(counts_at)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    u64 tiny = 0;
#pragma unroll 2
    for (int i = tid; i < vectors; i += kThreads) {
      const V16 v = vec(i);
      bool any = false;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float l = as_float(v.x[e]);
        const unsigned bits = __float_as_uint(l) >> 16;
        any |= l >= low && !tabled(bits);
        if (l >= low && tabled(bits)) atomicAdd(counts_at + place_of(bits), 1u);
      }
      if (any) {
#pragma unroll 1
        for (int e = i * N; e < (i + 1) * N; ++e) {
          const float l = as_float(slice[e]);
          if (l >= low && !tabled(__float_as_uint(l) >> 16)) tiny += weight(l);
        }
      }
    }
    const u64 block_tiny = block_scan(tiny, sh);
    if (tid == kThreads - 1)
      for (int r = 0; r < C; ++r) *peer(&sh.block_total[rank], r) = block_tiny;
    if (tid == 0) sh.found_bin = -1;
    sync();
    tiny = 0;
    for (int r = 0; r < C; ++r) tiny += sh.block_total[r];
    u64 n[PER], w[PER], mine = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) n[e] = 0;
    for (int r = 0; r < C; ++r) {
      const unsigned* other = peer(counts_at, r) + tid * PER;
#pragma unroll
      for (int e = 0; e < PER; e += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(other + e);
        n[e] += x.x, n[e + 1] += x.y, n[e + 2] += x.z, n[e + 3] += x.w;
      }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      w[e] = n[e] ? weight(value_at(tid * PER + e)) : 0;
      weight_at[tid * PER + e] = w[e];
      mine += n[e] * w[e];
    }
    const u64 upto = block_scan(mine, sh);
    if (tid == kThreads - 1) sh.found_before = upto;
    __syncthreads();
    const u64 goal = share(sh.found_before + tiny);
    u64 before = upto - mine + (tid * PER >= kValues / 2 ? tiny : 0);  // the tiny values lie between the halves
    if (before < goal && goal <= before + mine) {
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const u64 all = n[e] * w[e];
        if (before < goal && goal <= before + all) {
          sh.found_bin = (int)key_of<T>(value_at(tid * PER + e));
          sh.total[0] = quotient_up(goal - before, w[e]);
        }
        before += all;
      }
    }
    __syncthreads();
    by_value = sh.found_bin >= 0;  // else the cut is among the tiny values: the general search finds it
    if (by_value) {
      const unsigned key = (unsigned)sh.found_bin;
      const u64 r = sh.total[0];
      if (key > cut) cut = key, ties = r;
      else if (key == cut) ties = min(ties, r);
    }
    __syncthreads();
  }
  for (int stage = 0; stage < 2; ++stage) {  // 0: top-k; 1: top-p among what top-k left
    if (stage == 0 ? !use_k : !use_p || by_value) continue;
    // the lowest logit that takes part; NaN (none) above an infinite k_cut
    const float next = value_of<T>(k_cut + 1);
    const float lowest = stage == 0 || k_cut == 0 || next <= low ? low : next;
    auto takes_part = [&](float l) { return l >= lowest; };
    if (tid == 0) sh.listed = 0;
    listed = false;
    for_each([&](int, float l) {
      const int bin = bin_of(l);
      if (takes_part(l)) atomicAdd(&sh.hist[buffer][0][bin], 1u);
    });
    sync();
    const u64 tied = stage == 1 && k_ties ? k_ties * weight(value_of<T>(k_cut)) : 0;
    const u64 counted = collect(false);
    const u64 counts = block_scan(counted, sh);
    int candidates = kList + 1;
    u64 goal = k, before = 0;
    if (tid == 0) sh.found_bin = kBins;
    if (tid == kThreads - 1) sh.found_before = counts;
    __syncthreads();
    if (stage == 0 && sh.found_before < goal) {  // fewer than k have a weight: all stay
      __syncthreads();
      continue;
    }
    u64 about = counted, sum_about = counts, goal_about = goal;
    if (stage == 1) {
      const float centre = bins_per > 0.f ? top - (float)tid / bins_per : top;
      about = counted ? counted * weight(fmaxf(centre, low)) : 0;
      sum_about = block_scan(about, sh);
      __syncthreads();
      if (tid == kThreads - 1) sh.found_before = sum_about;
      __syncthreads();
      goal_about = share(sh.found_before + tied);
    }
    if (counted && sum_about >= goal_about && sum_about - about < goal_about) {
      // near an edge of the bin, the neighbour too
      const float part = stage == 0 ? 0.5f : (float)(goal_about - (sum_about - about)) / (float)about;
      sh.found_bin = part < 0.05f ? max(tid - 1, 0) : tid;
      sh.last_bin = part > 0.95f ? min(tid + 1, kBins - 1) : tid;
    }
    __syncthreads();
    const int d1 = sh.found_bin, d2 = sh.last_bin;  // d1 == kBins: the cut seems to lie among the ties of top-k
    if (d1 < kBins && tid == d2) sh.found_before = counts;
    __syncthreads();
    if (stage == 1 && d1 < kBins && k_ties == 0) candidates = (int)min(sh.found_before, (u64)kList + 1);
    // the logits in question, whatever their bins: keys base .. high
    unsigned high = key_of<T>(top), base = key_of<T>(low);
    if (d1 == kBins) {
      high = base, base = base + 1;  // none
    } else if (bins_per > 0.f) {
      const float hi = edge_of(d1, -0.5f), lo = edge_of(d2, 0.5f);
      if (hi < top) high = key_of<T>(hi);
      if (lo > low && d2 < kBins - 1) base = key_of<T>(lo);
      high = max(high, base);
    }
    bool gather = candidates <= kList;
    bool all = false, weigh = true, reuse = stage == 1;  // weigh: add up all weights (counts), once
    for (int pass = 0;;) {
      const bool none = high < base;
      const unsigned span = none ? 0 : high - base;  // bins of 2^shift keys
      const int shift = span < kBins ? 0 : 32 - __clz(span) - kBinBits;
      u64 above = 0, total = 0;
      const float high_value = none ? -inf : value_of<T>(high), base_value = none ? inf : value_of<T>(base);
      const float reach_value = gather ? inf : high_value;
      auto count_key = [&](float l) {  // into the histogram of keys
        const unsigned key = key_of<T>(l);
        if (key > high || key < base) return;
        const int at = (int)((high - key) >> shift);
        if (stage == 0) {
          atomicAdd(&sh.hist[buffer][0][at], 1u);
        } else {
          add_weight(buffer, at, weight(l));
        }
      };
      if (weigh && stage == 0) {
        for_each([&](int i, float l) {
          if (l > high_value) ++above;
          else if (l >= base_value) append(key_of<T>(l), first + i);
        });
      } else if (weigh) {
        for_each_by_warp([&](int i, const float (&l)[kBatch]) {
          u64 w[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) w[u] = weight(l[u]);
          unsigned hits = 0;
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const bool in = takes_part(l[u]);
            total += in ? w[u] : 0;
            above += in && l[u] > high_value ? w[u] : 0;
            hits |= in && l[u] >= base_value && l[u] <= reach_value ? 1u << u : 0;
          }
          while (hits) {
            const int u = __ffs(hits) - 1;
            hits &= hits - 1;
            const int at = i + 32 * u;
            append(key_of<T>(as_float(RESIDENT ? slice[at] : row[at])), first + at);
          }
        });
      }
      if (weigh) {  // the block's sums to every block
        weighed = above, weighed_high = high_value;
        const u64 block_above = block_scan(above, sh);
        __syncthreads();
        const u64 block_total = block_scan(total, sh);
        if (tid == kThreads - 1)
          for (int r = 0; r < C; ++r)
            *peer(&sh.block_above[rank], r) = block_above, *peer(&sh.block_total[rank], r) = block_total;
        listed = sh.listed <= kRoom;
      }
      if (listed) {
        for (int i = tid; i < sh.listed; i += kThreads) count_key(value_of<T>(~(unsigned)(sh.list[i] >> 32)));
      } else {
        for_each([&](int, float l) {
          if (l >= base_value && l <= high_value && takes_part(l)) count_key(l);
        });
      }
      sync();
      if (weigh) {
        u64 sum = tied;
        for (int r = 0; r < C; ++r) sum += sh.block_total[r], before += sh.block_above[r];
        if (stage == 1) goal = share(sum);
      }
      const u64 mine = collect(stage == 1);
      const u64 sum = before + block_scan(mine, sh);
      if (tid == kThreads - 1) sh.found_bin = kBins, sh.found_before = sum;
      __syncthreads();
      const bool below = sh.found_before < goal, beside = before >= goal;
      __syncthreads();
      if (beside || below) {
        const bool whole = high == key_of<T>(top) && base == key_of<T>(low);
        if (whole || (below && d1 == kBins)) {  // among the ties of top-k
          all = true;
          break;
        }
        high = key_of<T>(top), base = key_of<T>(low), before = 0;  // not here: search all
        gather = weigh = reuse = listed = false;
        continue;
      }
      weigh = false;
      if (gather) {
        gather = false;
        const int n = join_lists();
        if (n >= 0) {
          if (rank == 0) finish(n, goal);
          return;
        }
      }
      if (sum >= goal && sum - mine < goal) sh.found_bin = tid, sh.found_before = sum - mine;
      __syncthreads();
      before = sh.found_before;
      high -= (unsigned)sh.found_bin << shift;
      if (shift == 0 || ++pass == 4) break;  // at least 9 bits a pass: four are enough for 32
      base = max(base, high - ((1u << shift) - 1u));
    }
    if (all) before = sh.found_before;
    __syncthreads();
    const unsigned key = all ? k_cut : high;
    const u64 unit = stage == 0 ? 1 : weight(value_of<T>(key));
    u64 r = quotient_up(goal - before, max(unit, 1ull));
    if (stage == 0) k_cut = key, k_ties = r;
    else if (all) r = min(r, k_ties);
    else if (reuse) weighed_cut = key;
    if (key > cut) cut = key, ties = r;
    else if (key == cut) ties = min(ties, r);
  }

  // ---- the draw: a warp owns a contiguous range, so that sums run by index
  const float cut_value = value_of<T>(cut);
  u64 above = 0;
  unsigned tied = 0;
  if (cut == weighed_cut) {  // top-p has added up all weights but those of its bins
    above = weighed;
    if (listed) {
      if (tid < kWarps) sh.extra[tid] = 0, sh.extra_ties[tid] = 0;
      __syncthreads();
      for (int i = tid; i < sh.listed; i += kThreads) {
        const float l = value_of<T>(~(unsigned)(sh.list[i] >> 32));
        const int owner = (int)((unsigned)sh.list[i] - first) / N / per_warp;
        if (l > cut_value && l <= weighed_high) atomicAdd(&sh.extra[owner], weight(l));
        if (l == cut_value) atomicAdd(&sh.extra_ties[owner], 1u);
      }
      __syncthreads();
      if (lane == 0) above += sh.extra[warp], tied = sh.extra_ties[warp];
    } else {
      for_each_by_warp([&](int, const float (&l)[kBatch]) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          tied += l[u] == cut_value;
          if (l[u] > cut_value && l[u] <= weighed_high) above += weight(l[u]);
        }
      });
    }
  } else if (by_value) {
#pragma unroll 2
    for (int i = v0 + lane; i < v1; i += 32) {
      const V16 v = vec(i);
      u64 w[N];
      bool tiny = false;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float l = as_float(v.x[e]);
        const unsigned bits = __float_as_uint(l) >> 16;
        const bool in = l > cut_value;
        tied += l == cut_value;
        tiny |= in && !tabled(bits);
        w[e] = 0;
        if (in && tabled(bits)) w[e] = weight_at[place_of(bits)];
      }
#pragma unroll
      for (int e = 0; e < N; ++e) above += w[e];
      if (tiny) {
#pragma unroll 1
        for (int e = i * N; e < (i + 1) * N; ++e) {
          const float l = as_float(slice[e]);
          if (l > cut_value && !tabled(__float_as_uint(l) >> 16)) above += weight(l);
        }
      }
    }
  } else {
    for_each_by_warp([&](int, const float (&l)[kBatch]) {
      bool any = false;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        tied += l[u] == cut_value;
        any |= l[u] > cut_value;
      }
      if (!any) return;
      u64 w[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) w[u] = weight(l[u]);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) above += l[u] > cut_value ? w[u] : 0;
    });
  }
  tied = __reduce_add_sync(~0u, tied);
#pragma unroll
  for (int m = 16; m; m >>= 1) above += __shfl_xor_sync(~0u, above, m);
  if (lane < C) {
    *peer(&sh.warp_weight[rank * kWarps + warp], lane) = above;
    *peer(&sh.warp_ties[rank * kWarps + warp], lane) = tied;
  }
  sync();
  // each warp finds the range that holds the draw from all warps' sums, four per lane
  const u64 unit = weight(cut_value);
  constexpr int E = (RESIDENT ? kMaxCluster : 2) * kWarps / 32;
  u64 w[E], t[E], weights = 0, tie_sum = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane * E + e;
    w[e] = i < C * kWarps ? sh.warp_weight[i] : 0;
    t[e] = i < C * kWarps ? sh.warp_ties[i] : 0;
    tie_sum += t[e];
  }
  u64 tie_before = tie_sum;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const u64 o = __shfl_up_sync(~0u, tie_before, m);
    if (lane >= m) tie_before += o;
  }
  tie_before -= tie_sum;
  u64 ahead[E];  // ties before each range
#pragma unroll
  for (int e = 0; e < E; ++e) {
    ahead[e] = tie_before;
    w[e] += (min(ties, tie_before + t[e]) - min(ties, tie_before)) * unit;
    tie_before += t[e];
    weights += w[e];
  }
  u64 upto = weights;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const u64 o = __shfl_up_sync(~0u, upto, m);
    if (lane >= m) upto += o;
  }
  const u64 goal = target(__shfl_sync(~0u, upto, 31));
  u64 running = upto - weights;
  int owner = -1;
  u64 owner_before = 0, owner_ties = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (owner < 0 && running <= goal && goal < running + w[e])
      owner = lane * E + e, owner_before = running, owner_ties = ahead[e];
    running += w[e];
  }
  const int from = __ffs(__ballot_sync(~0u, owner >= 0)) - 1;
  owner = __shfl_sync(~0u, owner, from);
  auto weight_of = [&](float l) {
    const unsigned bits = __float_as_uint(l) >> 16;
    return by_value && tabled(bits) ? weight_at[place_of(bits)] : weight(l);
  };
  if (owner == rank * kWarps + warp) {
    u64 sum = __shfl_sync(~0u, owner_before, from), seen = __shfl_sync(~0u, owner_ties, from);
    for (int i0 = v0; i0 < v1; i0 += 32) {
      const int i = i0 + lane;
      V16 v;
      unsigned mine = 0;
      u64 heavy = 0;
      if (i < v1) {
        v = vec(i);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float l = as_float(v.x[e]);
          mine += l == cut_value;
          if (l > cut_value) heavy += weight_of(l);
        }
      }
      unsigned tb = mine;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const unsigned o = __shfl_up_sync(~0u, tb, m);
        if (lane >= m) tb += o;
      }
      const u64 t0 = seen + tb - mine;
      heavy += (min(ties, t0 + mine) - min(ties, t0)) * unit;
      u64 hb = heavy;
#pragma unroll
      for (int m = 1; m < 32; m <<= 1) {
        const u64 o = __shfl_up_sync(~0u, hb, m);
        if (lane >= m) hb += o;
      }
      u64 at = sum + hb - heavy;
      if (at <= goal && goal < at + heavy) {
        u64 tt = t0;
        int pick = -1;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float l = as_float(v.x[e]);
          if (l > cut_value) at += weight_of(l);
          else if (l == cut_value && tt++ < ties) at += unit;
          if (pick < 0 && at > goal) pick = e;
        }
        p.tokens[b] = first + i * N + pick;
      }
      sum += __shfl_sync(~0u, hb, 31);
      seen += __shfl_sync(~0u, tb, 31);
      if (sum > goal) break;
    }
  }
  if (C > 1) cluster.sync();  // no block leaves while another reads its shared memory
}

template <typename T, bool RESIDENT, int kThreads>
cudaError_t launch(const SampleParams& p, int blocks, int cluster, int bytes, cudaStream_t st) {
  const auto kernel = sample_rows<T, RESIDENT, kThreads>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             RESIDENT ? kMaxBytes : kRaw * (int)sizeof(u64));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T>
cudaError_t launch(SampleParams& p, int batch, cudaStream_t st) {
  const int size = sizeof(T);
  auto slice = [&](int n) { return (int)(((long long)p.vocab + n - 1) / n + 15) / 16 * 16; };
  auto fits = [&](int n) { return slice(n) <= kMaxElements && slice(n) * size <= kMaxBytes; };
  // Blocks per row: up to 8 that keep 2048 elements each and run at once with the other rows' (what fits of
  // clusters of 2, 4 and 8: 148, 71 and 33 with two blocks of 512 threads on an SM, 74, 33 and 15 with one of 1024).
  // Rows whose cut or weights come from the table of values (bf16, no top-k, top-p) take blocks of 1024: with the
  // table two blocks of 512 do not fit an SM. More than 4 give nothing there, since each block adds up all blocks'
  // counts (33 rows of 128256: 32 us on 4 x 1024, 50 on 8 x 512 without the table; one row 34 and 31 on 4 and 8).
  const bool no_k = !p.top_k && (p.top_k_all <= 0 || p.top_k_all >= p.vocab);
  const bool by_value = size == 2 && no_k && p.vocab > kList && (p.top_p || p.top_p_all < 1.f);
  int cluster = 1, threads = 512;
  while (cluster < kMaxCluster && p.vocab >= cluster * 4096 && batch <= (cluster == 1 ? 148 : cluster == 2 ? 71 : 33))
    cluster *= 2;
  // Beyond 148 rows two blocks of 512 with the table share an SM while the row leaves room (155 rows of 19592: 33 us,
  // 42 on 1 x 1024; 32000: 61 and 51).
  const int block_bytes = slice(1) * size + kTableBytes + (int)sizeof(Shared<512, 3>) + 1024;
  const bool pairs = by_value && batch > 148 && 2 * block_bytes <= 228 * 1024;
  if (pairs) {
    cluster = 1;
  } else if (by_value || slice(cluster) >= 32000 || slice(cluster) * size > 72 * 1024) {
    // Much work per block: 1024 threads (40 plain rows of 128256 33 us on 2 x 1024, 35 on 4 x 512; one row with top-k
    // 15.3 us on 8 x 1024, 11.5 on 8 x 512).
    threads = 1024;
    cluster = 1;
    while (cluster < kMaxCluster &&
           ((p.vocab >= cluster * 4096 && batch <= (cluster == 1 ? 74 : cluster == 2 ? 33 : by_value ? 0 : 15)) ||
            (!fits(cluster) && batch < 148)))
      cluster *= 2;
  }
  if (!fits(cluster)) {  // from 148 rows on: one block per row reads it in every pass
    p.slice = slice(1);
    return launch<T, false, 512>(p, batch, 1, kRaw * sizeof(u64), st);
  }
  p.slice = slice(cluster);
  // The table of values goes behind the slice.
  const int bytes = p.slice * size;
  if (size == 2 && (threads == 1024 || pairs)) p.table = bytes;
  const int all = bytes + (p.table ? kTableBytes : 0);
  if (threads == 1024) return launch<T, true, 1024>(p, batch * cluster, cluster, all, st);
  return launch<T, true, 512>(p, batch * cluster, cluster, all, st);
}

}  // namespace

extern "C" int ek_sample(const EkSampleArgs* a, void* stream) {
  using ek::fail;
  if (!a) return fail(EK_E_INVALID, "NULL arguments");
  if (a->batch < 0 || a->vocab < 1) return fail(EK_E_INVALID, "bad sizes batch=%d vocab=%d", a->batch, a->vocab);
  if (a->vocab > kMaxVocab) return fail(EK_E_UNSUPPORTED, "vocab %d (at most %d)", a->vocab, kMaxVocab);
  if (a->batch > (1 << 27)) return fail(EK_E_UNSUPPORTED, "batch %d", a->batch);
  if (a->batch == 0) return EK_SUCCESS;
  if (!a->logits || !a->uniforms || !a->tokens) return fail(EK_E_INVALID, "NULL pointer argument");
  SampleParams p = {};
  p.logits = a->logits;
  p.row_stride = a->row_stride;
  p.uniforms = a->uniforms;
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.tokens = reinterpret_cast<long long*>(a->tokens);
  p.temperature_all = a->temperature_all;
  p.top_k_all = a->top_k_all;
  p.top_p_all = a->top_p_all;
  p.min_p_all = a->min_p_all;
  p.vocab = a->vocab;
  // every sum stays below 2^62, and a weight is at most 2^46
  int bits = 62;
  for (long long n = 1; n < a->vocab; n *= 2) --bits;
  p.weight_bits = bits < 46 ? bits : 46;
  ek::DeviceGuard g(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->logits_f32 ? launch<float>(p, a->batch, st) : launch<__nv_bfloat16>(p, a->batch, st);
  return e == cudaSuccess ? EK_SUCCESS : ek::cuda_fail(e, "ek_sample launch");
}
