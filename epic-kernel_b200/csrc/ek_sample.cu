// Token sampling: temperature, top-k, top-p and min-p, then one draw per row.
//
// All filters keep a prefix of the order (logit descending, index ascending),
// so a cut is a pair: the key of the last kept logit, and how many of its ties
// stay. top-k counts tokens and top-p adds weights over the same search: a
// histogram of 512 bins over the logits' range, then histograms over the
// order-preserving integer keys of the bin that holds the cut, until a bin is
// one value (two or three passes).
//
// Weights are exp((l - max) / T) in double, rounded to fixed point (at least
// 43 bits below the largest), so every sum is exact, in any order of the
// atomics, and a launch repeats bit for bit. Single precision would not do: a
// flat row has 10^5 borders that are 10^-5 apart, and each border's error
// moves some tokens.
//
// A row is spread over a cluster of 1 to 8 blocks that hold it in shared
// memory, so it is read from HBM once; the blocks exchange maxima, histograms
// and sums through distributed shared memory. Bound: the bytes of the logits
// for large batches with few kept tokens, else the weights (about 14 double
// operations each); for one row, the latency of the load and of two cluster
// barriers per pass.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "ek_host.h"

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = kThreads;
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 49152;  // elements per block: 192 KB of fp32; a bin's 16-bit limbs add up below 2^32
using u64 = unsigned long long;

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
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

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
struct Weight {
  float top;
  double top_d, c;     // c = 32 log2(e) / T
  const double* table; // 2^(j / 32), shared memory
  int bits;

  __device__ __forceinline__ u64 operator()(float l) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52
    const double x = ((double)l - top_d) * c;
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
    return l == top ? 1ull << bits : (u64)__double_as_longlong(whole) & 0xfffffffffffffull;
  }
};

struct Shared {
  unsigned hist[2][3][kBins];  // counts, or the three 16-bit limbs of weights
  double table[32];
  u64 scan[kWarps];
  float top[kMaxCluster], low[kMaxCluster];  // maxima and minima of the blocks
  u64 warp_weight[kMaxCluster * kWarps];     // per warp of the cluster: weight above the cut, ties
  unsigned warp_ties[kMaxCluster * kWarps];
  u64 found_before;
  int found_bin;
  int first[kMaxCluster];
};

// Inclusive scan over the block's threads.
__device__ u64 block_scan(u64 v, Shared& sh) {
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

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_rows(const SampleParams p) {
  using V16 = Vec<T>;
  constexpr int N = V16::N;
  extern __shared__ uint4 dynamic[];
  T* slice = reinterpret_cast<T*>(dynamic);
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int first = min(p.vocab, rank * p.slice), count = min(p.vocab - first, p.slice);
  const T* row = static_cast<const T*>(p.logits) + b * p.row_stride + first;
  auto sync = [&] {
    if (C > 1) cluster.sync();
    else __syncthreads();
  };
  if (C > 1) cluster.barrier_arrive();  // peers' shared memory may be written once all have started
  auto peer = [&](auto* at, int r) { return C > 1 ? cluster.map_shared_rank(at, r) : at; };

  // ---- load the slice (NaN as -inf, padded with -inf), maximum and minimum
  const float inf = INFINITY;
  float top = -inf, low = inf;
  auto clean = [&](T x) {
    const float l = as_float(x);
    if (l > -inf) top = fmaxf(top, l), low = fminf(low, l);
    return l == l ? x : (T)-inf;
  };
  const int padded = (count + N - 1) / N * N, vectors = padded / N;
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {
    const int whole = count / N;
    constexpr int U = 4;
    for (int i = tid; i < whole; i += U * kThreads) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < whole) w[u] = __ldg(reinterpret_cast<const uint4*>(row) + i + u * kThreads);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < whole) {
          V16 v = *reinterpret_cast<V16*>(&w[u]);
#pragma unroll
          for (int e = 0; e < N; ++e) v.x[e] = clean(v.x[e]);
          reinterpret_cast<uint4*>(slice)[i + u * kThreads] = *reinterpret_cast<uint4*>(&v);
        }
    }
    for (int i = whole * N + tid; i < padded; i += kThreads) slice[i] = i < count ? clean(row[i]) : (T)-inf;
  } else {
    constexpr int U = 8;
    for (int i = tid; i < padded; i += U * kThreads) {
      T w[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < count) w[u] = row[i + u * kThreads];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u * kThreads < padded)
          slice[i + u * kThreads] = i + u * kThreads < count ? clean(w[u]) : (T)-inf;
    }
  }
  if (tid < 32) sh.table[tid] = exp2((double)tid / 32.0);
  for (int i = tid; i < 3 * kBins; i += kThreads) sh.hist[0][0][i] = 0;
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
    low = fminf(low, __shfl_xor_sync(~0u, low, m));
  }
  {
    float* wt = reinterpret_cast<float*>(sh.scan);
    if (lane == 0) wt[2 * warp] = top, wt[2 * warp + 1] = low;
    __syncthreads();
    if (warp == 0) {
      top = lane < kWarps ? wt[2 * lane] : -inf, low = lane < kWarps ? wt[2 * lane + 1] : inf;
#pragma unroll
      for (int m = 16; m; m >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(~0u, top, m));
        low = fminf(low, __shfl_xor_sync(~0u, low, m));
      }
    }
    if (C > 1) cluster.barrier_wait();
    if (warp == 0) {
      if (lane < C) *peer(&sh.top[rank], lane) = top, *peer(&sh.low[rank], lane) = low;
    }
  }
  sync();
  top = sh.top[0], low = sh.low[0];
  for (int r = 1; r < C; ++r) top = fmaxf(top, sh.top[r]), low = fminf(low, sh.low[r]);

  const float temp = p.temperature ? p.temperature[b] : p.temperature_all;
  if (!(temp > 0.f) || top == -inf) {  // the first of the largest; nothing above -inf gives 0
    int at = 0x7fffffff;
    if (top > -inf)
      for (int i = tid; i < count; i += kThreads)
        if (as_float(slice[i]) == top) {
          at = first + i;
          break;
        }
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
  const int k = p.top_k ? p.top_k[b] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[b] : p.min_p_all;
  const Weight weight{top, (double)top, 46.166241308446828 / (double)temp, sh.table, p.weight_bits};
  // below `low` a weight rounds to 0 and the token can never be drawn
  low = fmaxf(low, __double2float_ru((double)top - (double)temp * (0.6931471805599453 * (p.weight_bits + 1))));

  // ---- cuts: keys above `cut` stay, and the first `ties` (by index) of those equal to it
  unsigned cut = key_of<T>(low);
  u64 ties = ~0ull;
  if (min_p > 0.f) {
    const double lowest = (double)top + (double)temp * log((double)fminf(min_p, 1.f));
    float l = __double2float_ru(lowest);
    if (sizeof(T) == 2) {  // the next bf16 at or above
      const __nv_bfloat16 up = __float2bfloat16_ru(l);
      l = __bfloat162float(up);
    }
    cut = max(cut, key_of<T>(fminf(l, top)));
  }
  unsigned k_cut = 0;  // top-k keeps keys above, and k_ties equal ones
  u64 k_ties = 0;
  int buffer = 0;
  const float bins_per = top > low && top < inf ? (float)kBins / (top - low) : 0.f;
  auto bin_of = [&](float l) { return min((int)((top - l) * bins_per), kBins - 1); };
  for (int stage = 0; stage < 2; ++stage) {  // 0: top-k; 1: top-p among what top-k left
    if (stage == 0 ? (k <= 0 || k >= p.vocab) : !(top_p < 1.f)) continue;
    u64 goal = stage == 0 ? (u64)k : 0, before = 0;
    unsigned high = 0, base = 0;  // keys still in question
    int bin1 = -1, shift = 0;
    bool all = false;
    for (;;) {
      auto& hist = sh.hist[buffer];
      for (int i = tid; i < vectors; i += kThreads) {
        const uint4 raw = reinterpret_cast<const uint4*>(slice)[i];
        const V16 v = *reinterpret_cast<const V16*>(&raw);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float l = as_float(v.x[e]);
          if (!(l >= low)) continue;
          int bin = bin_of(l);
          if (bin1 >= 0 && bin != bin1) continue;
          const unsigned key = key_of<T>(l);
          if (stage == 1 && key <= k_cut) continue;
          if (bin1 >= 0) {
            if (key > high || key < base) continue;
            bin = (int)((high - key) >> shift);
          }
          if (stage == 0) {
            atomicAdd(&hist[0][bin], 1u);
          } else {
            const u64 w = weight(l);
            atomicAdd(&hist[0][bin], (unsigned)w & 0xffffu);
            atomicAdd(&hist[1][bin], (unsigned)(w >> 16) & 0xffffu);
            atomicAdd(&hist[2][bin], (unsigned)(w >> 32));
          }
        }
      }
      sync();
      // every block adds up all blocks' bins, one per thread
      u64 mine = 0;
      for (int r = 0; r < C; ++r) {
        const unsigned* other = peer(&hist[0][0], r);
        mine += other[tid];
        if (stage == 1) mine += (u64)other[kBins + tid] * 65536ull + ((u64)other[2 * kBins + tid] << 32);
      }
      // the other buffer is free: its last readers were past it before this barrier
      buffer ^= 1;
      for (int i = tid; i < 3 * kBins; i += kThreads) sh.hist[buffer][0][i] = 0;
      const u64 sum = before + block_scan(mine, sh);
      if (tid == kThreads - 1) sh.found_bin = kBins, sh.found_before = sum;
      __syncthreads();
      if (bin1 < 0) {
        const u64 total = sh.found_before;
        if (stage == 1) {
          const u64 tied = k_ties ? k_ties * weight(value_of<T>(k_cut)) : 0;
          goal = (u64)ceil((double)fmaxf(top_p, 0.f) * (double)(total + tied));
          goal = goal < 1 ? 1 : goal;  // the first token always stays
        }
        all = total < goal;  // the cut lies below all of these
      }
      __syncthreads();
      if (all) break;
      if (sum >= goal && sum - mine < goal) sh.found_bin = tid, sh.found_before = sum - mine;
      __syncthreads();
      const int found = sh.found_bin;
      before = sh.found_before;
      if (bin1 < 0) {
        // bounds of the bin, widened by the rounding of bin_of; bin1 itself stays the filter
        bin1 = found;
        high = key_of<T>(top), base = key_of<T>(low);
        if (bins_per > 0.f) {
          const float margin = (top - low) * 0x1p-18f + fmaxf(fabsf(top), fabsf(low)) * 0x1p-20f;
          const float hi = top - (float)found / bins_per + margin, lo = top - (float)(found + 1) / bins_per - margin;
          if (hi < top) high = key_of<T>(hi);
          if (lo > low && found < kBins - 1) base = key_of<T>(lo);
        }
      } else {
        high -= (unsigned)found << shift;
        if (shift == 0) break;
        base = max(base, high - ((1u << shift) - 1u));
      }
      const unsigned span = high - base;  // bins of 2^shift keys
      shift = span < kBins ? 0 : 32 - __clz(span) - 9;
    }
    __syncthreads();
    if (all && stage == 0) continue;
    const unsigned key = all ? k_cut : high;
    if (all) before = sh.found_before;
    const u64 unit = stage == 0 ? 1 : weight(value_of<T>(key));
    u64 r = (goal - before + unit - 1) / unit;
    if (stage == 0) k_cut = key, k_ties = r;
    else if (all) r = min(r, k_ties);
    if (key > cut) cut = key, ties = r;
    else if (key == cut) ties = min(ties, r);
  }

  // ---- the draw: a warp owns a contiguous range, so that sums run by index
  const int per_warp = (vectors + kWarps - 1) / kWarps;
  const int v0 = min(vectors, warp * per_warp), v1 = min(vectors, v0 + per_warp);
  const float cut_value = value_of<T>(cut);
  u64 above = 0;
  unsigned tied = 0;
  for (int i = v0 + lane; i < v1; i += 32) {
    const uint4 raw = reinterpret_cast<const uint4*>(slice)[i];
    const V16 v = *reinterpret_cast<const V16*>(&raw);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float l = as_float(v.x[e]);
      if (l > cut_value) above += weight(l);
      else if (l == cut_value) ++tied;
    }
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
  constexpr int E = kMaxCluster * kWarps / 32;
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
  const u64 total = __shfl_sync(~0u, upto, 31);
  const float u = p.uniforms[b];
  u64 goal = (u64)((double)(u > 0.f ? fminf(u, 1.f) : 0.f) * (double)total);
  goal = min(goal, total - 1);
  u64 running = upto - weights;
  int owner = -1;
  u64 owner_before = 0, owner_ties = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (owner < 0 && running <= goal && goal < running + w[e]) owner = lane * E + e, owner_before = running, owner_ties = ahead[e];
    running += w[e];
  }
  const unsigned who = __ballot_sync(~0u, owner >= 0);
  const int from = __ffs(who) - 1;
  owner = __shfl_sync(~0u, owner, from);
  if (owner == rank * kWarps + warp) {
    u64 sum = __shfl_sync(~0u, owner_before, from), seen = __shfl_sync(~0u, owner_ties, from);
    for (int i0 = v0; i0 < v1; i0 += 32) {
      const int i = i0 + lane;
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (i < v1) raw = reinterpret_cast<const uint4*>(slice)[i];
      const V16 v = *reinterpret_cast<const V16*>(&raw);
      unsigned mine = 0;
      u64 heavy = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float l = as_float(v.x[e]);
        if (i < v1 && l == cut_value) ++mine;
        if (i < v1 && l > cut_value) heavy += weight(l);
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
          if (l > cut_value) at += weight(l);
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

template <typename T>
cudaError_t launch(const SampleParams& p, int batch, int cluster, cudaStream_t st) {
  const int bytes = p.slice * (int)sizeof(T);
  cudaError_t e = cudaFuncSetAttribute(sample_rows<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kMaxSlice * (int)sizeof(T));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)batch * cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_rows<T>, p);
}

}  // namespace

extern "C" int ek_sample(const EkSampleArgs* a, void* stream) {
  using ek::fail;
  if (!a) return fail(EK_E_INVALID, "NULL arguments");
  if (a->batch < 0 || a->vocab < 1) return fail(EK_E_INVALID, "bad sizes batch=%d vocab=%d", a->batch, a->vocab);
  const int size = a->logits_f32 ? 4 : 2;
  if (a->vocab > kMaxCluster * kMaxSlice)
    return fail(EK_E_UNSUPPORTED, "vocab %d (at most %d)", a->vocab, kMaxCluster * kMaxSlice);
  if (a->batch > (1 << 27)) return fail(EK_E_UNSUPPORTED, "batch %d", a->batch);
  if (a->batch == 0) return EK_SUCCESS;
  if (!a->logits || !a->uniforms || !a->tokens) return fail(EK_E_INVALID, "NULL pointer argument");
  SampleParams p;
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
  // every sum stays below 2^62, and a weight below 2^48 (three limbs)
  int bits = 62;
  for (long long n = 1; n < a->vocab; n *= 2) --bits;
  p.weight_bits = bits < 46 ? bits : 46;
  // Blocks per row: as many as keep 2048 elements each, up to 8, so that a few rows use the whole cluster's
  // bandwidth; with many rows, only as many as hold the row in 64 KB each (three blocks fit an SM).
  int cluster = 1;
  while (cluster < kMaxCluster &&
         ((long long)a->vocab * size > cluster * 65536ll ||
          (a->vocab >= cluster * 4096 && (long long)a->batch * cluster < 296)))
    cluster *= 2;
  p.slice = (int)(((long long)a->vocab + cluster - 1) / cluster + 15) / 16 * 16;
  ek::DeviceGuard g(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->logits_f32 ? launch<float>(p, a->batch, cluster, st)
                                      : launch<__nv_bfloat16>(p, a->batch, cluster, st);
  return e == cudaSuccess ? EK_SUCCESS : ek::cuda_fail(e, "ek_sample launch");
}
