// Token sampling: temperature, top-k, top-p and min-p, then one draw per row.
//
// All filters keep a prefix of the order (logit descending, index ascending),
// so a cut is a pair (key of the last kept logit, number of its ties that
// stay). Both cuts come from a radix selection over order-preserving 32-bit
// keys: top-k counts tokens, top-p adds weights. Weights are exp((l - max)/T)
// in double, rounded to fixed point, so their sums are exact, independent of
// the order of the atomics, and the same in every launch; a token differs from
// the one that real arithmetic picks only if the uniform falls within about
// 1e-11 of a border.
#include <cuda_bf16.h>

#include "ek_host.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
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
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Order-preserving key; -0 counts as +0 and NaN as -inf.
__device__ __forceinline__ unsigned key_of(float l) {
  unsigned u = __float_as_uint(l != l ? -INFINITY : l + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

struct Weight {
  double top, inv_t, one;
  // Fixed-point weight of logit `l`, 0 for -inf.
  __device__ u64 operator()(float l) const {
    if (l == (float)top) return (u64)one;
    const double t = ((double)l - top) * inv_t;
    return t > -745. ? (u64)__double2ull_rn(exp(t) * one) : 0;
  }
};

__device__ u64 block_sum(u64 v, u64* scratch) {
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(~0u, v, m);
  __syncthreads();
  if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
  __syncthreads();
  v = scratch[threadIdx.x % 32];
#pragma unroll
  for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(~0u, v, m);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_rows(const SampleParams p) {
  __shared__ u64 scratch[kWarps];
  __shared__ u64 hist[256];
  __shared__ unsigned s_prefix;
  __shared__ u64 s_before, s_goal;
  __shared__ int s_pick;
  const int b = blockIdx.x, V = p.vocab, tid = threadIdx.x;
  const T* row = static_cast<const T*>(p.logits) + b * p.row_stride;
  const float temp = p.temperature ? p.temperature[b] : p.temperature_all;
  const int k = p.top_k ? p.top_k[b] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[b] : p.min_p_all;

  // the largest key and its first index
  u64 best = 0;
  for (int i = tid; i < V; i += kThreads) {
    const u64 c = (u64)key_of(as_float(row[i])) << 32 | (0xffffffffu - (unsigned)i);
    best = c > best ? c : best;
  }
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const u64 o = __shfl_xor_sync(~0u, best, m);
    best = o > best ? o : best;
  }
  if (tid % 32 == 0) scratch[tid / 32] = best;
  __syncthreads();
  best = scratch[tid % 32];
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    const u64 o = __shfl_xor_sync(~0u, best, m);
    best = o > best ? o : best;
  }
  const float top = value_of((unsigned)(best >> 32));
  const int top_at = (int)(0xffffffffu - (unsigned)best);
  if (!(temp > 0.f) || top == -INFINITY) {
    if (tid == 0) p.tokens[b] = top_at;
    return;
  }
  const Weight weight{(double)top, 1.0 / (double)temp, (double)(1ull << p.weight_bits)};

  // cut: keys above `cut` stay, and the first `ties` (by index) of those equal to it
  const unsigned lowest = key_of(-INFINITY) + 1;  // -inf never stays
  unsigned cut = lowest, k_cut = lowest;
  long long ties = V, k_ties = V;
  if (min_p > 0.f) {
    const double low = (double)top + (double)temp * log((double)fminf(min_p, 1.f));
    cut = max(cut, key_of(__double2float_ru(low)));
  }
  for (int stage = 0; stage < 2; ++stage) {  // 0: top-k; 1: top-p among what top-k left
    if (stage == 0 ? (k <= 0 || k >= V) : !(top_p < 1.f)) continue;
    u64 goal = k;
    if (stage == 1) {
      u64 above = 0, equal = 0;
      for (int i = tid; i < V; i += kThreads) {
        const float l = as_float(row[i]);
        const unsigned key = key_of(l);
        if (key > k_cut) above += weight(l);
        else if (key == k_cut) ++equal;
      }
      equal = block_sum(equal, scratch);
      const u64 total = block_sum(above, scratch) + weight(value_of(k_cut)) * min(equal, (u64)k_ties);
      goal = (u64)ceil((double)fmaxf(top_p, 0.f) * (double)total);
      goal = goal < 1 ? 1 : goal;  // the first token always stays
    }
    unsigned prefix = 0;
    u64 before = 0;  // tokens (weight) above the digit range under search
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
      __syncthreads();
      const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
      for (int i = tid; i < V; i += kThreads) {
        const float l = as_float(row[i]);
        const unsigned key = key_of(l);
        if (key >= k_cut && (key & mask) == prefix) atomicAdd(&hist[key >> shift & 255], stage == 0 ? 1ull : weight(l));
      }
      __syncthreads();
      if (tid == 0) {
        u64 sum = before;
        int d = 255;
        while (d > 0 && sum + hist[d] < goal) sum += hist[d--];
        s_prefix = prefix | (unsigned)d << shift;
        s_before = sum;
      }
      __syncthreads();
      prefix = s_prefix;
      before = s_before;
    }
    if (prefix < lowest) continue;  // top-k with fewer than k tokens above -inf: all stay
    const u64 unit = stage == 0 ? 1 : weight(value_of(prefix));
    long long r = (long long)((goal - before + unit - 1) / unit);
    if (stage == 0) k_cut = prefix, k_ties = r;
    else if (prefix == k_cut) r = min(r, k_ties);
    if (prefix > cut) cut = prefix, ties = r;
    else if (prefix == cut) ties = min(ties, r);
  }

  // running weights by index: a thread owns a contiguous range
  const int per = (V + kThreads - 1) / kThreads;
  const int lo = min(V, tid * per), hi = min(V, lo + per);
  u64 equal = 0;
  for (int i = lo; i < hi; ++i) equal += key_of(as_float(row[i])) == cut;
  // exclusive scans over threads (ties first, then weights)
  static __shared__ u64 scan[kThreads];
  auto exclusive = [&](u64 v) {
    __syncthreads();
    scan[tid] = v;
    __syncthreads();
    for (int m = 1; m < kThreads; m <<= 1) {
      const u64 o = tid >= m ? scan[tid - m] : 0;
      __syncthreads();
      scan[tid] += o;
      __syncthreads();
    }
    return scan[tid] - v;
  };
  const u64 tie0 = exclusive(equal);
  u64 mine = 0, t = tie0;
  for (int i = lo; i < hi; ++i) {
    const float l = as_float(row[i]);
    const unsigned key = key_of(l);
    if (key > cut || (key == cut && (long long)t++ < ties)) mine += weight(l);
  }
  const u64 w0 = exclusive(mine);
  if (tid == kThreads - 1) {
    const u64 total = w0 + mine;
    const float u = p.uniforms[b];
    u64 goal = (u64)((double)(u > 0.f ? u : 0.f) * (double)total);
    s_goal = goal < total ? goal : total - 1;
    s_pick = top_at;
  }
  __syncthreads();
  const u64 goal = s_goal;
  if (w0 <= goal && goal < w0 + mine) {
    u64 sum = w0;
    t = tie0;
    for (int i = lo; i < hi; ++i) {
      const float l = as_float(row[i]);
      const unsigned key = key_of(l);
      if (key > cut || (key == cut && (long long)t++ < ties)) sum += weight(l);
      if (sum > goal) {
        s_pick = i;
        break;
      }
    }
  }
  __syncthreads();
  if (tid == 0) p.tokens[b] = s_pick;
}

}  // namespace

extern "C" int ek_sample(const EkSampleArgs* a, void* stream) {
  using ek::fail;
  if (!a) return fail(EK_E_INVALID, "NULL arguments");
  if (a->batch < 0 || a->vocab < 1) return fail(EK_E_INVALID, "bad sizes batch=%d vocab=%d", a->batch, a->vocab);
  if (a->batch == 0) return EK_SUCCESS;
  if (a->vocab > (1 << 22)) return fail(EK_E_UNSUPPORTED, "vocab %d (at most %d)", a->vocab, 1 << 22);
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
  // every sum stays below 2^63
  int bits = 62;
  for (int n = 1; n < a->vocab; n *= 2) --bits;
  p.weight_bits = bits < 46 ? bits : 46;
  ek::DeviceGuard g(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->logits_f32) sample_rows<float><<<a->batch, kThreads, 0, st>>>(p);
  else sample_rows<__nv_bfloat16><<<a->batch, kThreads, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? EK_SUCCESS : ek::cuda_fail(e, "ek_sample launch");
}
