// 8-bit KV cache: rows are quantised as they are written and read back as bf16.
//
// Per (token, KV head), with D values x: s = bf16_up(max|x| / 127), at least
// 2^-126; code = round_half_away(x / s); value = code * s. Rounding s up keeps
// |x| / s <= 127. s has 8 significant bits, as x has, so x / s is either
// exactly half an integer or at least 1/1020 away from one: 2|x| = (2k + 1) s
// compares two integers below 2^9 * 2^8 over a common exponent. Adding 2^-12
// to |x| * (1 / s) (fp32, error below 2^-14) and rounding to nearest therefore
// gives the exact half-away-from-zero code without a division per element.
//
// Bound: bytes (2 B in and 1 B out per element for a write, the reverse for a
// read, plus 2 B of scale per head). A thread moves 16 elements (two 16-byte
// loads, one 16-byte store) of each of two heads, loaded together, so 4 (D =
// 64) or 8 (D = 128) lanes share a head and one maximum needs 2 or 3 shuffles.
// 32001 rows of 8 heads of 128: written in 38 us (5.2 TB/s), read in 31 (6.4);
// 65536 rows read in 63 us (6.5 TB/s). One head at a time, with conversions of
// each code, took 54, 34 and 69 us.
#include <cuda_bf16.h>

#include "ek_host.h"

namespace {

struct CopyParams {
  EkKvTensor values[2], cache[2];  // K, V
  const int32_t* start;
  long long start_all;
  int length, capacity, heads;
};

constexpr int kThreads = 256;
constexpr int kUnroll = 2;

// Heads of one sequence: blockIdx.x over (row, head), kUnroll * kThreads / LANES of them, blockIdx.y the sequence,
// blockIdx.z K or V.
template <int D, bool WRITE>
__global__ void __launch_bounds__(kThreads) kv_copy(const CopyParams p) {
  constexpr int LANES = D / 16, PER_BLOCK = kThreads / LANES;
  const int b = blockIdx.y, kv = blockIdx.z, lane = threadIdx.x % LANES;
  const EkKvTensor& x = p.values[kv];
  const EkKvTensor& c = p.cache[kv];
  const long long start = p.start ? (long long)p.start[b] : p.start_all;
  __nv_bfloat16* value[kUnroll];
  int8_t* code[kUnroll];
  __nv_bfloat16* scale[kUnroll];
  bool live[kUnroll], inside[kUnroll];
  uint4 lo[kUnroll], hi[kUnroll];
  float s[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const unsigned at = (blockIdx.x * kUnroll + u) * PER_BLOCK + threadIdx.x / LANES;
    live[u] = at < (unsigned)p.length * (unsigned)p.heads;
    const unsigned i = at / (unsigned)p.heads, h = at - i * (unsigned)p.heads;
    const long long row = start + i;
    inside[u] = live[u] && row >= 0 && row < p.capacity;
    value[u] = static_cast<__nv_bfloat16*>(x.data) + b * x.stride_batch + i * x.stride_row + h * x.stride_head + lane * 16;
    code[u] = static_cast<int8_t*>(c.data) + b * c.stride_batch + row * c.stride_row + h * c.stride_head + lane * 16;
    scale[u] = static_cast<__nv_bfloat16*>(c.scales) + b * c.scale_stride_batch + row * c.scale_stride_row +
               h * c.scale_stride_head;
    lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
    s[u] = 0.f;
    if (!inside[u]) continue;
    if (WRITE) {
      lo[u] = __ldg(reinterpret_cast<const uint4*>(value[u]));
      hi[u] = __ldg(reinterpret_cast<const uint4*>(value[u]) + 1);
    } else {
      lo[u] = __ldg(reinterpret_cast<const uint4*>(code[u]));
      s[u] = __bfloat162float(*scale[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    uint32_t w[8] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w};
    if (WRITE) {
      // |x| as integers: NaN > inf > finite
      unsigned tops = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) tops = __vmaxu2(tops, w[j] & 0x7fff7fffu);
      unsigned top = max(tops << 16, tops & 0xffff0000u);
#pragma unroll
      for (int m = LANES / 2; m; m >>= 1) top = max(top, __shfl_xor_sync(~0u, top, m));
      const bool finite = top < 0x7f800000u;
      // top / 127 has 8 significant bits or is 1 / (127 * 256) away from all such numbers: a factor of 1 - 2^-20 puts the
      // product just below the first kind and changes nothing for the second
      unsigned t = (__float_as_uint(__uint_as_float(top) * (float)((1.0 - 0x1p-20) / 127.0)) + 0xffffu) & 0xffff0000u;
      t = finite ? max(t, 0x00800000u) : 0x7fff0000u;
      const float inv = __fdividef(1.f, __uint_as_float(t));  // t is 2^-126 .. 2^121
      const uint32_t keep = finite ? ~0u : 0u;  // codes of a head that reads back as NaN are 0
      if (!inside[u]) continue;
      // x / s moved 2^-12 away from zero, then to the nearest whole number by an addition of 1.5 * 2^23: the low byte
      uint32_t out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t pair = w[2 * j + e / 2];
          const uint32_t v = e & 1 ? pair & 0xffff0000u : pair << 16;
          const float away = __uint_as_float((v & 0x80000000u) | 0x39800000u);
          z[e] = __float_as_uint(fmaf(__uint_as_float(v), inv, away) + 12582912.f);
        }
        out[j] = __byte_perm(__byte_perm(z[0], z[1], 0x0040), __byte_perm(z[2], z[3], 0x0040), 0x5410) & keep;
      }
      *reinterpret_cast<uint4*>(code[u]) = make_uint4(out[0], out[1], out[2], out[3]);
      if (lane == 0) *scale[u] = __ushort_as_bfloat16((unsigned short)(t >> 16));
    } else if (live[u]) {
      uint32_t out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t v = w[j / 2] >> (16 * (j & 1));
        const __nv_bfloat162 r =
            __floats2bfloat162_rn((float)(int8_t)(v & 0xff) * s[u], (float)(int8_t)(v >> 8 & 0xff) * s[u]);
        out[j] = *reinterpret_cast<const uint32_t*>(&r);
      }
      reinterpret_cast<uint4*>(value[u])[0] = make_uint4(out[0], out[1], out[2], out[3]);
      reinterpret_cast<uint4*>(value[u])[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
  }
}

bool strides16(const EkKvTensor& t, int elements) {
  return t.stride_batch % elements == 0 && t.stride_row % elements == 0 && t.stride_head % elements == 0;
}

int copy(const EkKvCopyArgs* a, void* stream, bool write) {
  using ek::fail;
  if (!a) return fail(EK_E_INVALID, "NULL arguments");
  if (a->batch < 0 || a->length < 0 || a->capacity < 0 || a->kv_heads < 1)
    return fail(EK_E_INVALID, "bad sizes batch=%d length=%d capacity=%d kv_heads=%d", a->batch, a->length,
                a->capacity, a->kv_heads);
  if (a->head_dim != 64 && a->head_dim != 128)
    return fail(EK_E_UNSUPPORTED, "head_dim %d (supported: 64, 128)", a->head_dim);
  if (a->batch == 0 || a->length == 0) return EK_SUCCESS;
  if (a->batch > 65535) return fail(EK_E_UNSUPPORTED, "batch %d (at most 65535)", a->batch);
  const EkKvTensor* values[2] = {&a->k_values, &a->v_values};
  const EkKvTensor* cache[2] = {&a->k_cache, &a->v_cache};
  CopyParams p;
  for (int i = 0; i < 2; ++i) {
    if (!values[i]->data || !ek::aligned16(values[i]->data) || !strides16(*values[i], 8))
      return fail(EK_E_INVALID, "bf16 rows must be 16-byte aligned with strides of 16 bytes");
    if (a->capacity > 0 && (!cache[i]->data || !cache[i]->scales || !ek::aligned16(cache[i]->data) ||
                            !strides16(*cache[i], 16)))
      return fail(EK_E_INVALID, "cache codes must be 16-byte aligned with strides of 16 bytes, with scales");
    p.values[i] = *values[i];
    p.cache[i] = *cache[i];
  }
  p.start = a->start;
  p.start_all = a->start_all;
  p.length = a->length;
  p.capacity = a->capacity;
  p.heads = a->kv_heads;
  const int per_block = kUnroll * kThreads / (a->head_dim / 16);
  const long long blocks = ((long long)a->length * a->kv_heads + per_block - 1) / per_block;
  if ((long long)a->length * a->kv_heads > 0x7fffffffll) return fail(EK_E_UNSUPPORTED, "length * kv_heads beyond 2^31");
  ek::DeviceGuard g(a->device);
  const dim3 grid((unsigned)blocks, a->batch, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->head_dim == 64) {
    if (write) kv_copy<64, true><<<grid, kThreads, 0, st>>>(p);
    else kv_copy<64, false><<<grid, kThreads, 0, st>>>(p);
  } else {
    if (write) kv_copy<128, true><<<grid, kThreads, 0, st>>>(p);
    else kv_copy<128, false><<<grid, kThreads, 0, st>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? EK_SUCCESS : ek::cuda_fail(e, write ? "ek_kv_write launch" : "ek_kv_read launch");
}

}  // namespace

extern "C" int ek_kv_write(const EkKvCopyArgs* a, void* stream) { return copy(a, stream, true); }
extern "C" int ek_kv_read(const EkKvCopyArgs* a, void* stream) { return copy(a, stream, false); }
