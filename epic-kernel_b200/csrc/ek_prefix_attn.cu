// Decode attention of B sequences over a shared prefix plus their own rows.
//
//   o_b = softmax(scale * q_b [Kp; Ko_b]^T) [Vp; Vo_b]
//
// The prefix rows are the same for all sequences, so one KV head's rows serve
// batch * group query rows at once and are read once instead of `batch` times.
// The softmax is split over the keys: every work item (a KV head, a set of
// query rows and a range of keys) keeps a running maximum m, sum l and
// unnormalised output o in fp32 over one pass, writes (o, m, l) to the
// workspace, and a second kernel joins the items of a row.
//
// `few_rows` computes an item for up to 8 query rows with mma.m16n8k16 on the
// transposed products, S^T = K Q^T and O^T = V^T P^T, so that the 16-row side
// of the instruction carries keys (or dimensions) and the 8-row side the query
// rows. K and V go from global memory to fragment registers with 16-byte
// loads: the contraction order over d is free, so lane c of a quad takes 8
// (bf16) or 16 (int8) consecutive dimensions and q is laid out to match. P^T
// becomes a B fragment by one 8x8 transpose in registers. 8-bit codes are
// exact in bf16; K's scale multiplies the score and V's scale the probability.
// Bound: bytes (4 flops per byte and query row).
#include <cuda_bf16.h>

#include "ek_host.h"

namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

struct Store {
  const char* k;
  const char* v;
  const __nv_bfloat16* ks;
  const __nv_bfloat16* vs;
  long long k_batch, k_row, k_head, v_batch, v_row, v_head;  // bytes
  long long ks_batch, ks_row, ks_head, vs_batch, vs_row, vs_head;  // elements
};

struct AttnParams {
  Store prefix, own;
  const __nv_bfloat16* q;
  long long q_batch, q_head;
  __nv_bfloat16* out;
  long long out_batch, out_head;
  float* lse;
  const int32_t* own_lens;
  float* part_o;   // [slots][batch * q_heads][D]
  float2* part_ml; // [slots][batch * q_heads]: running maximum (base 2), sum
  int batch, q_heads, kv_heads, group;
  int prefix_len, max_own;
  int prefix_chunk, own_chunk;    // keys per item
  int prefix_slots, own_slots;    // items per row
  int prefix_tiles, group_tiles;  // tiles of 8 rows: of batch * group, of group
  float scale_log2;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Two int8 codes in the low bytes of the halves of x, as a bf16 pair: 128 + (c & 127)
// minus 128 (c >= 0) or 256 (c < 0), all exact.
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t x) {
  const uint32_t v = (x & 0x007f007fu) | 0x43004300u, bias = (x & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                   *reinterpret_cast<const __nv_bfloat162*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The fragments of 16 keys of one KV head.
template <int D, bool I8>
struct Rows {
  // K: keys lane/4 and lane/4 + 8, dimensions by quad lane; V: keys 2c, 2c+1, 2c+8, 2c+9 of quad lane c,
  // dimensions by lane/4
  static constexpr int KV = I8 ? D / 64 : D / 32;  // 16-byte pieces of a key per quad lane
  static constexpr int VW = I8 ? D / 32 : D / 16;  // 4-byte words of a key per lane/4
  uint4 k[2][KV];
  uint32_t v[4][VW];
  float ks[2], vs[2][2];
};

template <int D, bool I8>
__device__ __forceinline__ void load_rows(Rows<D, I8>& r, const Store& s, long long b, int head, int t0, int t1) {
  const int lane = threadIdx.x % 32, c = lane % 4, j = lane / 4;
  const char* kb = s.k + b * s.k_batch + head * s.k_head + c * 16;
  const char* vb = s.v + b * s.v_batch + head * s.v_head;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = t0 + j + 8 * i;
    const bool in = t < t1;
#pragma unroll
    for (int m = 0; m < r.KV; ++m)
      r.k[i][m] = in ? __ldg(reinterpret_cast<const uint4*>(kb + t * s.k_row + m * 64)) : make_uint4(0, 0, 0, 0);
    if (I8) r.ks[i] = in ? __bfloat162float(s.ks[b * s.ks_batch + t * s.ks_row + head * s.ks_head]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + 2 * c + (i & 1) + (i & 2) * 4;
    const bool in = t < t1;
    const char* at = vb + t * s.v_row;
    if (I8 && D == 64) {
      const uint2 x = in ? __ldg(reinterpret_cast<const uint2*>(at + j * 8)) : make_uint2(0, 0);
      r.v[i][0] = x.x, r.v[i][1] = x.y;
    } else {
#pragma unroll
      for (int m = 0; m < r.VW / 4; ++m) {
        const uint4 x = in ? __ldg(reinterpret_cast<const uint4*>(at + m * 128 + j * 16)) : make_uint4(0, 0, 0, 0);
        r.v[i][4 * m] = x.x, r.v[i][4 * m + 1] = x.y, r.v[i][4 * m + 2] = x.z, r.v[i][4 * m + 3] = x.w;
      }
    }
  }
  if (I8) {
    // scales of keys lane/4 (+8), where P is still laid out by key
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = t0 + j + 8 * i;
      r.vs[i][0] = t < t1 ? __bfloat162float(s.vs[b * s.vs_batch + t * s.vs_row + head * s.vs_head]) : 0.f;
    }
  }
}

// Dimension of element ee (0 .. D/8 - 1) that lane/4 = j holds of V.
template <int D, bool I8>
__device__ __forceinline__ int v_dim(int j, int ee) {
  if (I8) return j * (D / 8) + ee;
  return (ee / 8) * 64 + j * 8 + ee % 8;
}

template <int D, bool I8>
__global__ void __launch_bounds__(kWarps * 32) few_rows(const AttnParams p) {
  constexpr int KT = D / 16;  // 16-wide steps over the dimensions
  __shared__ float s_o[kWarps][8][D];
  __shared__ float s_m[kWarps][8], s_l[kWarps][8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = lane % 4, j = lane / 4;

  // the item
  long long id = blockIdx.x;
  const long long prefix_items = (long long)p.prefix_slots * p.prefix_tiles * p.kv_heads;
  const bool shared = id < prefix_items;
  int head, tile, slot, seq = 0, t0, t1;
  if (shared) {
    head = (int)(id % p.kv_heads), id /= p.kv_heads;
    tile = (int)(id % p.prefix_tiles);
    slot = (int)(id / p.prefix_tiles);
    t0 = slot * p.prefix_chunk;
    t1 = min(p.prefix_len, t0 + p.prefix_chunk);
  } else {
    id -= prefix_items;
    head = (int)(id % p.kv_heads), id /= p.kv_heads;
    tile = (int)(id % p.group_tiles), id /= p.group_tiles;
    seq = (int)(id % p.batch);
    slot = (int)(id / p.batch);
    t0 = slot * p.own_chunk;
    t1 = min(min(max(p.own_lens[seq], 0), p.max_own), t0 + p.own_chunk);
    if (t0 >= t1) return;
  }
  const Store& store = shared ? p.prefix : p.own;
  const int rows = shared ? p.batch * p.group : p.group;
  // row n of the tile -> (sequence, query head)
  auto locate = [&](int n, int& b, int& h) {
    const int r = tile * 8 + n;
    b = shared ? r / p.group : seq;
    h = head * p.group + (shared ? r % p.group : r);
    return r < rows;
  };

  // q of row lane/4 as B fragments: the dimensions that quad lane c holds of K
  uint32_t q[KT][2];
  {
    int b, h;
    const bool in = locate(j, b, h);
    const __nv_bfloat16* at = p.q + b * p.q_batch + h * p.q_head;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int d = I8 ? (kt / 4) * 64 + c * 16 + (kt % 4) * 4 : (kt / 2) * 32 + c * 8 + (kt % 2) * 4;
      const uint2 x = in ? __ldg(reinterpret_cast<const uint2*>(at + d)) : make_uint2(0, 0);
      q[kt][0] = x.x, q[kt][1] = x.y;
    }
  }

  float o[KT][4] = {};  // O^T: dimensions v_dim(j, 2 kt), v_dim(j, 2 kt + 1) of rows 2c, 2c + 1
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  for (int t = t0 + warp * 16; t < t1; t += kWarps * 16) {
    Rows<D, I8> r;
    load_rows<D, I8>(r, store, seq, head, t, t1);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (I8) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint32_t w0 = reinterpret_cast<const uint32_t*>(&r.k[0][kt / 4])[kt % 4];
        const uint32_t w1 = reinterpret_cast<const uint32_t*>(&r.k[1][kt / 4])[kt % 4];
        mma_16x8x16(s, codes_to_bf16(__byte_perm(w0, w0, 0x1100)), codes_to_bf16(__byte_perm(w1, w1, 0x1100)),
                    codes_to_bf16(__byte_perm(w0, w0, 0x3322)), codes_to_bf16(__byte_perm(w1, w1, 0x3322)), q[kt][0],
                    q[kt][1]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] *= r.ks[i / 2];
    } else {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&r.k[0][kt / 2]) + (kt % 2) * 2;
        const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&r.k[1][kt / 2]) + (kt % 2) * 2;
        mma_16x8x16(s, w0[0], w1[0], w0[1], w1[1], q[kt][0], q[kt][1]);
      }
    }
    // s[0], s[1]: key t + j of rows 2c, 2c + 1; s[2], s[3]: key t + j + 8
    float fix[2];
    bool grew = false;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      s[n] = t + j < t1 ? s[n] * p.scale_log2 : -INFINITY;
      s[2 + n] = t + j + 8 < t1 ? s[2 + n] * p.scale_log2 : -INFINITY;
      float top = fmaxf(s[n], s[2 + n]);
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
      const float next = fmaxf(m[n], top);
      const float base = next == -INFINITY ? 0.f : next;
      fix[n] = exp2_approx(m[n] - base);
      grew |= next != m[n];
      m[n] = next;
      s[n] = exp2_approx(s[n] - base);
      s[2 + n] = exp2_approx(s[2 + n] - base);
      l[n] = l[n] * fix[n] + s[n] + s[2 + n];
    }
    if (grew) {
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        o[kt][0] *= fix[0], o[kt][1] *= fix[1];
        o[kt][2] *= fix[0], o[kt][3] *= fix[1];
      }
    }
    if (I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = s[i] == 0.f ? 0.f : s[i] * r.vs[i / 2][0];
    }
    // probabilities are rounded to bf16 for the product: half a step is 2^-8 of each, as for V itself
    const uint32_t b0 = transpose_8x8(pack_bf16(s[0], s[1])), b1 = transpose_8x8(pack_bf16(s[2], s[3]));
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      uint32_t a[4];
      if (I8) {
        const int w = kt / 2, e = (kt % 2) * 2;  // word and first byte of element 2 kt
        const uint32_t even = e == 0 ? 0x4400 : 0x6622, odd = e == 0 ? 0x5511 : 0x7733;
        a[0] = codes_to_bf16(__byte_perm(r.v[0][w], r.v[1][w], even));
        a[1] = codes_to_bf16(__byte_perm(r.v[0][w], r.v[1][w], odd));
        a[2] = codes_to_bf16(__byte_perm(r.v[2][w], r.v[3][w], even));
        a[3] = codes_to_bf16(__byte_perm(r.v[2][w], r.v[3][w], odd));
      } else {
        a[0] = __byte_perm(r.v[0][kt], r.v[1][kt], 0x5410);
        a[1] = __byte_perm(r.v[0][kt], r.v[1][kt], 0x7632);
        a[2] = __byte_perm(r.v[2][kt], r.v[3][kt], 0x5410);
        a[3] = __byte_perm(r.v[2][kt], r.v[3][kt], 0x7632);
      }
      mma_16x8x16(o[kt], a[0], a[1], a[2], a[3], b0, b1);
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) l[n] += __shfl_xor_sync(~0u, l[n], x);
    if (j == 0) s_m[warp][2 * c + n] = m[n], s_l[warp][2 * c + n] = l[n];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      s_o[warp][2 * c + n][v_dim<D, I8>(j, 2 * kt)] = o[kt][n];
      s_o[warp][2 * c + n][v_dim<D, I8>(j, 2 * kt + 1)] = o[kt][2 + n];
    }
  }
  __syncthreads();
  // join the warps
  const long long total_rows = (long long)p.batch * p.q_heads;
  const int part = (shared ? 0 : p.prefix_slots) + slot;
  for (int i = threadIdx.x; i < 8 * D; i += kWarps * 32) {
    const int n = i / D, d = i % D;
    int b, h;
    if (!locate(n, b, h)) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][n]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, lsum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2_approx(s_m[w][n] - base);
      sum += s_o[w][n][d] * f;
      lsum += s_l[w][n] * f;
    }
    const long long at = part * total_rows + (long long)b * p.q_heads + h;
    p.part_o[at * D + d] = sum;
    if (d == 0) p.part_ml[at] = make_float2(top, lsum);
  }
}

// One warp per (sequence, query head) joins its items.
template <int D>
__global__ void __launch_bounds__(128) join(const AttnParams p) {
  const long long row = blockIdx.x * 4ll + threadIdx.x / 32, rows = (long long)p.batch * p.q_heads;
  const int lane = threadIdx.x % 32;
  if (row >= rows) return;
  const int b = (int)(row / p.q_heads), h = (int)(row % p.q_heads);
  const int len = min(max(p.own_lens[b], 0), p.max_own);
  const int parts = p.prefix_slots + (len + p.own_chunk - 1) / p.own_chunk;
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 32) top = fmaxf(top, p.part_ml[i * rows + row].x);
#pragma unroll
  for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
  const float base = top == -INFINITY ? 0.f : top;
  float o[D / 32] = {}, l = 0.f;
  for (int i = 0; i < parts; ++i) {
    const float2 ml = p.part_ml[i * rows + row];
    const float f = exp2_approx(ml.x - base);
    l += ml.y * f;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] += f * p.part_o[(i * rows + row) * D + lane * (D / 32) + e];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key: zeros
  __nv_bfloat16* out = p.out + b * p.out_batch + h * p.out_head + lane * (D / 32);
#pragma unroll
  for (int e = 0; e < D / 32; e += 2)
    *reinterpret_cast<uint32_t*>(out + e) = pack_bf16(o[e] * inv, o[e + 1] * inv);
  if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (base + log2f(l)) * 0.6931471805599453f;
}

int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// Keys per item and items per row, so that the items fill the GPU once or twice.
struct Plan {
  int prefix_chunk, prefix_slots, own_chunk, own_slots;
  long long part_bytes;
};

int make_plan(const EkPrefixAttnArgs* a, Plan& pl) {
  using ek::fail;
  if (!a) return fail(EK_E_INVALID, "NULL arguments");
  if (a->batch < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads)
    return fail(EK_E_INVALID, "bad sizes batch=%d q_heads=%d kv_heads=%d", a->batch, a->q_heads, a->kv_heads);
  if (a->head_dim != 64 && a->head_dim != 128)
    return fail(EK_E_UNSUPPORTED, "head_dim %d (supported: 64, 128)", a->head_dim);
  if (a->prefix_len < 0 || a->own_capacity < 0 || a->max_own_len < 0 || a->max_own_len > a->own_capacity)
    return fail(EK_E_INVALID, "bad lengths prefix_len=%d own_capacity=%d max_own_len=%d", a->prefix_len,
                a->own_capacity, a->max_own_len);
  if ((long long)a->batch * a->q_heads > (1 << 22))
    return fail(EK_E_UNSUPPORTED, "batch * q_heads beyond %d", 1 << 22);
  int sms = 0;
  cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, a->device);
  if (e != cudaSuccess) return ek::cuda_fail(e, "cudaDeviceGetAttribute");
  const int group = a->q_heads / a->kv_heads;
  const long long want = 4ll * sms;
  const long long tiles = (long long)div_up((long long)a->batch * group, 8) * a->kv_heads;
  auto chunk = [&](long long len, long long items) {
    const long long splits = items < want ? div_up(want, items) : 1;
    const long long c = div_up(div_up(len, splits), 64) * 64ll;
    return (int)(c < 64 ? 64 : c);
  };
  pl.prefix_chunk = chunk(a->prefix_len, tiles > 0 ? tiles : 1);
  pl.prefix_slots = div_up(a->prefix_len, pl.prefix_chunk);
  const long long own = (long long)a->batch * div_up(group, 8) * a->kv_heads;
  pl.own_chunk = chunk(a->max_own_len, own > 0 ? own : 1);
  pl.own_slots = div_up(a->max_own_len, pl.own_chunk);
  pl.part_bytes = (long long)(pl.prefix_slots + pl.own_slots) * a->batch * a->q_heads * (a->head_dim * 4 + 8);
  return EK_SUCCESS;
}

// Fills one side of `s`; checks alignment and kind when there are rows.
int take_store(const EkKvTensor& k, const EkKvTensor& v, bool rows, bool i8, const char* name, Store& s) {
  using ek::fail;
  if (rows) {
    const int unit = i8 ? 16 : 8;
    for (const EkKvTensor* t : {&k, &v}) {
      if (!t->data || !ek::aligned16(t->data) || t->stride_batch % unit || t->stride_row % unit || t->stride_head % unit)
        return fail(EK_E_INVALID, "%s rows must be 16-byte aligned with strides of 16 bytes", name);
      if ((t->scales != nullptr) != i8) return fail(EK_E_INVALID, "prefix and own rows must be of one kind");
    }
  }
  const int size = i8 ? 1 : 2;
  s.k = static_cast<const char*>(k.data), s.v = static_cast<const char*>(v.data);
  s.ks = static_cast<const __nv_bfloat16*>(k.scales), s.vs = static_cast<const __nv_bfloat16*>(v.scales);
  s.k_batch = k.stride_batch * size, s.k_row = k.stride_row * size, s.k_head = k.stride_head * size;
  s.v_batch = v.stride_batch * size, s.v_row = v.stride_row * size, s.v_head = v.stride_head * size;
  s.ks_batch = k.scale_stride_batch, s.ks_row = k.scale_stride_row, s.ks_head = k.scale_stride_head;
  s.vs_batch = v.scale_stride_batch, s.vs_row = v.scale_stride_row, s.vs_head = v.scale_stride_head;
  return EK_SUCCESS;
}

template <int D, bool I8>
cudaError_t launch(const AttnParams& p, cudaStream_t st) {
  const long long items = (long long)p.prefix_slots * p.prefix_tiles * p.kv_heads +
                          (long long)p.own_slots * p.group_tiles * p.kv_heads * p.batch;
  if (items > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  if (items > 0) few_rows<D, I8><<<(unsigned)items, kWarps * 32, 0, st>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  join<D><<<div_up((long long)p.batch * p.q_heads, 4), 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace

extern "C" int64_t ek_prefix_attention_workspace(const EkPrefixAttnArgs* a) {
  Plan pl;
  return make_plan(a, pl) ? -1 : pl.part_bytes;
}

extern "C" int ek_prefix_attention(const EkPrefixAttnArgs* a, void* stream) {
  using ek::fail;
  Plan pl;
  int rc = make_plan(a, pl);
  if (rc) return rc;
  if (a->batch == 0) return EK_SUCCESS;
  if (!a->q || !a->out || !a->own_lens) return fail(EK_E_INVALID, "NULL pointer argument");
  if (!ek::aligned16(a->q) || a->q_stride_batch % 8 || a->q_stride_head % 8)
    return fail(EK_E_INVALID, "q must be 16-byte aligned with strides of 16 bytes");
  if (!ek::aligned16(a->out) || a->out_stride_batch % 8 || a->out_stride_head % 8)
    return fail(EK_E_INVALID, "out must be 16-byte aligned with strides of 16 bytes");
  if (pl.part_bytes > 0 && (!a->workspace || !ek::aligned16(a->workspace) || a->workspace_bytes < pl.part_bytes))
    return fail(EK_E_INVALID, "workspace of %lld bytes, 16-byte aligned, needed", pl.part_bytes);
  const bool i8 = (a->prefix_len > 0 ? a->prefix_k.scales : a->own_k.scales) != nullptr;
  AttnParams p;
  if ((rc = take_store(a->prefix_k, a->prefix_v, a->prefix_len > 0, i8, "prefix", p.prefix))) return rc;
  if ((rc = take_store(a->own_k, a->own_v, a->max_own_len > 0, i8, "own", p.own))) return rc;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_batch = a->q_stride_batch, p.q_head = a->q_stride_head;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.out_batch = a->out_stride_batch, p.out_head = a->out_stride_head;
  p.lse = a->lse;
  p.own_lens = a->own_lens;
  p.batch = a->batch, p.q_heads = a->q_heads, p.kv_heads = a->kv_heads;
  p.group = a->q_heads / a->kv_heads;
  p.prefix_len = a->prefix_len, p.max_own = a->max_own_len;
  p.prefix_chunk = pl.prefix_chunk, p.own_chunk = pl.own_chunk;
  p.prefix_slots = pl.prefix_slots, p.own_slots = pl.own_slots;
  p.prefix_tiles = div_up((long long)a->batch * p.group, 8);
  p.group_tiles = div_up(p.group, 8);
  const long long rows = (long long)a->batch * a->q_heads;
  p.part_o = static_cast<float*>(a->workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (pl.prefix_slots + pl.own_slots) * rows * a->head_dim);
  p.scale_log2 = a->scale * kLog2e;
  ek::DeviceGuard g(a->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->head_dim == 64) e = i8 ? launch<64, true>(p, st) : launch<64, false>(p, st);
  else e = i8 ? launch<128, true>(p, st) : launch<128, false>(p, st);
  return e == cudaSuccess ? EK_SUCCESS : ek::cuda_fail(e, "ek_prefix_attention launch");
}
