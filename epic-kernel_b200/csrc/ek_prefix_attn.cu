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
// rows. With 8-bit rows the contraction order over d is free, so lane c of a
// quad takes 16 consecutive codes and q is laid out to match. P^T becomes a B
// fragment by one 8x8 transpose in registers. 8-bit codes are exact in bf16;
// K's scale multiplies the score and V's scale the probability. Bound: bytes
// (4 flops per byte and query row); with 8-bit rows the instructions that widen
// the codes. `many_rows` takes the prefix when it serves many query rows.
// Times: 256 sequences, 24 heads over 8 KV heads of 128, up to 512 own bf16
// rows (270 MB): 53 us alone, 5.1 TB/s; 61 sequences, 32 heads, up to 1023
// own 8-bit rows (64 MB): 40 us, the longest sequence's blocks last; 16
// sequences, 32 heads of 64 over 2048 shared rows and up to 256 own: 9 us.
#include <cuda_bf16.h>

#include <cstring>

#include "ek_host.h"
#include "ek_tcgen05.cuh"

namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

__device__ int g_attention_status;  // 1: a wait inside a kernel ran out

struct Scales {  // of 8-bit rows, which come by tensor maps themselves
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  long long k_batch, k_row, k_head, v_batch, v_row, v_head;  // elements
};

struct AttnParams {
  Scales prefix, own;
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
  int prefix_slots, own_slots;    // items per row, at most
  int wide_rows, wide_slots, narrow_slots;  // prefix items of the rows of a KV head below wide_rows, and of the others
  int prefix_tiles, group_tiles;  // tiles of 8 rows: of batch * group, of group
  float scale_log2;
};

// Programmatic launches: the next kernel of the stream may start; the one before has ended and its writes are visible.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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

// ---------------------------------------------------------------------------
// `few_rows`: an item of up to 8 query rows of one KV head. A loader warp brings
// 64 keys a stage into shared memory by TMA (K and V of the head, swizzled), and
// each of four warps takes 16 of them.
template <int D, bool I8>
struct Few {
  static constexpr int KEYS = 64, BOX = 32;            // keys of a stage, and of a TMA copy
  static constexpr int TILE = KEYS * D * (I8 ? 1 : 2);  // bytes of a stage's K (or V)
  static constexpr int STAGES = I8 ? (D == 128 ? 3 : 4) : (D == 128 ? 2 : 3);
  static constexpr int OFF_BAR = 2 * STAGES * TILE;
  static constexpr int SMEM = OFF_BAR + 2 * STAGES * 8 + 16 + kWarps * 8 * 8;
  static_assert(kWarps * 8 * D * 4 <= 2 * STAGES * TILE, "the warps' O in the place of the stages");
};

// A tensor map of rows [batch][row][head][D] and where the coordinates go: the dimensions behind D are sorted by stride.
struct RowMap {
  CUtensorMap map;
  int8_t head, row, batch;  // place of the coordinate, or -1: the dimension is not there (one entry, or stride 0)

  __device__ __forceinline__ void load(void* dst, int d, int h, int r, int b, uint64_t* bar) const {
    const int c0 = head == 0 ? h : row == 0 ? r : batch == 0 ? b : 0;
    const int c1 = head == 1 ? h : row == 1 ? r : batch == 1 ? b : 0;
    const int c2 = head == 2 ? h : row == 2 ? r : batch == 2 ? b : 0;
    ek::tma_load_4d(dst, &map, d, c0, c1, c2, bar);
  }
};

struct FewParams {
  RowMap prefix_k, prefix_v, own_k, own_v;
  AttnParams a;
};

template <int D, bool I8>
__global__ void __launch_bounds__(kWarps * 32 + 32) few_rows(const __grid_constant__ FewParams fp) {
  using C = Few<D, I8>;
  constexpr int KT = D / 16;  // 16-wide steps over the dimensions
  const AttnParams& p = fp.a;
  launch_next();
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + C::STAGES;
  volatile int* abort = reinterpret_cast<volatile int*>(empty + C::STAGES);
  float* s_m = reinterpret_cast<float*>(smem + C::OFF_BAR + 2 * C::STAGES * 8 + 16);
  float* s_l = s_m + kWarps * 8;
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32, c = lane % 4, j = lane / 4;

  // the item
  long long id = blockIdx.x;
  const long long prefix_items = (long long)p.prefix_slots * p.prefix_tiles * p.kv_heads;
  const bool shared = id < prefix_items;
  int head, tile, slot, seq = 0;
  if (shared) {
    head = (int)(id % p.kv_heads), id /= p.kv_heads;
    tile = (int)(id % p.prefix_tiles);
    slot = (int)(id / p.prefix_tiles);
  } else {
    id -= prefix_items;
    head = (int)(id % p.kv_heads), id /= p.kv_heads;
    tile = (int)(id % p.group_tiles), id /= p.group_tiles;
    seq = (int)(id % p.batch);
    slot = (int)(id / p.batch);
  }
  const int chunk = shared ? p.prefix_chunk : p.own_chunk, t0 = slot * chunk;
  const int t1 = min(t0 + chunk, shared ? p.prefix_len : min(max(__ldg(p.own_lens + seq), 0), p.max_own));
  if (t0 >= t1) return;
  const int steps = (t1 - t0 + C::KEYS - 1) / C::KEYS;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) ek::mbar_init(full + i, 1), ek::mbar_init(empty + i, kWarps);
    *abort = 0;
    ek::fence_mbar_init();
  }
  __syncthreads();
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // for a whole warp, which goes on or gives up together
    return __all_sync(~0u, ek::mbar_wait_bounded(bar, parity, abort)) != 0;
  };
  const int rows = shared ? p.batch * p.group : p.group;
  // row n of the tile -> (sequence, query head)
  auto locate = [&](int n, int& b, int& h) {
    const int r = tile * 8 + n;
    b = shared ? r / p.group : seq;
    h = head * p.group + (shared ? r % p.group : r);
    return r < rows;
  };
  float o[KT][4] = {};  // O^T: two dimensions of rows 2c, 2c + 1
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  if (warp == kWarps) {
    int n = 0;
    for (; n < steps; ++n) {
      const int s = n % C::STAGES, t = t0 + n * C::KEYS;
      if (n >= C::STAGES && !wait(empty + s, (n / C::STAGES - 1) & 1)) break;
      if (ek::elect_one()) {
        // copies of 32 keys, those that begin before the end
        const int boxes = t + C::BOX < t1 ? 2 : 1;
        ek::mbar_arrive_expect_tx(full + s, boxes * (C::TILE / 2) * 2);
        for (int kv = 0; kv < 2; ++kv) {
          const RowMap& map = shared ? (kv ? fp.prefix_v : fp.prefix_k) : kv ? fp.own_v : fp.own_k;
          uint8_t* to = smem + (2 * s + kv) * C::TILE;
          constexpr int ROW = I8 ? D : 128;  // bytes of a row of a copy
          for (int blk = 0; blk < (I8 ? 1 : D / 64); ++blk)
            for (int half = 0; half < boxes; ++half)
              map.load(to + (blk * C::KEYS + half * C::BOX) * ROW, blk * 64, head, t + half * C::BOX, seq, full + s);
        }
      }
      __syncwarp();
    }
    // The last copy of each stage lands before the stages hold O, also where a warp that gave up did not wait for it.
    int quiet = 0;
    for (int i = max(0, n - C::STAGES); i < n; ++i) ek::mbar_wait_bounded(full + i % C::STAGES, (i / C::STAGES) & 1, &quiet);
  } else {
    // q of row lane/4 as B fragments
    uint32_t q[KT][2];
    {
      int b, h;
      const bool in = locate(j, b, h);
      const __nv_bfloat16* at = p.q + b * p.q_batch + h * p.q_head;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if (I8) {  // the dimensions that quad lane c takes of K: 16 codes at a time
          const uint2 x = in ? __ldg(reinterpret_cast<const uint2*>(at + (kt / 4) * 64 + c * 16 + (kt % 4) * 4)) : make_uint2(0, 0);
          q[kt][0] = x.x, q[kt][1] = x.y;
        } else {
          q[kt][0] = in ? __ldg(reinterpret_cast<const uint32_t*>(at + kt * 16 + c * 2)) : 0u;
          q[kt][1] = in ? __ldg(reinterpret_cast<const uint32_t*>(at + kt * 16 + c * 2 + 8)) : 0u;
        }
      }
    }
    const Scales& scales = shared ? p.prefix : p.own;
    const __nv_bfloat16* ksb = scales.k + seq * scales.k_batch + head * scales.k_head;
    const __nv_bfloat16* vsb = scales.v + seq * scales.v_batch + head * scales.v_head;
    float ks[2], vs[2];  // scales of keys j and j + 8 of the step
    auto load_scales = [&](int t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = t + j + 8 * i < t1;
        ks[i] = in ? __bfloat162float(ksb[(t + j + 8 * i) * scales.k_row]) : 0.f;
        vs[i] = in ? __bfloat162float(vsb[(t + j + 8 * i) * scales.v_row]) : 0.f;
      }
    };
    if (I8) load_scales(t0 + warp * 16);
    bool ok = true;
    for (int n = 0; n < steps; ++n) {
      const int st = n % C::STAGES, t = t0 + n * C::KEYS + warp * 16;
      if (!(ok = wait(full + st, (n / C::STAGES) & 1))) break;
      if (t < t1) {
        const uint32_t kt0 = ek::smem_u32(smem + 2 * st * C::TILE), vt0 = kt0 + C::TILE;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (I8) {
#pragma unroll
          for (int m4 = 0; m4 < KT / 4; ++m4) {
            uint4 w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = warp * 16 + j + 8 * i, ch = m4 * 4 + c;
              w[i] = ek::lds128(kt0 + r * D + ((D == 128 ? ch ^ (r & 7) : ch ^ (r >> 1 & 3)) << 4));
            }
            const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&w[0]);
            const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&w[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              mma_16x8x16(s, codes_to_bf16(__byte_perm(w0[e], w0[e], 0x1100)), codes_to_bf16(__byte_perm(w1[e], w1[e], 0x1100)),
                          codes_to_bf16(__byte_perm(w0[e], w0[e], 0x3322)), codes_to_bf16(__byte_perm(w1[e], w1[e], 0x3322)),
                          q[m4 * 4 + e][0], q[m4 * 4 + e][1]);
          }
        } else {
          const int r = warp * 16 + lane % 16;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const int ch = 2 * kt + lane / 16;
            uint32_t a[4];
            ek::ldmatrix4<false>(a, kt0 + ch / 8 * (C::KEYS * 128) + r * 128 + ((ch % 8 ^ (r & 7)) << 4));
            mma_16x8x16(s, a[0], a[1], a[2], a[3], q[kt][0], q[kt][1]);
          }
        }
        // s[0], s[1]: key t + j of rows 2c, 2c + 1; s[2], s[3]: key t + j + 8
        float fix[2];
        bool grew = false;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[i] = t + j + 8 * (i / 2) < t1 ? s[i] * (I8 ? p.scale_log2 * ks[i / 2] : p.scale_log2) : -INFINITY;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = fmaxf(s[r], s[2 + r]);
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 4));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 8));
          top = fmaxf(top, __shfl_xor_sync(~0u, top, 16));
          const float next = fmaxf(m[r], top);
          const float base = next == -INFINITY ? 0.f : next;
          fix[r] = exp2_approx(m[r] - base);
          grew |= next != m[r];
          m[r] = next;
          s[r] = exp2_approx(s[r] - base);
          s[2 + r] = exp2_approx(s[2 + r] - base);
          l[r] = l[r] * fix[r] + s[r] + s[2 + r];
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
          for (int i = 0; i < 4; ++i) s[i] *= vs[i / 2];  // (0 past the end)
          load_scales(t + C::KEYS);
        }
        // probabilities are rounded to bf16 for the product: half a step is 2^-8 of each, as for V itself
        const uint32_t b0 = transpose_8x8(pack_bf16(s[0], s[1])), b1 = transpose_8x8(pack_bf16(s[2], s[3]));
        if (I8) {
          uint32_t v[4][D / 32];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = warp * 16 + 2 * c + (i & 1) + (i & 2) * 4;
            if (D == 128) {
              const uint4 x = ek::lds128(vt0 + r * 128 + ((j ^ (r & 7)) << 4));
              v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
            } else {
              const uint2 x = *reinterpret_cast<const uint2*>(smem + (2 * st + 1) * C::TILE + r * 64 +
                                                              ((j / 2 ^ (r >> 1 & 3)) << 4) + (j & 1) * 8);
              v[i][0] = x.x, v[i][1] = x.y;
            }
          }
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const int w = kt / 2, e = (kt % 2) * 2;  // word and first byte of element 2 kt
            const uint32_t even = e == 0 ? 0x4400 : 0x6622, odd = e == 0 ? 0x5511 : 0x7733;
            mma_16x8x16(o[kt], codes_to_bf16(__byte_perm(v[0][w], v[1][w], even)),
                        codes_to_bf16(__byte_perm(v[0][w], v[1][w], odd)), codes_to_bf16(__byte_perm(v[2][w], v[3][w], even)),
                        codes_to_bf16(__byte_perm(v[2][w], v[3][w], odd)), b0, b1);
          }
        } else {
          const int r = warp * 16 + lane % 8 + lane / 16 * 8;
          // rows past the end may hold anything, NaN too, which 0 would not cancel: keys 2c, 2c + 1 and eight on
          uint32_t keep[2] = {~0u, ~0u};
          if (t + 16 > t1) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              keep[i] = (t + 2 * c + 8 * i < t1 ? 0xffffu : 0u) | (t + 2 * c + 8 * i + 1 < t1 ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const int ch = 2 * kt + (lane / 8 & 1);
            uint32_t a[4];
            ek::ldmatrix4<true>(a, vt0 + ch / 8 * (C::KEYS * 128) + r * 128 + ((ch % 8 ^ (r & 7)) << 4));
            mma_16x8x16(o[kt], a[0] & keep[0], a[1] & keep[0], a[2] & keep[1], a[3] & keep[1], b0, b1);
          }
        }
      }
      __syncwarp();
      if (lane == 0) ek::mbar_arrive(empty + st);
    }
    if (!ok) m[0] = m[1] = l[0] = l[1] = NAN;  // a wait ran out: the result is NaN and the status is set
  }
  __syncthreads();  // all stages are done with
  if (threadIdx.x == 0 && *abort) g_attention_status = 1;
  float* s_o = reinterpret_cast<float*>(smem);  // [warp][8][D]
  if (warp < kWarps) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n] += __shfl_xor_sync(~0u, l[n], x);
      if (j == 0) s_m[warp * 8 + 2 * c + n] = m[n], s_l[warp * 8 + 2 * c + n] = l[n];
      float* at = s_o + (warp * 8 + 2 * c + n) * D;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        // 8-bit rows: lane/4 holds D / 8 consecutive dimensions
        at[I8 ? j * (D / 8) + 2 * kt : kt * 16 + j] = o[kt][n];
        at[I8 ? j * (D / 8) + 2 * kt + 1 : kt * 16 + j + 8] = o[kt][2 + n];
      }
    }
  }
  __syncthreads();
  // join the warps
  const long long total_rows = (long long)p.batch * p.q_heads;
  const int part = (shared ? 0 : p.prefix_slots) + slot;
  for (int i = threadIdx.x; i < 8 * (D / 4); i += kWarps * 32 + 32) {
    const int n = i / (D / 4), d = i % (D / 4) * 4;
    int b, h;
    if (!locate(n, b, h)) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * 8 + n]);
    const float base = top == -INFINITY ? 0.f : top;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float lsum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2_approx(s_m[w * 8 + n] - base);
      const float4 x = *reinterpret_cast<const float4*>(s_o + (w * 8 + n) * D + d);
      sum.x += x.x * f, sum.y += x.y * f, sum.z += x.z * f, sum.w += x.w * f;
      lsum += s_l[w * 8 + n] * f;
    }
    const long long at = part * total_rows + (long long)b * p.q_heads + h;
    *reinterpret_cast<float4*>(p.part_o + at * D + d) = sum;
    if (d == 0) p.part_ml[at] = make_float2(top, lsum);
  }
}

// ---------------------------------------------------------------------------
// `many_rows`: the prefix for many query rows, on tcgen05.
//
// One block takes one KV head, up to 256 query rows and a range of keys, in
// tiles of 128 keys. S = Q K^T (128 x 128 fp32) and O += P V (128 x D) stay in
// tensor memory; P goes there as bf16 and is read as the A operand. Two softmax
// warpgroups work in turn with the tensor core. They take S into registers at
// once, so that one S buffer serves both: the next scores are computed while
// exponentials are taken, and no warpgroup waits for the products of its own
// tile. With more than 128 rows
// the warpgroups hold two row tiles and share every K and V tile ("wide");
// with fewer they hold the same rows and take alternate key tiles, each with a
// running maximum, sum and O of its own ("narrow"). A thread owns one row, so
// the row maximum and sum need no shuffles. O is rescaled only when a maximum
// grows by more than 2^8; until then the old one stays in use, which changes
// no ratio.
//
// P is rounded to bf16, V's type, by at most 2^-8 of each probability (times V's scale, with 8-bit rows), while the sums
// keep it in fp32. The rest of P as a second operand would double the products with V, half of the tensor core's work.
//
// K and V tiles come by TMA (128-byte swizzle) into a ring, in the order in
// which the products use them. 8-bit tiles land in a raw ring and four warps
// widen them to bf16 in the swizzled layout; the scales of keys multiply
// scores and probabilities, as in few_rows.
//
// Bound: 256 rows take 4 * 256 * 128 * D flops a tile, 2048 tensor cycles at
// D = 128, and 2 * 128 * 128 exponentials, 2048 cycles at 16 a cycle; and the
// power limit. 256 sequences of 24 heads of 128 (768 rows per KV head) over
// 32768 bf16 rows: 89 us, 1.16 PFLOP/s. With 8-bit rows the widening warps
// (16384 codes a tile, 1356 cycles if nothing else runs): 160 us, and 46 us for
// 61 sequences of 32 heads over 16001 rows.
template <int D, bool I8>
struct Many {
  static constexpr int BLOCKS = D / 64;               // 64-element column blocks of a tile
  static constexpr int TILE = 128 * D * 2;            // bytes of a bf16 tile
  static constexpr int RAW = 128 * D;                 // bytes of an 8-bit tile
  // K and V have rings of their own: two warps consume them, and each must see every phase of its barriers
  static constexpr int KS = D == 64 ? 4 : I8 ? 2 : 3, VS = D == 64 ? 4 : 2;
  static constexpr int RAW_STAGES = I8 ? (D == 128 ? 2 : 4) : 0;
  static constexpr int WARPS = I8 ? 16 : 12;          // 8 softmax, [4 widening,] loads, scores, values, 1 idle
  static constexpr int LOADER = WARPS - 4, SCORES = WARPS - 3, VALUES = WARPS - 2;
  // registers per thread: at launch, of the softmax, widening and other warpgroups
  static constexpr int REGS = I8 ? 128 : 168, SOFTMAX_REGS = I8 ? 200 : 208, WIDEN_REGS = 72, OTHER_REGS = I8 ? 40 : 88;
  static_assert(2 * SOFTMAX_REGS + (I8 ? WIDEN_REGS : 0) + OTHER_REGS == WARPS / 4 * REGS, "registers of the block");
  static constexpr int OFF_K = 2 * TILE;              // after two Q tiles
  static constexpr int OFF_V = OFF_K + KS * TILE;
  static constexpr int OFF_RAW = OFF_V + VS * TILE;
  static constexpr int OFF_SCALE = OFF_RAW + RAW_STAGES * RAW;
  static constexpr int SCALE_BYTES = I8 ? 2 * 2 * 128 * 4 : 0;  // warpgroup, k / v, key
  static constexpr int OFF_BAR = OFF_SCALE + SCALE_BYTES;
  static constexpr int BARS = 2 * KS + 2 * VS + 2 * RAW_STAGES + 6 + 3;
  static constexpr int OUT_ROW = D * 4 + 16;          // bytes of a row of O on its way out; eight rows meet all banks
  static_assert(256 * OUT_ROW <= OFF_RAW, "rows of O in the place of Q, K and V");
  static constexpr int S = 0, P = 128, O = 256;       // columns of tensor memory: scores, P and O of both warpgroups
  static constexpr int SMEM = OFF_BAR + BARS * 8 + 16;
};

struct ManyParams {
  RowMap k, v;
  AttnParams a;
  int rows, wide_blocks, narrow_rows;  // rows of a KV head; blocks of 256; rows left for a narrow block
  int wide_splits, wide_tiles, narrow_splits, narrow_tiles;  // splits of the keys and 128-key tiles of each
  // Masked scores are -inf times the scale, so that is kept positive. scale < 0: q is negated. scale = 0: q is 0
  // (infinities and NaN are NaN, as 0 times their products).
  uint32_t q_flip;              // bits of q to turn
  int q_zero;
};


// Columns from `keys` on of 32 scores become -inf.
__device__ __forceinline__ void mask_tail(uint32_t (&x)[32], int keys) {
#pragma unroll
  for (int e = 0; e < 32; ++e)
    if (e >= keys) x[e] = 0xff800000u;
}

__device__ __forceinline__ uint64_t score_pair(const uint32_t (&x)[32], int e) {
  return ek::pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1]));
}

template <int D, bool I8>
__global__ void __launch_bounds__(Many<D, I8>::WARPS * 32, 1) many_rows(const __grid_constant__ ManyParams p) {
  using C = Many<D, I8>;
  launch_next();
  extern __shared__ __align__(1024) uint8_t smem[];  // atoms of the swizzle start on 1024 bytes
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* k_empty = k_full + C::KS;
  uint64_t* v_full = k_empty + C::KS;
  uint64_t* v_empty = v_full + C::VS;
  uint64_t* raw_full = v_empty + C::VS;
  uint64_t* raw_empty = raw_full + C::RAW_STAGES;
  uint64_t* s_full = raw_empty + C::RAW_STAGES;
  uint64_t* p_full = s_full + 2;
  uint64_t* p_empty = p_full + 2;   // the products with P are done
  uint64_t* s_empty = p_empty + 2;  // the scores are in registers
  uint64_t* q_full = s_empty + 1;
  uint64_t* drained = q_full + 1;
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_at + 1);
  const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0);  // uniform

  // the item
  int id = blockIdx.x;
  const int wide_items = p.wide_blocks * p.wide_splits * p.a.kv_heads;
  const bool wide = id < wide_items;
  if (!wide) id -= wide_items;
  const int splits = wide ? p.wide_splits : p.narrow_splits, per = wide ? p.wide_tiles : p.narrow_tiles;
  const int split = id % splits;
  id /= splits;
  const int head = id % p.a.kv_heads;
  const int row0 = wide ? id / p.a.kv_heads * 256 : p.wide_blocks * 256;
  const int row1 = wide ? min(p.rows, row0 + 256) : p.rows;
  const int tile0 = split * per;
  const int tiles = min(per, (p.a.prefix_len + 127) / 128 - tile0);

  if (warp == C::SCORES) ek::tmem_alloc(tmem_at, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::KS; ++i) ek::mbar_init(k_full + i, I8 ? 4 : 1), ek::mbar_init(k_empty + i, 1);
    for (int i = 0; i < C::VS; ++i) ek::mbar_init(v_full + i, I8 ? 4 : 1), ek::mbar_init(v_empty + i, 1);
    for (int i = 0; i < C::RAW_STAGES; ++i) ek::mbar_init(raw_full + i, 1), ek::mbar_init(raw_empty + i, 4);
    for (int i = 0; i < 2; ++i) ek::mbar_init(s_full + i, 1), ek::mbar_init(p_full + i, 4), ek::mbar_init(p_empty + i, 1);
    ek::mbar_init(s_empty, 4), ek::mbar_init(q_full, 8), ek::mbar_init(drained, 2);
    *abort = 0;
    ek::fence_mbar_init();
  }
  ek::tcgen05_before_sync();
  __syncthreads();
  ek::tcgen05_after_sync();
  const uint32_t tmem = *tmem_at;

  // Order in which tiles are fetched: K_0 .. K_{lead-1}, then V_i, K_{i+lead} in turn, then the last V. Item n:
  const int items = 2 * tiles, lead = min(C::KS, tiles);
  auto item = [&](int n, bool& is_v) {
    const int m = n - lead, both = 2 * (tiles - lead);
    is_v = m >= both || (m >= 0 && m % 2 == 0);
    return m < 0 ? n : m >= both ? m - (tiles - lead) : m / 2 + (is_v ? 0 : lead);
  };
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // for a whole warp, which goes on or gives up together
    return __all_sync(~0u, ek::mbar_wait_bounded(bar, parity, abort)) != 0;
  };
  // Where the softmax or the tensor core would stand still. With 8-bit rows polls would slow the widening warps, which
  // the others wait for (256 x 24 heads of 128, 32768 rows: 218 us with polls, 160 without).
  auto spin = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(~0u, ek::mbar_wait_bounded<!I8>(bar, parity, abort)) != 0;
  };
  // One arrival per warp: 128 on one barrier are serialised.
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (threadIdx.x % 32 == 0) ek::mbar_arrive(bar);
  };

  if (warp < 8) {
    ek::registers_up<C::SOFTMAX_REGS>();
    {  // Q rows into the swizzled tiles, zeros past the last; eight loads at a time
      constexpr int PIECES = D / 8, ROWS = 32 / PIECES, BATCH = 8;
      const int piece = threadIdx.x % PIECES, r0 = warp * 32 + threadIdx.x % 32 / PIECES;
      const int rows = wide ? 32 : 16, first = wide ? r0 : warp * 16 + threadIdx.x % 32 / PIECES;
      for (int i = 0; i < rows; i += ROWS * BATCH) {
        uint4 x[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          const int r = first + i + u * ROWS, at = row0 + r;
          x[u] = make_uint4(0, 0, 0, 0);
          if (i + u * ROWS < rows && at < row1) {
            const int b = at / p.a.group, h = head * p.a.group + at % p.a.group;
            x[u] = __ldg(reinterpret_cast<const uint4*>(p.a.q + b * p.a.q_batch + h * p.a.q_head) + piece);
          }
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          if (i + u * ROWS >= rows) continue;
          const int r = first + i + u * ROWS, t = r % 128;
          if (p.q_zero || p.q_flip) {
            auto turn = [&](uint32_t y) {
              const uint32_t nan = __vcmpeq2(y & 0x7f807f80u, 0x7f807f80u) & 0x7fc07fc0u;
              return p.q_zero ? nan : y ^ p.q_flip;
            };
            x[u] = make_uint4(turn(x[u].x), turn(x[u].y), turn(x[u].z), turn(x[u].w));
          }
          *reinterpret_cast<uint4*>(smem + r / 128 * C::TILE + piece / 8 * 16384 + t * 128 + ((piece % 8 ^ (t & 7)) << 4)) = x[u];
        }
      }
      ek::fence_proxy_async_smem();
      arrive(q_full);
    }
    const int w = warp / 4, t = threadIdx.x % 128;
    const int row = row0 + (wide ? w * 128 : 0) + t;
    const bool idle = row0 + (wide ? w * 128 : 0) + (warp % 4) * 32 >= row1;  // no row in this warp
    const uint32_t lanes = tmem + ((uint32_t)(warp % 4 * 32) << 16);
    const uint32_t ts = lanes + C::S, tp = lanes + C::P + w * 64, to = lanes + C::O + w * D;
    const int mine = wide ? tiles : (tiles - w + 1) / 2;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const float scale = p.a.scale_log2;
    auto key_scale = [&](int use, int kv) {
      const int key = (tile0 + (wide ? use : 2 * use + w)) * 128 + t;
      if (use >= mine || key >= p.a.prefix_len) return kv ? 0.f : 1.f;  // masked scores stay -inf
      const Scales& s = p.a.prefix;
      return __bfloat162float(kv ? s.v[key * s.v_row + head * s.v_head] : s.k[key * s.k_row + head * s.k_head]);
    };
    float next_ks = 0.f, next_vs = 0.f;
    if (I8) next_ks = key_scale(0, 0), next_vs = key_scale(0, 1);
    // A warp whose wait runs out still comes to the next tile's barrier, where the warpgroup leaves together (with bf16
    // rows there is none, and it leaves alone).
    for (int use = 0; use < mine && (I8 || ok); ++use) {
      const int tile = tile0 + (wide ? use : 2 * use + w);
      const int keys = min(128, p.a.prefix_len - tile * 128);
      const float* ks = nullptr;
      const float* vs = nullptr;
      if (I8) {
        float* sc = reinterpret_cast<float*>(smem + C::OFF_SCALE) + w * 256;
        auto sync = [&] {
          if (w == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
          else asm volatile("bar.sync 2, 128;" ::: "memory");
        };
        auto agree = [&](bool x) { return w == 0 ? ek::barrier_all<1, 128>(x) : ek::barrier_all<2, 128>(x); };
        if (!(ok = agree(ok))) break;  // else the scales of the tile before are done with
        sc[t] = next_ks * scale, sc[128 + t] = next_vs;
        sync();
        ks = sc, vs = sc + 128;
        next_ks = key_scale(use + 1, 0), next_vs = key_scale(use + 1, 1);
      }
      if (!(ok = spin(s_full + w, use & 1))) continue;
      ek::tcgen05_after_sync();
      if (idle) {
        arrive(s_empty);
        if (use > 0 && !(ok = spin(p_empty + w, (use - 1) & 1))) continue;
      } else {
        uint32_t x[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) ek::tmem_ld32(x[c], ts + c * 32);
        ek::tmem_wait_ld(x[0]);
#pragma unroll
        for (int c = 1; c < 4; ++c) ek::tmem_after(x[c]);
        ek::tcgen05_before_sync();
        arrive(s_empty);
        if (I8) {  // scores in units of base 2
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 f = *reinterpret_cast<const float4*>(ks + c * 32 + e);
              const float2 a = ek::unpair(ek::mul2(score_pair(x[c], e), ek::pair(f.x, f.y)));
              const float2 b = ek::unpair(ek::mul2(score_pair(x[c], e + 2), ek::pair(f.z, f.w)));
              x[c][e] = __float_as_uint(a.x), x[c][e + 1] = __float_as_uint(a.y);
              x[c][e + 2] = __float_as_uint(b.x), x[c][e + 3] = __float_as_uint(b.y);
            }
        }
        if (keys < 128) {
#pragma unroll
          for (int c = 0; c < 4; ++c) mask_tail(x[c], keys - c * 32);
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          top[c] = __uint_as_float(x[c][0]);
#pragma unroll
          for (int e = 1; e < 31; e += 2) top[c] = ek::max3_nan(top[c], __uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1]));
          top[c] = ek::max3_nan(top[c], __uint_as_float(x[c][31]), top[c]);
        }
        const float high = ek::max3_nan(ek::max3_nan(top[0], top[1], top[2]), top[3], top[3]) * (I8 ? 1.f : scale);
        const float grown = ek::max3_nan(m, high, high);
        if (use == 0) m = grown;
        // O and P are free once the products of the tile before are done
        if (use > 0 && !(ok = spin(p_empty + w, (use - 1) & 1))) continue;
        ek::tcgen05_after_sync();
        const bool far = grown > m + 8.f || grown != grown;
        if (__any_sync(~0u, far)) {
          const float fix = far ? exp2_approx(m - grown) : 1.f;
          if (far) m = grown, l *= fix;
          if (use > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              ek::tmem_ld16(o, to + c * 16);
              ek::tmem_wait_ld(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fix);
              ek::tmem_st16(to + c * 16, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : m;
        const uint64_t slope = ek::pair(scale, scale), shift = ek::pair(-base, -base);
        uint64_t sums[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t out[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const uint64_t s2 = score_pair(x[c], e);
            const float2 t2 = ek::unpair(I8 ? ek::add2(s2, shift) : ek::fma2(s2, slope, shift));
            float2 pr = make_float2(exp2_approx(t2.x), exp2_approx(t2.y));
            uint64_t p2 = ek::pair(pr.x, pr.y);
            sums[e / 2 & 1] = ek::add2(sums[e / 2 & 1], p2);
            if (I8) {
              const float2 f = *reinterpret_cast<const float2*>(vs + c * 32 + e);
              pr = ek::unpair(ek::mul2(p2, ek::pair(f.x, f.y)));
            }
            out[e / 2] = pack_bf16(pr.x, pr.y);
          }
          ek::tmem_st16(tp + c * 16, out);
        }
        const float2 sum2 = ek::unpair(ek::add2(sums[0], sums[1]));
        l += sum2.x + sum2.y;
        ek::tmem_wait_st();
      }
      ek::tcgen05_before_sync();
      arrive(p_full + w);
    }
    if (ok && mine > 0) ok = wait(p_empty + w, (mine - 1) & 1);
    ek::tcgen05_after_sync();
    // All products of both warpgroups are done: Q, K and V are free, unless a wait ran out. Then all rows are NaN, and
    // the status is set.
    ok = ek::barrier_all<3, 256>(ok);
    if (!ok) m = NAN, l = NAN;
    if (!idle) {
      const int b = row / p.a.group, h = head * p.a.group + row % p.a.group;
      const long long total_rows = (long long)p.a.batch * p.a.q_heads;
      const long long at = (wide ? split : 2 * split + w) * total_rows + (long long)b * p.a.q_heads + h;
      if (row < row1) p.a.part_ml[at] = make_float2(m, l);
      // each row of O through shared memory as one bulk copy: a thread's own 16-byte stores would fill half sectors
      if (mine > 0 && ok) {
        uint8_t* mine_row = smem + (w * 128 + t) * C::OUT_ROW;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          ek::tmem_ld32(r, to + c * 32);
          ek::tmem_wait_ld(r);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint4*>(mine_row + c * 128 + e * 16) = make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
        }
        ek::fence_proxy_async_smem();
        if (row < row1) ek::bulk_store(p.a.part_o + at * D, mine_row, D * 4);
        ek::bulk_store_wait();
      }
    }
    ek::tcgen05_before_sync();
  } else if (I8 && warp < C::LOADER) {
    ek::registers_down<C::WIDEN_REGS>();
    const int t = threadIdx.x - 256;
    for (int n = 0; n < items; ++n) {
      constexpr int RS = I8 ? C::RAW_STAGES : 1;
      bool is_v;
      const int tile = item(n, is_v), rs = n % RS;
      const int stages = is_v ? C::VS : C::KS, cs = tile % stages;
      if (!wait(raw_full + rs, (n / RS) & 1)) break;
      if (tile >= stages && !wait((is_v ? v_empty : k_empty) + cs, (tile / stages - 1) & 1)) break;
      const uint8_t* raw = smem + C::OFF_RAW + rs * C::RAW;
      uint8_t* to = smem + (is_v ? C::OFF_V : C::OFF_K) + cs * C::TILE;
#pragma unroll 2
      for (int i = t; i < 128 * D / 16; i += 128) {
        const int r = i / (D / 16), piece = i % (D / 16);
        const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 16);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t y[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[2 * e] = codes_to_bf16(__byte_perm(w[e], w[e], 0x1100));
          y[2 * e + 1] = codes_to_bf16(__byte_perm(w[e], w[e], 0x3322));
        }
        // two 16-byte pieces of the 128-byte row; the second block writes them in the other order, so
        // that the eight lanes of a row hit different banks
        uint8_t* row = to + piece / 4 * 16384 + r * 128;
        const int c0 = piece % 4 * 2, flip = D == 128 ? piece / 4 : 0;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool hi = (e ^ flip) & 1;
          *reinterpret_cast<uint4*>(row + (((c0 + (hi ? 1 : 0)) ^ (r & 7)) << 4)) =
              hi ? make_uint4(y[4], y[5], y[6], y[7]) : make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
      ek::fence_proxy_async_smem();
      arrive((is_v ? v_full : k_full) + cs);
      arrive(raw_empty + rs);
    }
  } else {
    ek::registers_down<C::OTHER_REGS>();
    if (warp == C::LOADER) {
      constexpr int RS = I8 ? C::RAW_STAGES : 1, BYTES = I8 ? C::RAW : C::TILE;
      // buffer and barriers of item n
      auto slot = [&](int n, bool& is_v, int& tile, uint64_t*& f, uint64_t*& e, int& round, uint8_t*& to) {
        tile = item(n, is_v);
        const int stages = I8 ? RS : is_v ? C::VS : C::KS, at = I8 ? n : tile;
        round = at / stages;
        f = (I8 ? raw_full : is_v ? v_full : k_full) + at % stages;
        e = (I8 ? raw_empty : is_v ? v_empty : k_empty) + at % stages;
        to = smem + (I8 ? C::OFF_RAW : is_v ? C::OFF_V : C::OFF_K) + at % stages * BYTES;
      };
      bool is_v;
      int n = 0, tile, round, k_tiles = 0, v_tiles = 0;
      uint64_t *f, *e;
      uint8_t* to;
      for (; n < items; ++n) {
        slot(n, is_v, tile, f, e, round, to);
        if (round > 0 && !wait(e, (round - 1) & 1)) break;
        const int key = (tile0 + tile) * 128;
        const RowMap& map = is_v ? p.v : p.k;
        if (ek::elect_one()) {
          ek::mbar_arrive_expect_tx(f, BYTES);
          for (int blk = 0; blk < (I8 ? 1 : C::BLOCKS); ++blk)
            map.load(to + blk * 16384, blk * 64, head, key, 0, f);
        }
        __syncwarp();
        k_tiles += !is_v, v_tiles += is_v;
      }
      // The last copy of each buffer lands before the block ends, also where a warp that gave up did not wait for it.
      int quiet = 0;
      auto land = [&](uint64_t* f, int stages, int count) {
        for (int i = max(0, count - stages); i < count; ++i) ek::mbar_wait_bounded(f + i % stages, (i / stages) & 1, &quiet);
      };
      if (I8) land(raw_full, RS, n);
      else land(k_full, C::KS, k_tiles), land(v_full, C::VS, v_tiles);
    } else if (warp == C::SCORES || warp == C::VALUES) {
      // Two warps issue the products, so that neither's waits hold up the other's: the queue of issued products is
      // short, and a thread that issues is in step with the tensor core.
      constexpr uint32_t SD = ek::mma_desc(128, 128, false), OD = ek::mma_desc(128, D, true);
      const int count = wide ? 2 * tiles : tiles;  // products; number i belongs to warpgroup i % 2
      if (warp == C::SCORES) {
        // S = Q K^T of product i, once the scores before it have been taken
        for (int i = 0; i < count && (i > 0 || wait(q_full, 0)); ++i) {
          const int w = i % 2, t = wide ? i / 2 : i;
          if (!spin(k_full + t % C::KS, (t / C::KS) & 1) || (i > 0 && !spin(s_empty, (i - 1) & 1))) break;
          ek::tcgen05_after_sync();
          const uint32_t base = ek::smem_u32(smem);
          const uint32_t q = base + (wide ? w * C::TILE : 0), k = base + C::OFF_K + t % C::KS * C::TILE;
          if (ek::elect_one()) {
#pragma unroll
            for (int kt = 0; kt < D / 16; ++kt) {
              const uint32_t off = kt / 4 * 16384 + kt % 4 * 32;
              ek::mma_ss(tmem + C::S, ek::smem_desc(q + off, 16), ek::smem_desc(k + off, 16), SD, kt > 0);
            }
            ek::mma_commit(s_full + w);
            if (!wide || w == 1) ek::mma_commit(k_empty + t % C::KS);
          }
          __syncwarp();
        }
      } else {
        // O += P V of product i
        for (int i = 0; i < count; ++i) {
          const int w = i % 2, t = wide ? i / 2 : i;
          if (!spin(v_full + t % C::VS, (t / C::VS) & 1) || !spin(p_full + w, (i / 2) & 1)) break;
          ek::tcgen05_after_sync();
          const uint32_t v = ek::smem_u32(smem) + C::OFF_V + t % C::VS * C::TILE;
          if (ek::elect_one()) {
#pragma unroll
            for (int kt = 0; kt < 8; ++kt)
              ek::mma_ts(tmem + C::O + w * D, tmem + C::P + w * 64 + kt * 8, ek::smem_desc(v + kt * 2048, 16384), OD,
                         i > 1 || kt > 0);
            ek::mma_commit(p_empty + w);
            if (!wide || w == 1) ek::mma_commit(v_empty + t % C::VS);
          }
          __syncwarp();
        }
      }
      // tensor memory is freed below: nothing may be in flight
      int quiet = 0;
      if (ek::elect_one()) ek::mma_commit(drained);
      __syncwarp();
      ek::mbar_wait_bounded(drained, 0, &quiet);
    }
  }
  __syncwarp();
  wait_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort) g_attention_status = 1;
  if (warp == C::SCORES) {
    ek::tcgen05_after_sync();
    ek::tmem_free(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// A warp, or W warps of a block, per (sequence, query head) join its items: of 32 items, lane i takes the maximum and
// sum of item i, then the lanes go through the rows of O with 16-byte loads, two items (D = 64) or one at a time. Warp
// w of W takes every W-th item. Bound: latency (9 to 11 us behind 256 sequences of 24 heads, 6144 rows of up to 10
// items).
constexpr int kJoinWarps = 8;

template <int D, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) join(const AttnParams p) {
  constexpr int LANES = D / 4, AT_ONCE = 32 / LANES;
  const long long row = W == 1 ? blockIdx.x * 4ll + threadIdx.x / 32 : blockIdx.x, rows = (long long)p.batch * p.q_heads;
  const int lane = threadIdx.x % 32, sub = lane / LANES, piece = lane % LANES, warp = W == 1 ? 0 : threadIdx.x / 32;
  if (W == 1 && row >= rows) {
    wait_before();
    return;
  }
  const int b = (int)(row / p.q_heads), h = (int)(row % p.q_heads);
  const int len = min(max(p.own_lens[b], 0), p.max_own);
  const int shared = b * p.group + h % p.group < p.wide_rows ? p.wide_slots : p.narrow_slots;
  const int all = shared + (len + p.own_chunk - 1) / p.own_chunk, parts = (all - warp + W - 1) / W;
  auto place = [&](int j) {
    const int i = j * W + warp;
    return (long long)(i < shared ? i : i - shared + p.prefix_slots) * rows + row;
  };
  wait_before();  // the lengths are inputs, what follows is not
  float top = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < parts; i0 += 32) {
    const int n = min(32, parts - i0);
    const float2 ml = lane < n ? __ldcg(p.part_ml + place(i0 + lane)) : make_float2(-INFINITY, 0.f);
    float next = ml.x;
#pragma unroll
    for (int x = 16; x; x >>= 1) next = fmaxf(next, __shfl_xor_sync(~0u, next, x));
    next = fmaxf(next, top);
    const float base = next == -INFINITY ? 0.f : next, old = exp2_approx(top - base);
    top = next;
    // an item without keys has no o
    const float f = ml.y == 0.f ? 0.f : exp2_approx(ml.x - base);
    float sum = f == 0.f ? 0.f * ml.y : f * ml.y;
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(~0u, sum, x);
    l = l * old + sum;
    o.x *= old, o.y *= old, o.z *= old, o.w *= old;
    const unsigned holds = __ballot_sync(~0u, lane < n && ml.y != 0.f);
#pragma unroll 8
    for (int i = 0; i < n; i += AT_ONCE) {
      const int k = i + sub;
      const float fk = __shfl_sync(~0u, f, k & 31);
      if (k < n && (holds >> k & 1)) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + place(i0 + k) * D) + piece);
        o.x += fk * x.x, o.y += fk * x.y, o.z += fk * x.z, o.w += fk * x.w;
      }
    }
  }
  if (AT_ONCE == 2) {
    o.x += __shfl_xor_sync(~0u, o.x, 16), o.y += __shfl_xor_sync(~0u, o.y, 16);
    o.z += __shfl_xor_sync(~0u, o.z, 16), o.w += __shfl_xor_sync(~0u, o.w, 16);
  }
  if (W > 1) {
    __shared__ float4 warp_o[W][LANES];
    __shared__ float2 warp_ml[W];
    if (sub == 0) warp_o[warp][piece] = o;
    if (lane == 0) warp_ml[warp] = make_float2(top, l);
    __syncthreads();
    if (warp > 0) return;
    for (int w = 0; w < W; ++w) top = fmaxf(top, warp_ml[w].x);
    const float base = top == -INFINITY ? 0.f : top;
    l = 0.f, o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = exp2_approx(warp_ml[w].x - base);
      const float4 x = warp_o[w][piece];
      l += f * warp_ml[w].y;
      o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no key: zeros
  if (sub == 0)
    *reinterpret_cast<uint2*>(p.out + b * p.out_batch + h * p.out_head + piece * 4) =
        make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
  if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (top == -INFINITY ? 0.f : top) * 0.6931471805599453f + logf(l);
}

int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// How the keys are split.
struct Plan {
  bool many;  // prefix on the tensor core
  int prefix_chunk, prefix_slots, own_chunk, own_slots;
  int wide_blocks, narrow_rows, wide_splits, wide_tiles, narrow_splits, narrow_tiles;
  long long part_bytes;
};

// many_rows takes the prefix from here on: more than two tiles of 8 query rows per KV head, and that many elements of
// K that few_rows would go through, its tiles of 8 rows times the prefix. Times of whole calls in us, few against many,
// heads of 128: 16 KV heads, bf16, 32768 rows of prefix: 70 / 72 at 16 query rows, 88 / 74 at 24; 4096 rows: 33 / 31 at
// 32 (2^25 elements), 39 / 35 at 48. 8 KV heads, 8192 rows, 32 query rows (2^25): 27 / 27 bf16, 35 / 31 int8; 512 rows:
// 22 / 31 at 256 query rows, 61 / 49 at 1024. int8, 16 KV heads, 32768 rows: 93 / 96 at 16 query rows, 127 / 97 at 24.
constexpr int kManyFrom = 17;
constexpr long long kManyElements = 1ll << 25;

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
  if (a->prefix_len > 1 << 30 || a->own_capacity > 1 << 30)
    return fail(EK_E_UNSUPPORTED, "more than %d rows", 1 << 30);
  if ((long long)a->batch * a->q_heads > (1 << 22))
    return fail(EK_E_UNSUPPORTED, "batch * q_heads beyond %d", 1 << 22);
  int sms = 0;
  cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, a->device);
  if (e != cudaSuccess) return ek::cuda_fail(e, "cudaDeviceGetAttribute");
  std::memset(&pl, 0, sizeof(pl));
  const int group = a->q_heads / a->kv_heads, rows = a->batch * group;
  // few_rows: items that fill the GPU once: four blocks fit an SM, three with bf16 rows of 128. One sequence, 32 query
  // heads of 128, 32768 rows of prefix, for 1, 2, 3, 4 and 6 items per SM: bf16 47, 39, 39, 44, 43 us, int8 61, 43, 39,
  // 37, 43 us.
  const bool i8 = (a->prefix_len > 0 ? a->prefix_k.scales : a->own_k.scales) != nullptr;
  const long long want = (a->head_dim == 128 && !i8 ? 3ll : 4ll) * sms;
  auto chunk = [&](long long len, long long splits) {
    const long long c = div_up(div_up(len, splits), 64) * 64ll;
    return (int)(c < 64 ? 64 : c);
  };
  const long long tiles = (long long)div_up(rows, 8) * a->kv_heads;
  pl.many = rows >= kManyFrom && tiles * a->prefix_len * a->head_dim >= kManyElements;
  // The blocks are dealt to prefix and own rows by their keys, so that all run at once: 16 sequences over 2048 shared
  // rows and up to 256 own 16.4 us, 18.4 if each part fills the GPU; 11 over 2808 and up to 264 18.4 and 22.5.
  const long long own = (long long)a->batch * div_up(group, 8) * a->kv_heads;
  const long long prefix_keys = pl.many ? 0 : tiles * a->prefix_len, own_keys = own * a->max_own_len;
  const long long for_own = own_keys > 0 ? want * own_keys / (prefix_keys + own_keys) : 0, for_prefix = want - for_own;
  pl.own_chunk = chunk(a->max_own_len, for_own > own ? div_up(for_own, own) : 1);  // of unequal lengths: rather more
  pl.own_slots = div_up(a->max_own_len, pl.own_chunk);
  if (!pl.many) {
    pl.prefix_chunk = chunk(a->prefix_len, tiles > 0 && tiles < for_prefix ? for_prefix / tiles : 1);
    pl.prefix_slots = div_up(a->prefix_len, pl.prefix_chunk);
  } else {
    // Blocks of 256 rows (wide), and one of the rest, which is narrow up to 128 rows. A wide tile costs two
    // units, a narrow one one; the smallest share of units whose items all run at once.
    pl.wide_blocks = rows / 256 + (rows % 256 > 128);
    pl.narrow_rows = rows % 256 > 128 ? 0 : rows % 256;
    const long long keys = div_up(a->prefix_len, 128), narrow = pl.narrow_rows ? 1 : 0;
    const long long units = (2ll * pl.wide_blocks + narrow) * keys * a->kv_heads;
    const long long blocks = (pl.wide_blocks + narrow) * a->kv_heads;
    const long long most = blocks <= sms ? sms : 4 * blocks;
    long long share = div_up(units, most);
    for (;; ++share) {
      pl.wide_tiles = div_up(share, 2), pl.narrow_tiles = (int)share;
      pl.wide_splits = div_up(keys, pl.wide_tiles), pl.narrow_splits = div_up(keys, pl.narrow_tiles);
      if (((long long)pl.wide_blocks * pl.wide_splits + narrow * pl.narrow_splits) * a->kv_heads <= most) break;
      if (share >= 2 * keys) break;
    }
    const int wide_slots = pl.wide_blocks ? pl.wide_splits : 0, narrow_slots = narrow ? 2 * pl.narrow_splits : 0;
    pl.prefix_slots = wide_slots > narrow_slots ? wide_slots : narrow_slots;
  }
  pl.part_bytes = (long long)(pl.prefix_slots + pl.own_slots) * a->batch * a->q_heads * (a->head_dim * 4 + 8);
  return EK_SUCCESS;
}

// Map of rows [batch][rows][heads][d]: copies of `box` rows of one head, 64 bf16 values (128-byte swizzle) or `d` codes
// wide. Rows past the end read as zeros.
int encode_rows(RowMap& m, const EkKvTensor& t, int batch, int rows, int heads, int d, bool i8, int box,
                CUtensorMapSwizzle swizzle) {
  ek::EncodeTiledFn enc = ek::get_encoder();
  if (!enc) return ek::fail(EK_E_CUDA, "cuTensorMapEncodeTiled is unavailable");
  const long long size = i8 ? 1 : 2;
  struct Dim {
    long long n, stride;
    int8_t* place;
    bool rows;
  } dims[3] = {{heads, t.stride_head * size, &m.head, false},
               {rows, t.stride_row * size, &m.row, true},
               {batch, t.stride_batch * size, &m.batch, false}};
  long long widest = d * size;
  for (Dim& x : dims) {
    if (x.n == 1 || x.stride == 0) x.n = 1, x.stride = 0;  // not there: a repeated head or sequence
    if (x.stride > widest) widest = x.stride;
  }
  for (Dim& x : dims)
    if (x.n == 1) x.stride = widest;
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2 - i; ++j)
      if (dims[j].stride > dims[j + 1].stride) {
        const Dim x = dims[j];
        dims[j] = dims[j + 1], dims[j + 1] = x;
      }
  cuuint64_t sizes[4] = {(cuuint64_t)d}, strides[3];
  cuuint32_t boxes[4] = {(cuuint32_t)(i8 ? d : 64)};
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  for (int i = 0; i < 3; ++i) {
    *dims[i].place = dims[i].n == 1 ? -1 : i;
    sizes[i + 1] = (cuuint64_t)dims[i].n, strides[i] = (cuuint64_t)dims[i].stride;
    boxes[i + 1] = dims[i].rows ? box : 1;
  }
  const CUresult r = enc(&m.map, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, t.data, sizes,
                         strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return ek::fail(EK_E_INVALID, "tensor map of K or V rows failed (CUresult %d)", (int)r);
  return EK_SUCCESS;
}

// Checks alignment and kind of K and V when there are rows, and takes their scales.
int take_rows(const EkKvTensor& k, const EkKvTensor& v, int rows, bool i8, const char* name, Scales& s) {
  using ek::fail;
  if (rows > 0) {
    const int unit = i8 ? 16 : 8;
    for (const EkKvTensor* t : {&k, &v}) {
      if (!t->data || !ek::aligned16(t->data) || t->stride_batch % unit || t->stride_row % unit || t->stride_head % unit)
        return fail(EK_E_INVALID, "%s rows must be 16-byte aligned with strides of 16 bytes", name);
      if (rows > 1 && t->stride_row == 0) return fail(EK_E_INVALID, "%s rows with a stride of 0", name);
      if ((t->scales != nullptr) != i8) return fail(EK_E_INVALID, "prefix and own rows must be of one kind");
    }
  }
  s.k = static_cast<const __nv_bfloat16*>(k.scales), s.v = static_cast<const __nv_bfloat16*>(v.scales);
  s.k_batch = k.scale_stride_batch, s.k_row = k.scale_stride_row, s.k_head = k.scale_stride_head;
  s.v_batch = v.scale_stride_batch, s.v_row = v.scale_stride_row, s.v_head = v.scale_stride_head;
  return EK_SUCCESS;
}

// Launches `kernel`; `overlap`: it may start while the launch before it in the stream still runs (once all of that
// one's blocks have passed launch_next or ended), and waits for its results itself.
template <typename P>
cudaError_t start(void (*kernel)(P), const P& p, long long blocks, int threads, int bytes, bool overlap, cudaStream_t st) {
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  cudaError_t e;
  if (bytes > 48 * 1024 &&
      (e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) != cudaSuccess)
    return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// few_rows, then many_rows beside it, then join. The first is an ordinary launch, so what ran before is done when any
// of them reads; many_rows reads nothing of few_rows and ends after it (wait_before), join waits for many_rows.
template <int D, bool I8>
cudaError_t launch(const FewParams& p, const ManyParams* many, cudaStream_t st) {
  using M = Many<D, I8>;
  static_assert(M::SMEM <= 227 * 1024 && Few<D, I8>::SMEM <= 227 * 1024, "shared memory");
  cudaError_t e;
  const long long items = (long long)p.a.prefix_slots * p.a.prefix_tiles * p.a.kv_heads +
                          (long long)p.a.own_slots * p.a.group_tiles * p.a.kv_heads * p.a.batch;
  if (items > 0 &&
      (e = start(few_rows<D, I8>, p, items, kWarps * 32 + 32, Few<D, I8>::SMEM, false, st)) != cudaSuccess)
    return e;
  if (many) {
    // The warpgroups take more registers out of those that the block is launched with. The build compares the numbers;
    // this keeps a library built in another way from waiting for good.
    cudaFuncAttributes attr;
    if ((e = cudaFuncGetAttributes(&attr, many_rows<D, I8>)) != cudaSuccess) return e;
    if (attr.numRegs != M::REGS) return cudaErrorLaunchOutOfResources;
    const int blocks = (many->wide_blocks * many->wide_splits + (many->narrow_rows ? many->narrow_splits : 0)) * p.a.kv_heads;
    if ((e = start(many_rows<D, I8>, *many, blocks, M::WARPS * 32, M::SMEM, items > 0, st)) != cudaSuccess) return e;
  }
  // Few rows of many items get a block each. Whole calls, a warp against a block per row: 32 rows 47 / 39 us (one
  // sequence, 32768 rows of prefix, D = 128), 512 rows 41 / 35, 1952 rows 86 / 84, 4096 rows 84 / 91.
  const long long rows = (long long)p.a.batch * p.a.q_heads;
  if (rows <= 2048 && p.a.prefix_slots + p.a.own_slots > 8)
    return start(join<D, kJoinWarps>, p.a, (int)rows, kJoinWarps * 32, 0, items > 0 || many, st);
  return start(join<D, 1>, p.a, div_up(rows, 4), 128, 0, items > 0 || many, st);
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
  ek::DeviceGuard g(a->device);
  const bool i8 = (a->prefix_len > 0 ? a->prefix_k.scales : a->own_k.scales) != nullptr;
  FewParams few;
  AttnParams& p = few.a;
  if ((rc = take_rows(a->prefix_k, a->prefix_v, a->prefix_len, i8, "prefix", p.prefix))) return rc;
  if ((rc = take_rows(a->own_k, a->own_v, a->max_own_len > 0 ? a->own_capacity : 0, i8, "own", p.own))) return rc;
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
  p.wide_rows = pl.wide_blocks * 256;
  p.wide_slots = pl.wide_splits;
  p.narrow_slots = pl.many ? 2 * pl.narrow_splits : pl.prefix_slots;
  p.scale_log2 = a->scale * kLog2e;
  const int d = a->head_dim;
  const CUtensorMapSwizzle wide_rows = CU_TENSOR_MAP_SWIZZLE_128B;
  const CUtensorMapSwizzle few_swizzle = i8 && d == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : wide_rows;
  auto encode = [&](RowMap& k, RowMap& v, const EkKvTensor& tk, const EkKvTensor& tv, int batch, int rows, int box,
                    CUtensorMapSwizzle swizzle) {
    const int r = encode_rows(k, tk, batch, rows, a->kv_heads, d, i8, box, swizzle);
    return r ? r : encode_rows(v, tv, batch, rows, a->kv_heads, d, i8, box, swizzle);
  };
  constexpr int kBox = Few<64, false>::BOX;
  if (a->max_own_len > 0 &&
      (rc = encode(few.own_k, few.own_v, a->own_k, a->own_v, a->batch, a->own_capacity, kBox, few_swizzle)))
    return rc;
  ManyParams m;
  if (pl.many) {
    if ((rc = encode(m.k, m.v, a->prefix_k, a->prefix_v, 1, a->prefix_len, 128, i8 ? CU_TENSOR_MAP_SWIZZLE_NONE : wide_rows)))
      return rc;
    m.a = p;
    m.rows = a->batch * p.group;
    m.wide_blocks = pl.wide_blocks, m.narrow_rows = pl.narrow_rows;
    m.wide_splits = pl.wide_splits, m.wide_tiles = pl.wide_tiles;
    m.narrow_splits = pl.narrow_splits, m.narrow_tiles = pl.narrow_tiles;
    m.q_flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    m.q_zero = p.scale_log2 == 0.f;
    m.a.scale_log2 = m.q_zero ? kLog2e : fabsf(p.scale_log2);
    p.prefix_tiles = 0;  // nothing of the prefix is left for few_rows
  } else if (a->prefix_len > 0 &&
             (rc = encode(few.prefix_k, few.prefix_v, a->prefix_k, a->prefix_v, 1, a->prefix_len, kBox, few_swizzle))) {
    return rc;
  }
  const ManyParams* many = pl.many ? &m : nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->head_dim == 64) e = i8 ? launch<64, true>(few, many, st) : launch<64, false>(few, many, st);
  else e = i8 ? launch<128, true>(few, many, st) : launch<128, false>(few, many, st);
  return e == cudaSuccess ? EK_SUCCESS : ek::cuda_fail(e, "ek_prefix_attention launch");
}

extern "C" int ek_prefix_attention_status(int device, int32_t* out, int clear) {
  if (!out) return ek::fail(EK_E_INVALID, "NULL argument");
  ek::DeviceGuard g(device);
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(out, g_attention_status, sizeof(int32_t));
  const int32_t zero = 0;
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(zero));
  return e == cudaSuccess ? EK_SUCCESS : ek::cuda_fail(e, "ek_prefix_attention_status");
}
