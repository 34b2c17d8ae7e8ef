// W8A8 integer projections (sm_100a, tcgen05 kind::i8 + TMA): the quantiser of
// activations and weights, and the product with its scales.
//
//   xs[t] = amax(x[t]) / 127,   xq[t] = round(x[t] * 127 / amax)       (per token)
//   y[t, j] = (xq[t] . wq[j]) * xs[t] * ws[j] (+ bias[j])              (int32 sums, exact)
// and for a gate_up weight y[t, j] = silu(g) * u with g, u the two halves'
// columns, in fp32 up to the one rounding to bf16.  127^2 K < 2^31 holds up to
// K = 131072, so no sum overflows.
//
// Quantiser.  A row's magnitudes are compared as integers (bf16 without its sign
// bit orders like its value, and NaN above infinity), two per instruction; a NaN
// makes the row's scale NaN, so it is not lost.
//
// Product.  A CTA computes 128 tokens x TN weight rows: one warp keeps a ring of
// {128 bytes of K} TMA boxes of both operands full (128-byte swizzle; what lies
// outside the matrices arrives as zeros, so any M, N and K work), one thread
// issues tcgen05.mma with int32 accumulators in TMEM, four warps drain finished
// tiles.  The grid is persistent and the accumulator double-buffered, so a tile's
// epilogue runs under the next tile's products.  Tokens are the MMA's rows: an
// epilogue thread owns one token, its scale is one register, the weights' scales
// are broadcast from shared memory, and gate and up columns (interleaved in groups
// of 16 rows when the weight is laid out) meet in the same thread.  TN is chosen
// per call (pick_tiling).  A decode batch loads only its own token rows; the MMA's
// other rows read whatever lies behind them in shared memory, into accumulators
// that nobody reads.  Where a call has few tiles and a long K, a cluster of up to 8
// CTAs shares a tile's K: each stages its int32 accumulators in its own shared
// memory, and each finishes its part of the tokens from all of them (integer sums:
// the order does not matter).
//
// Up to 8 tokens the product is a stream of the weights: no tensor core, no
// second launch.  Every CTA quantises the tokens for itself (they are a few KB),
// its first weights already on their way, and a warp takes two weight rows at a
// time (gate and up of one column) with dp4a.
//
// One B200, captured graphs, bf16 tokens, weights from HBM (from L2): 1 x 2048 x 2048 with
// bias 4.2 us (4.0); 64 x 12288 x 2048 with SwiGLU 10.4 (8.0), of codes 7.9; 64 x 2048 x
// 6144 9.1 (7.9), of codes 7.1; 4613 x 2048 x 6144 56, of which the product 40 (2.9 POP/s,
// tensor pipe 66 % busy).  One call among others, weights from L2: 5.0, 8.9 and 65 us for
// the first, second and last.
#include <algorithm>
#include <cstdint>
#include <mutex>

#include "common.cuh"
#include "gemm_common.cuh"
#include "tcgen05.cuh"

namespace nqt {
namespace {

using namespace gemm_detail;

// ------------------------------------------------------------------ quantiser
// The rule of a row whose largest |bf16| bits are `mx`: scale, factor and the codes of its values.  A value times the
// factor plus 1.5 2^23 is the rounded code in the sum's low bits: one rounding, no conversion (1024 x 6144
// from L2: 3.6 us; with a rounding and a conversion each 5.0).
//
// The codes are exactly round(x 127 / amax), ties to even, because the factor 127 / amax is rounded up.  Write x and amax
// as 8-bit integers times powers of two: a quotient q that is no tie is q / (254 255) or more away from one, and the factor
// moves it by 2^-23 q.  A tie 254 x = (2 j + 1) amax needs 127 to divide 2 j + 1, which is then 127, or amax's integer,
// and then the factor is a power of two.  So the only tie with an inexact factor is x = amax / 2, 63.5, whose even
// neighbour 64 is the upper one.
struct RowRule {
  float s, f, amax;
  bool plain;  // else 127 / amax overflows (a division each), or the row holds an infinity or a NaN
  __device__ __forceinline__ explicit RowRule(uint32_t mx) {
    amax = __uint_as_float(mx << 16);
    s = __fdiv_rn(amax, 127.f);
    f = amax == 0.f ? 0.f : __fdiv_rn(127.f, amax);
    if (fmaf(f, amax, -127.f) < 0.f) f = __uint_as_float(__float_as_uint(f) + 1u);  // up
    plain = f <= 3.0e38f && mx < 0x7f80u;
  }
  __device__ __forceinline__ uint32_t odd(uint32_t bf16_bits) const {
    const float v = __uint_as_float(bf16_bits << 16);
    const float t = f > 3.0e38f ? __fdiv_rn(v * 127.f, amax) : v * f;
    return static_cast<uint32_t>(__float2int_rn(t)) & 0xffu;
  }
  __device__ __forceinline__ uint32_t sum(uint32_t f32_bits) const {
    return __float_as_uint(fmaf(__uint_as_float(f32_bits), f, 12582912.f));
  }
  // four bf16 -> four codes
  __device__ __forceinline__ uint32_t codes(uint32_t a, uint32_t b) const {
    if (plain)
      return __byte_perm(__byte_perm(sum(a << 16), sum(a & 0xffff0000u), 0x0040),
                         __byte_perm(sum(b << 16), sum(b & 0xffff0000u), 0x0040), 0x5410);
    return odd(a & 0xffffu) | (odd(a >> 16) << 8) | (odd(b & 0xffffu) << 16) | (odd(b >> 16) << 24);
  }
  __device__ __forceinline__ uint2 codes(uint4 w) const { return make_uint2(codes(w.x, w.y), codes(w.z, w.w)); }
};

__device__ __forceinline__ uint32_t magnitude2(uint4 v, uint32_t m2) {
  m2 = __vmaxu2(m2, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu));
  return __vmaxu2(m2, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
}

// Vector v (8 elements) of a row of k; elements behind the row are zeros.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* src, int v, int k) {
  if (VEC) return *reinterpret_cast<const uint4*>(src + v * 8);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  const uint16_t* e = reinterpret_cast<const uint16_t*>(src) + v * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (v * 8 + i < k) w[i / 2] |= static_cast<uint32_t>(e[i]) << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One row by TPR threads; 4 or 6 vectors of 8 elements per thread stay in registers between the two passes, longer
// rows are read again (from L2).
template <int TPR, bool VEC>
__global__ void __launch_bounds__(256) int8_quantize_rows_kernel(const __nv_bfloat16* x, int64_t ldx, int m, int k,
                                                                 int8_t* q, int64_t ldq, float* scale) {
  constexpr int kRows = 256 / TPR;
  constexpr int kKeep = TPR == 128 ? 6 : 4;
  __shared__ uint32_t s_max[8];
  // Waiting first, then letting the product start: what came before this kernel has finished by then, so the product
  // may read its weights at once.
  grid_dependency_wait();
  grid_dependents_launch();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  const int lt = threadIdx.x % TPR;
  const bool live = row < m;
  const __nv_bfloat16* src = x + (live ? row : 0) * ldx;
  const int vecs = live ? (k + 7) / 8 : 0;

  auto load = [&](int v) -> uint4 { return load8<VEC>(src, v, k); };
  uint4 keep[kKeep];
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < kKeep; ++i) {
    const int v = lt + i * TPR;
    keep[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < vecs) keep[i] = load(v);
    m2 = magnitude2(keep[i], m2);
  }
  for (int v = lt + kKeep * TPR; v < vecs; v += TPR) m2 = magnitude2(load(v), m2);
  uint32_t mx = max(m2 & 0xffffu, m2 >> 16);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(kFull, mx, o));
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = mx;
    __syncthreads();
    const int w0 = threadIdx.x / TPR * (TPR / 32);
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) mx = max(mx, s_max[w0 + w]);
  }
  if (!live) return;
  const RowRule rule(mx);
  if (lt == 0) scale[row] = rule.s;
  auto store = [&](int v, uint4 w) {
    const uint2 c = rule.codes(w);
    int8_t* dst = q + row * ldq + v * 8;
    if (VEC) {
      *reinterpret_cast<uint2*>(dst) = c;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v * 8 + i < k) dst[i] = static_cast<int8_t>(((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 0xffu);
    }
  };
#pragma unroll
  for (int i = 0; i < kKeep; ++i)
    if (lt + i * TPR < vecs) store(lt + i * TPR, keep[i]);
  for (int v = lt + kKeep * TPR; v < vecs; v += TPR) store(v, load(v));
}

// ------------------------------------------------------------------ product
constexpr int kTileM = 128;   // tokens per tile (MMA M)
constexpr int kBlockK = 128;  // bytes of K per box, of which a stage holds one or two of each operand
constexpr int kThreads = 6 * 32;

enum Epilogue : int { kPlain = 0, kBias = 1, kSiluMul = 2 };  // the numbering of nqt_gemm_bf16

struct Int8Args {
  const float *xscale, *wscale;
  const __nv_bfloat16* bias;
  __nv_bfloat16* y;
  int64_t ldy;
  int32_t* status;
  int m, n, cols, kb;  // cols: output columns; kb: K blocks (of SUB boxes)
  int m_tiles, tiles;
  int epilogue;
  int early;  // the weights may be read before the previous kernel has finished
  int vec16;  // y rows allow 16-byte stores
  int tn, stages;
  int a_bytes;  // of a box of tokens: a multiple of 8 rows, up to 128
  int split;    // CTAs of a cluster that share a tile's K
  uint32_t tmem_cols;
};

constexpr int kMaxTN = 256, kMaxStages8 = 16;
constexpr int kTail8 = 2 * kMaxTN * 4 * 2 + (2 * kMaxStages8 + 4) * 8 + 64;  // scales, biases, barriers, flags
constexpr int kSmem8 = 227 * 1024;
constexpr int kRing8 = kSmem8 - kTail8 - 1024;  // 1024: the ring starts on a multiple of that
constexpr int kMaxSplit = 8;

// Bytes from one token's staged accumulators to the next's: 16 more than they need, against bank conflicts.
__host__ __device__ constexpr int split_pitch(int tn) { return tn * 4 + 16; }

__device__ __forceinline__ void mma_i8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor, kind::i8: s32 accumulate (bits 4-5 = 2), s8 A and B (bits 7-9 and 10-12 = 1), K-major.
__host__ __device__ constexpr uint32_t idesc_s8_s32(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(c0), "r"(c1)
      : "memory");
}

__device__ __forceinline__ int4 ld_cluster_i4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Four columns' sums over the cluster's partial accumulators at `addr` (the same place in every CTA), scaled.
__device__ __forceinline__ float4 join_4(uint32_t addr, int split, float sx, const float* sw) {
  int4 s = make_int4(0, 0, 0, 0);
#pragma unroll 4
  for (int c = 0; c < split; ++c) {
    const int4 v = ld_cluster_i4(map_rank(addr, c));
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  return make_float4(static_cast<float>(s.x) * (sx * sw[0]), static_cast<float>(s.y) * (sx * sw[1]),
                     static_cast<float>(s.z) * (sx * sw[2]), static_cast<float>(s.w) * (sx * sw[3]));
}

// The split tile's epilogue: this CTA's share of the token rows, from the staged accumulators of all the cluster's CTAs.
__device__ __forceinline__ void join_split(const Int8Args& a, const uint8_t* stage, int pitch, int rank, int m0, int n0,
                                           const float* sw, const float* sb) {
  const int rows = a.m - m0 < kTileM ? a.m - m0 : kTileM;
  const int r0 = rows * rank / a.split, r1 = rows * (rank + 1) / a.split;
  const bool silu = a.epilogue == kSiluMul;
  const int quads = silu ? a.tn / 8 : a.tn / 4;  // of output columns
  const int count = (r1 - r0) * quads;
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const int row = r0 + i / quads, q = i % quads;
    const int c = silu ? q / 4 * 32 + q % 4 * 4 : 4 * q;  // accumulator column
    const int col = silu ? n0 / 2 + 4 * q : n0 + c;
    if (col >= a.cols) continue;
    const float sx = a.xscale[m0 + row];
    const uint32_t addr = smem_addr(stage + row * pitch + c * 4);
    float4 v = join_4(addr, a.split, sx, sw + c);
    if (silu) {
      const float4 u = join_4(addr + 64, a.split, sx, sw + c + 16);
      v = make_float4(silu_mul(v.x, u.x), silu_mul(v.y, u.y), silu_mul(v.z, u.z), silu_mul(v.w, u.w));
    } else if (a.epilogue == kBias) {
      v = make_float4(v.x + sb[c], v.y + sb[c + 1], v.z + sb[c + 2], v.w + sb[c + 3]);
    }
    __nv_bfloat16* y = a.y + static_cast<int64_t>(m0 + row) * a.ldy + col;
    if (a.vec16 && col + 4 <= a.cols) {
      *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    } else {
      y[0] = __float2bfloat16_rn(v.x);
      if (col + 1 < a.cols) y[1] = __float2bfloat16_rn(v.y);
      if (col + 2 < a.cols) y[2] = __float2bfloat16_rn(v.z);
      if (col + 3 < a.cols) y[3] = __float2bfloat16_rn(v.w);
    }
  }
}

// 32 accumulators of one token -> outputs, stored at column `col` of row y (plain, bias) or col / 2 (gate and up
// columns in groups of 16).  `sw`, `sb`: the columns' scales and biases in shared memory; `width`: columns left in
// the tile.
__device__ __forceinline__ void finish_32(const Int8Args& a, const uint32_t (&r)[32], float sx, const float* sw,
                                          const float* sb, __nv_bfloat16* yrow, int col, int width) {
  float v[32];
#pragma unroll
  for (int e = 0; e < 32; e += 4) {
    const float4 w = *reinterpret_cast<const float4*>(sw + e);
    v[e] = static_cast<float>(static_cast<int32_t>(r[e])) * (sx * w.x);
    v[e + 1] = static_cast<float>(static_cast<int32_t>(r[e + 1])) * (sx * w.y);
    v[e + 2] = static_cast<float>(static_cast<int32_t>(r[e + 2])) * (sx * w.z);
    v[e + 3] = static_cast<float>(static_cast<int32_t>(r[e + 3])) * (sx * w.w);
  }
  int count = width < 32 ? width : 32, out0 = col;
  if (a.epilogue == kBias) {
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] += sb[e];
  } else if (a.epilogue == kSiluMul) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = silu_mul(v[e], v[e + 16]);
    count = 16;
    out0 = col / 2;
  }
  const int left = a.cols - out0;
  if (a.vec16 && left >= count && count % 8 == 0) {
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
      if (e >= count) break;
      *reinterpret_cast<uint4*>(yrow + out0 + e) =
          make_uint4(pack_bf16x2(v[e], v[e + 1]), pack_bf16x2(v[e + 2], v[e + 3]), pack_bf16x2(v[e + 4], v[e + 5]),
                     pack_bf16x2(v[e + 6], v[e + 7]));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e < count && e < left) yrow[out0 + e] = __float2bfloat16_rn(v[e]);
  }
}

// SPLIT: the grid has one cluster of a.split CTAs for each tile, each with its part of K; else it is persistent.
template <bool SPLIT, int SUB>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_int8_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                     const __grid_constant__ Int8Args a) {
  const int ST = a.stages, TN = a.tn;
  const int a_bytes = a.a_bytes, b_bytes = TN * kBlockK, stage_bytes = (a_bytes + b_bytes) * SUB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  // behind the ring, and at least 128 token rows behind its last stage's start
  float* s_sw = reinterpret_cast<float*>(smem_raw + kSmem8 - kTail8);  // [2][TN] scales, then [2][TN] biases
  float* s_sb = s_sw + 2 * kMaxTN;
  uint64_t* full = reinterpret_cast<uint64_t*>(s_sb + 2 * kMaxTN);
  uint64_t* empty = full + kMaxStages8;
  uint64_t* accf = empty + kMaxStages8;  // [2] accumulator complete
  uint64_t* acce = accf + 2;             // [2] accumulator read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acce + 2);
  volatile int* s_issued = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* s_consumed = s_issued + 1;
  volatile int* s_ready = s_consumed + 1;

  const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
  const int rank = SPLIT ? static_cast<int>(cluster_rank()) : 0;
  const int first = SPLIT ? static_cast<int>(blockIdx.x) / a.split : static_cast<int>(blockIdx.x);
  const int kb0 = SPLIT ? a.kb * rank / a.split : 0, kb1 = SPLIT ? a.kb * (rank + 1) / a.split : a.kb;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accf[b], 1);
      mbar_init(&acce[b], 4);
    }
    fence_barrier_init();
    *s_issued = 0;
    *s_consumed = 0;
    prefetch_tensormap(&xmap);
    prefetch_tensormap(&wmap);
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, a.tmem_cols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependents_launch();

  // The producer's and the issuer's loops are run by whole warps, and one elected lane issues: operands and descriptors
  // then stay in uniform registers.  (One lane's own loop cost some 20 clocks more for each product.)
  if (warp == 0) {
    {
      const bool lead = tc::elect_one();
      int it = 0, s = 0;  // K block, its stage and the stage's turn (divisions by ST would cost more than a block)
      uint32_t phase = 0;
      bool ok = true;
      // the first stages' weights do not depend on the previous kernel when the caller says so
      int ahead = 0;
      if (a.early && first < a.tiles) {
        const int n0 = first / a.m_tiles * TN;
        ahead = kb1 - kb0 < ST ? kb1 - kb0 : ST;
        for (int i = 0; i < ahead; ++i) {
          if (!lead) continue;
          mbar_arrive_expect_tx(&full[i], stage_bytes);
#pragma unroll
          for (int u = 0; u < SUB; ++u)
            tma_load_2d(smem + i * stage_bytes + a_bytes * SUB + u * b_bytes, &wmap, &full[i],
                        ((kb0 + i) * SUB + u) * kBlockK, n0);
        }
      }
      grid_dependency_wait();
      for (int tile = first; tile < a.tiles && ok; tile += gridDim.x) {
        const int m0 = tile % a.m_tiles * kTileM, n0 = tile / a.m_tiles * TN;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          if (it >= ST && !__all_sync(kFull, mbar_wait(&empty[s], phase ^ 1u, a.status))) {
            ok = false;
            break;
          }
          if (lead) {
            uint8_t* st = smem + s * stage_bytes;
            if (it >= ahead) {
              mbar_arrive_expect_tx(&full[s], stage_bytes);
#pragma unroll
              for (int u = 0; u < SUB; ++u)
                tma_load_2d(st + a_bytes * SUB + u * b_bytes, &wmap, &full[s], (kb * SUB + u) * kBlockK, n0);
            }
#pragma unroll
            for (int u = 0; u < SUB; ++u)
              tma_load_2d(st + u * a_bytes, &xmap, &full[s], (kb * SUB + u) * kBlockK, m0);
          }
          if (++s == ST) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
      if (lane == 0) *s_issued = it;
    }
  } else if (warp == 1) {
    {
      const bool lead = tc::elect_one();
      const uint32_t idesc = idesc_s8_s32(kTileM, TN);
      const uint64_t a_desc = tc::smem_desc_sw128(smem_addr(smem), 16, 1024);
      const uint64_t b_desc = tc::smem_desc_sw128(smem_addr(smem + a_bytes * SUB), 16, 1024);
      int it = 0, s = 0, t = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < a.tiles && ok; tile += gridDim.x, ++t) {
        const int buf = t & 1;
        if (t >= 2 && !__all_sync(kFull, mbar_wait(&acce[buf], ((t >> 1) - 1) & 1, a.status))) break;
        tc::fence_after_sync();
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
          if (!__all_sync(kFull, mbar_wait(&full[s], phase, a.status))) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          if (lead) {
            const uint32_t off = static_cast<uint32_t>(s * stage_bytes) >> 4;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              const uint64_t ad = a_desc + off + u * (a_bytes >> 4), bd = b_desc + off + u * (b_bytes >> 4);
#pragma unroll
              for (int kk = 0; kk < kBlockK / 32; ++kk)
                mma_i8_ss(tmem + buf * TN, ad + kk * 2, bd + kk * 2, idesc, kb > kb0 || u || kk ? 1u : 0u);
            }
            tc::commit(&empty[s]);
          }
          if (++s == ST) {
            s = 0;
            phase ^= 1u;
          }
        }
        if (ok && lead) tc::commit(&accf[buf]);
      }
      if (lane == 0) *s_consumed = it;
    }
  } else {
    const int quarter = warp & 3;
    const int et = threadIdx.x - 64;
    grid_dependency_wait();  // the tokens' scales, and y, which the previous kernel may still read
    int t = 0;
    for (int tile = first; tile < a.tiles; tile += gridDim.x, ++t) {
      const int buf = t & 1;
      const int m0 = tile % a.m_tiles * kTileM, n0 = tile / a.m_tiles * TN;
      float* sw = s_sw + buf * kMaxTN;
      float* sb = s_sb + buf * kMaxTN;
      for (int i = et; i < TN; i += 128) {
        sw[i] = n0 + i < a.n ? __ldg(a.wscale + n0 + i) : 0.f;
        if (a.epilogue == kBias) sb[i] = n0 + i < a.n ? __bfloat162float(a.bias[n0 + i]) : 0.f;
      }
      const int tok = m0 + quarter * 32 + lane;
      const float sx = tok < a.m ? a.xscale[tok] : 0.f;
      // One warp polls for the accumulator and the others wait in the barrier, which costs no issue slots: polling
      // warps slow the thread that issues the products.  Also: all are done with this buffer's scales of two tiles ago.
      if (warp == 2) {
        const bool ok = mbar_wait(&accf[buf], (t >> 1) & 1, a.status);
        if (lane == 0) *s_ready = ok ? 1 : 0;
      }
      epi_bar();
      if (!*s_ready) break;
      tc::fence_after_sync();
      const uint32_t src = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + buf * TN;
      if (SPLIT) {  // the products have read the ring: it takes the accumulators now
        if (m0 + quarter * 32 < a.m) {
#pragma unroll 1
          for (int c = 0; c < TN; c += 32) {
            uint32_t r[32];
            tc::ld_32x32b_x32(src + c, r);
            tc::wait_ld();
            uint8_t* dst = smem + (quarter * 32 + lane) * split_pitch(TN) + c * 4;
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (c + e < TN && tok < a.m) *reinterpret_cast<uint4*>(dst + e * 4) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
          }
        }
        break;
      }
      __nv_bfloat16* yrow = a.y + static_cast<int64_t>(tok) * a.ldy;
      const bool live_warp = m0 + quarter * 32 < a.m;
#pragma unroll 1
      for (int c = 0; c < TN; c += 32) {
        uint32_t r[32];
        if (live_warp) {
          tc::ld_32x32b_x32(src + c, r);
          tc::wait_ld();
        }
        if (c + 32 >= TN) {
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acce[buf]);
        }
        if (tok < a.m && n0 + c < a.n) finish_32(a, r, sx, sw + c, sb + c, yrow, n0 + c, TN - c);
      }
    }
  }
  tc::fence_before_sync();
  if (SPLIT) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    join_split(a, smem, split_pitch(TN), rank, first % a.m_tiles * kTileM, first / a.m_tiles * TN, s_sw, s_sb);
    __syncwarp();
    cluster_arrive();  // nobody's shared memory goes away while it is read
    cluster_wait();
  }
  __syncthreads();
  if (threadIdx.x == 0)  // after a wait that gave up: copies still in flight land before the CTA leaves
    for (int i = *s_consumed; i < *s_issued; ++i) mbar_wait(&full[i % ST], (i / ST) & 1, a.status);
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, a.tmem_cols);
  }
}

// An int8 matrix [rows, k] (row pitch ld bytes) in boxes of {128 bytes, box_rows}, 128-byte swizzle, zeros outside.
int encode_i8(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  auto encode = get_encode();
  if (encode == nullptr) return NQT_ERR_CUDA;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
  cuuint32_t box[2] = {kBlockK, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? NQT_OK : NQT_ERR_CUDA;
}

// ------------------------------------------------------------------ few tokens
constexpr int kGemvMaxM = 8;
constexpr int kGemvSmem = 96 * 1024;  // codes of the tokens

struct GemvArgs {
  const __nv_bfloat16* x;  // bf16 rows, or null: codes
  const int8_t* xq;
  int64_t ldx, ldxq;
  const float* xscale;
  const int8_t* w;
  int64_t ldw;
  const float* wscale;
  const __nv_bfloat16* bias;
  __nv_bfloat16* y;
  int64_t ldy;
  int m, n, cols, k, kpad;  // kpad: bytes of a token's codes in shared memory, a multiple of 16
  int epilogue;
  int xvec;  // x rows allow 16-byte loads (and k is a multiple of 8)
};

// 16 weights of a row from byte 16 c; bytes behind k are not read (the row may end there) and count as zeros.
__device__ __forceinline__ uint4 load_w16(const int8_t* row, int c, int k) {
  if (c * 16 + 16 <= k) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(row + c * 16));
    return v;
  }
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (c * 16 + i < k) w[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(row[c * 16 + i])) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// M: token slots, a power of two >= m.  A warp takes pairs of weight rows: neighbours, or a gate row and its up row.
template <int M>
__global__ void __launch_bounds__(256, 2) gemv_int8_kernel(const __grid_constant__ GemvArgs a) {
  extern __shared__ __align__(16) uint8_t s_codes[];  // [M][kpad]
  __shared__ uint32_t s_max[8];
  __shared__ float s_scale[M];
  constexpr int kAhead = 4;  // 16-byte chunks of each row in flight
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = (a.k + 15) / 16;
  const int pairs = (a.n + 1) / 2;
  const bool silu = a.epilogue == kSiluMul;
  // rows of pair i: gate_up: groups of 16 gate and 16 up rows
  auto row_of = [&](int i, int h) -> int { return silu ? i / 16 * 32 + h * 16 + i % 16 : 2 * i + h; };
  auto weights = [&](int i, int c0, uint4 (&w)[2][kAhead]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = row_of(i, h);
      const int8_t* p = a.w + static_cast<int64_t>(r < a.n ? r : 0) * a.ldw;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int c = c0 + u * 32 + lane;
        w[h][u] = make_uint4(0u, 0u, 0u, 0u);
        if (c < chunks && i < pairs) w[h][u] = load_w16(p, c, a.k);
      }
    }
  };
  int pair = blockIdx.x * 8 + warp;
  uint4 w[2][kAhead];
  grid_dependency_wait();
  weights(pair, 0, w);
  grid_dependents_launch();

  // the tokens' codes: M rows by 256 / M threads each (codes of absent rows and behind k are zeros)
  {
    constexpr int TPR = 256 / M;
    const int t = threadIdx.x / TPR, lt = threadIdx.x % TPR;
    uint8_t* dst = s_codes + t * a.kpad;
    if (a.x != nullptr) {
      const __nv_bfloat16* src = a.x + static_cast<int64_t>(t < a.m ? t : 0) * a.ldx;
      const int vecs = (a.k + 7) / 8;
      auto load = [&](int v) -> uint4 { return a.xvec ? load8<true>(src, v, a.k) : load8<false>(src, v, a.k); };
      constexpr int kKeep = 4;
      uint4 keep[kKeep];
      uint32_t m2 = 0;
#pragma unroll
      for (int i = 0; i < kKeep; ++i) {
        keep[i] = make_uint4(0u, 0u, 0u, 0u);
        if (lt + i * TPR < vecs) keep[i] = load(lt + i * TPR);
        m2 = magnitude2(keep[i], m2);
      }
      for (int v = lt + kKeep * TPR; v < vecs; v += TPR) m2 = magnitude2(load(v), m2);
      uint32_t mx = max(m2 & 0xffffu, m2 >> 16);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(kFull, mx, o));
      if (TPR > 32) {
        if (lane == 0) s_max[warp] = mx;
        __syncthreads();
        const int w0 = t * (TPR / 32);
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) mx = max(mx, s_max[w0 + i]);
      }
      const RowRule rule(mx);
      if (lt == 0) s_scale[t] = rule.s;
#pragma unroll
      for (int i = 0; i < kKeep; ++i)
        if (lt + i * TPR < vecs) *reinterpret_cast<uint2*>(dst + (lt + i * TPR) * 8) = rule.codes(keep[i]);
      for (int v = lt + kKeep * TPR; v < vecs; v += TPR) *reinterpret_cast<uint2*>(dst + v * 8) = rule.codes(load(v));
      for (int v = vecs + lt; v < a.kpad / 8; v += TPR) *reinterpret_cast<uint2*>(dst + v * 8) = make_uint2(0u, 0u);
    } else {
      const int8_t* src = a.xq + static_cast<int64_t>(t < a.m ? t : 0) * a.ldxq;
      for (int c = lt; c < a.kpad / 16; c += TPR) *reinterpret_cast<uint4*>(dst + c * 16) = load_w16(src, c, a.k);
      if (lt == 0) s_scale[t] = t < a.m ? a.xscale[t] : 0.f;
    }
  }
  __syncthreads();

  for (; pair < pairs; pair += gridDim.x * 8) {
    int acc[2][M];
#pragma unroll
    for (int t = 0; t < M; ++t) acc[0][t] = acc[1][t] = 0;
    for (int c0 = 0; c0 < chunks; c0 += 32 * kAhead) {
      uint4 cur[2][kAhead];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < kAhead; ++u) cur[h][u] = w[h][u];
      // the next weights: of this pair, or the first of the warp's next
      if (c0 + 32 * kAhead < chunks) weights(pair, c0 + 32 * kAhead, w);
      else weights(pair + gridDim.x * 8, 0, w);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int c = c0 + u * 32 + lane;
        if (c < chunks) {
#pragma unroll
          for (int t = 0; t < M; ++t) {
            const uint4 x = *reinterpret_cast<const uint4*>(s_codes + t * a.kpad + c * 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              int v = acc[h][t];
              v = __dp4a(static_cast<int>(cur[h][u].x), static_cast<int>(x.x), v);
              v = __dp4a(static_cast<int>(cur[h][u].y), static_cast<int>(x.y), v);
              v = __dp4a(static_cast<int>(cur[h][u].z), static_cast<int>(x.z), v);
              acc[h][t] = __dp4a(static_cast<int>(cur[h][u].w), static_cast<int>(x.w), v);
            }
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < M; ++t) acc[h][t] = __reduce_add_sync(kFull, acc[h][t]);
    // lane t finishes token t
    int v0 = acc[0][0], v1 = acc[1][0];
#pragma unroll
    for (int t = 1; t < M; ++t)
      if (lane == t) {
        v0 = acc[0][t];
        v1 = acc[1][t];
      }
    if (lane < a.m) {
      const int r0 = row_of(pair, 0), r1 = row_of(pair, 1);
      const float sx = s_scale[lane];
      float y0 = static_cast<float>(v0) * (sx * a.wscale[r0]);
      float y1 = r1 < a.n ? static_cast<float>(v1) * (sx * a.wscale[r1]) : 0.f;
      __nv_bfloat16* yrow = a.y + lane * a.ldy;
      if (silu) {
        const int col = pair / 16 * 16 + pair % 16;
        if (col < a.cols) yrow[col] = __float2bfloat16_rn(silu_mul(y0, y1));
      } else {
        if (a.epilogue == kBias) {
          y0 += __bfloat162float(a.bias[r0]);
          if (r1 < a.n) y1 += __bfloat162float(a.bias[r1]);
        }
        yrow[r0] = __float2bfloat16_rn(y0);
        if (r1 < a.n) yrow[r1] = __float2bfloat16_rn(y1);
      }
    }
  }
}

template <int M>
int launch_gemv(const GemvArgs& a, cudaStream_t s) {
  static DeviceOnce once;
  once([] {
    cudaFuncSetAttribute(gemv_int8_kernel<M>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemvSmem);
  });
  const int pairs = (a.n + 1) / 2;
  const int most = num_sms() * 2;  // resident at once: a warp goes on to its next pair
  const int grid = (pairs + 7) / 8 < most ? (pairs + 7) / 8 : most;
  const cudaError_t err = launch_pdl(gemv_int8_kernel<M>, dim3(grid), dim3(256), static_cast<size_t>(M) * a.kpad, s, a);
  if (err != cudaSuccess) {
    set_last_error("gemv_int8", err);
    return NQT_ERR_CUDA;
  }
  return NQT_OK;
}

int gemv_slots(int m) { return m <= 1 ? 1 : (m <= 2 ? 2 : (m <= 4 ? 4 : 8)); }

bool takes_gemv(int m, int k) {
  return m <= kGemvMaxM && static_cast<int64_t>(gemv_slots(m)) * ((k + 15) / 16 * 16) <= kGemvSmem;
}

int run_gemv(const GemvArgs& a, cudaStream_t s) {
  switch (gemv_slots(a.m)) {
    case 1: return launch_gemv<1>(a, s);
    case 2: return launch_gemv<2>(a, s);
    case 4: return launch_gemv<4>(a, s);
    default: return launch_gemv<8>(a, s);
  }
}

// ------------------------------------------------------------------ host
// CTAs that run at once in clusters of `split` (each CTA takes its SM whole; clusters leave some SMs over).
int max_ctas(int split) {
  static DeviceOnce once;
  static int most[kMaxSplit + 1];
  once([] {
    for (auto kernel : {gemm_int8_kernel<false, 1>, gemm_int8_kernel<false, 2>, gemm_int8_kernel<true, 1>,
                        gemm_int8_kernel<true, 2>})
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem8);
    most[1] = num_sms();
    for (int c = 2; c <= kMaxSplit; c *= 2) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(c);
      cfg.blockDim = dim3(kThreads);
      cfg.dynamicSmemBytes = kSmem8;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = c;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, gemm_int8_kernel<true, 1>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        clusters = 0;
      }
      most[c] = clusters * c;
    }
  });
  return most[split];
}

// Two boxes of K a stage where the ring then still has three stages.
int boxes_per_stage(int rows, int tn) { return 3 * 2 * (rows + tn) * kBlockK <= kRing8 ? 2 : 1; }

// Weight rows per tile, and the CTAs that share a tile's K.  The times of a wave's tiles in ns, fitted to a sweep over
// 16 to 4613 tokens and five weights on one B200.  A box of K costs its barriers and the issue of its products, about
// 120 with two boxes a stage and 270 with one, and wide tiles what they bring into shared memory.  So tiles are as
// narrow as one wave allows (products of codes, weights from HBM: 64 tokens x 12288 x 2048: width 96, 7.8 us, against 128,
// 8.5, and 192, 10.0), and K is shared where that saves more boxes than the cluster's two barriers and the exchange of
// rows x tn sums cost (128 tokens x 2048 x 6144: 7.7 us, against 8.7 undivided; 64 x 2048 x 2048: 5.5 against 4.7, so
// undivided).
struct Tiling {
  int tn, split;
};

Tiling pick_tiling(int m, int n, int boxes, int epilogue) {
  const int widths[] = {256, 224, 192, 160, 128, 96, 64, 32, 16};
  const int64_t sms = max_ctas(1);
  const int64_t m_tiles = (m + kTileM - 1) / kTileM;
  const int rows = m >= kTileM ? kTileM : (m + 7) / 8 * 8;
  Tiling best{256, 1};
  int64_t best_cost = INT64_MAX;
  for (int tn : widths) {
    if (epilogue == kSiluMul && tn % 32) continue;  // a group of gate and up rows stays together
    const int64_t tiles = m_tiles * ((n + tn - 1) / tn);
    const int64_t box = boxes_per_stage(rows, tn) == 2 ? std::max(120, (rows + tn) * 41 / 50)
                                                       : std::max(270, (rows + tn) * 9 / 10);
    for (int split = 1; split <= kMaxSplit; split *= 2) {
      if (split > 1 && (2 * split > boxes || tiles * split > max_ctas(split))) break;
      const int64_t cost = split == 1 ? (tiles + sms - 1) / sms * boxes * box
                                      : (boxes + split - 1) / split * box + 1300 + 75 * split + rows * tn / 6;
      if (cost <= best_cost) {
        best = {tn, split};
        best_cost = cost;
      }
    }
  }
  return best;
}

int launch_i8(const void* xq, int64_t ldxq, const void* w, int64_t ldw, int k, Int8Args a, cudaStream_t s) {
  const Tiling tiling = pick_tiling(a.m, a.n, a.kb, a.epilogue);
  a.tn = tiling.tn;
  a.split = tiling.split;
  const int rows = a.m >= kTileM ? kTileM : (a.m + 7) / 8 * 8;
  a.a_bytes = rows * kBlockK;
  const int box = a.a_bytes + a.tn * kBlockK;
  const int sub = a.kb > 1 ? boxes_per_stage(rows, a.tn) : 1;
  a.kb = (a.kb + sub - 1) / sub;
  const int stage = box * sub;
  // the MMA reads 128 token rows from each box's start: the last stage keeps that much before the tail
  const int reach = (sub - 1) * a.a_bytes + kTileM * kBlockK;
  a.stages = std::min(kRing8 / stage, kMaxStages8);
  while (a.stages > 1 && (a.stages - 1) * stage + reach > kRing8) --a.stages;
  a.tmem_cols = 32;
  while (a.tmem_cols < 2u * static_cast<uint32_t>(a.tn)) a.tmem_cols <<= 1;
  if (a.tn < 32) a.tmem_cols = 64;  // the epilogue reads 32 columns of either buffer
  CUtensorMap xmap, wmap;
  if (encode_i8(&xmap, xq, a.m, k, ldxq, rows) != NQT_OK || encode_i8(&wmap, w, a.n, k, ldw, a.tn) != NQT_OK) {
    set_last_message("gemm_int8: cuTensorMapEncodeTiled failed");
    return NQT_ERR_CUDA;
  }
  a.m_tiles = (a.m + kTileM - 1) / kTileM;
  const int64_t tiles = static_cast<int64_t>(a.m_tiles) * ((a.n + a.tn - 1) / a.tn);
  if (tiles > 0x3fffffff) return NQT_ERR_UNSUPPORTED;
  a.tiles = static_cast<int>(tiles);
  const int sms = num_sms();
  cudaError_t err;
  if (a.split > 1) {
    err = launch_pdl_cluster(sub == 2 ? gemm_int8_kernel<true, 2> : gemm_int8_kernel<true, 1>, dim3(a.tiles * a.split), dim3(kThreads), kSmem8, s, a.split, xmap,
                             wmap, a);
  } else {
    const int grid = a.tiles < sms ? a.tiles : sms;
    err = launch_pdl(sub == 2 ? gemm_int8_kernel<false, 2> : gemm_int8_kernel<false, 1>, dim3(grid), dim3(kThreads), kSmem8, s, xmap, wmap, a);
  }
  if (err != cudaSuccess) {
    set_last_error("gemm_int8", err);
    return NQT_ERR_CUDA;
  }
  return NQT_OK;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// `codes`: whether the call reads (or writes and reads) xq and xscale.
int check_gemm(bool codes, const void* xq, int64_t ldxq, const float* xscale, const void* w, int64_t ldw,
               const float* wscale, const void* bias, const void* y, int64_t ldy, int m, int n, int cols, int k,
               int epilogue) {
  if (!w || !wscale || !y || m < 0 || n < 1 || k < 1 || cols < 1) return NQT_ERR_ARG;
  if (epilogue != kPlain && epilogue != kBias && epilogue != kSiluMul) return NQT_ERR_ARG;
  if (epilogue == kBias && !bias) return NQT_ERR_ARG;
  if (epilogue == kSiluMul ? (n % 32 != 0 || cols > n / 2) : cols != n) return NQT_ERR_ARG;
  if (k > 131072) return NQT_ERR_UNSUPPORTED;  // the int32 sums could overflow
  if (m > INT32_MAX - (kTileM - 1) || n > INT32_MAX - (kMaxTN - 1)) return NQT_ERR_UNSUPPORTED;  // whole tiles of them
  if (codes && (!xq || !xscale || !aligned(xq, 16) || ldxq % 16 || ldxq < k)) return NQT_ERR_ARG;
  if (!aligned(w, 16) || ldw % 16 || ldw < k || ldy < cols || !aligned(y, 2)) return NQT_ERR_ARG;
  return NQT_OK;
}

int run_gemm(const void* xq, int64_t ldxq, const float* xscale, const void* w, int64_t ldw, const float* wscale,
             const void* bias, void* y, int64_t ldy, int m, int n, int cols, int k, int epilogue, int early,
             int32_t* status, cudaStream_t s) {
  Int8Args a{};
  a.xscale = xscale;
  a.wscale = wscale;
  a.bias = static_cast<const __nv_bfloat16*>(bias);
  a.y = static_cast<__nv_bfloat16*>(y);
  a.ldy = ldy;
  a.status = status;
  a.m = m;
  a.n = n;
  a.cols = cols;
  a.kb = (k + kBlockK - 1) / kBlockK;
  a.epilogue = epilogue;
  a.early = early;
  a.vec16 = aligned(y, 16) && ldy % 8 == 0;
  return launch_i8(xq, ldxq, w, ldw, k, a, s);
}

GemvArgs gemv_args(const void* x, int64_t ldx, const void* xq, int64_t ldxq, const float* xscale, const void* w,
                   int64_t ldw, const float* wscale, const void* bias, void* y, int64_t ldy, int m, int n, int cols,
                   int k, int epilogue) {
  GemvArgs a{};
  a.x = static_cast<const __nv_bfloat16*>(x);
  a.ldx = ldx;
  a.xq = static_cast<const int8_t*>(xq);
  a.ldxq = ldxq;
  a.xscale = xscale;
  a.w = static_cast<const int8_t*>(w);
  a.ldw = ldw;
  a.wscale = wscale;
  a.bias = static_cast<const __nv_bfloat16*>(bias);
  a.y = static_cast<__nv_bfloat16*>(y);
  a.ldy = ldy;
  a.m = m;
  a.n = n;
  a.cols = cols;
  a.k = k;
  a.kpad = (k + 15) / 16 * 16;
  a.epilogue = epilogue;
  a.xvec = x != nullptr && aligned(x, 16) && ldx % 8 == 0 && k % 8 == 0;
  return a;
}

int run_quantize(const void* x, int64_t ldx, int m, int k, void* q, int64_t ldq, float* scale, cudaStream_t s) {
  const bool vec = aligned(x, 16) && ldx % 8 == 0 && k % 8 == 0 && aligned(q, 8) && ldq % 8 == 0;
  const __nv_bfloat16* xp = static_cast<const __nv_bfloat16*>(x);
  int8_t* qp = static_cast<int8_t*>(q);
  // A warp per row where its lanes hold the row (k <= 1024: 4613 x 1024 from HBM on one B200 4.0 us, against 7.7 with four
  // warps), and up to 2048 when there are rows enough for the GPU (4613 x 2048: 7.1 us, against 9.3); else four warps,
  // which hold 6144 elements (4613 x 6144: 14.5 us, 5.9 TB/s, against 15.9 with eight warps).
  const bool warp_rows = k <= 1024 || (k <= 2048 && m >= 8 * num_sms());
  auto kernel = warp_rows ? (vec ? int8_quantize_rows_kernel<32, true> : int8_quantize_rows_kernel<32, false>)
                          : (vec ? int8_quantize_rows_kernel<128, true> : int8_quantize_rows_kernel<128, false>);
  const unsigned grid = warp_rows ? (static_cast<unsigned>(m) + 7) / 8 : (static_cast<unsigned>(m) + 1) / 2;
  const cudaError_t err = launch_pdl(kernel, dim3(grid), dim3(256), 0, s, xp, ldx, m, k, qp, ldq, scale);
  if (err != cudaSuccess) {
    set_last_error("int8_quantize_rows", err);
    return NQT_ERR_CUDA;
  }
  return NQT_OK;
}

}  // namespace
}  // namespace nqt

using namespace nqt;

extern "C" int nqt_int8_quantize_rows(const void* x, int64_t ldx, int m, int k, void* q, int64_t ldq, float* scale,
                                      void* stream) {
  if (m < 0 || k < 1 || ldx < k || ldq < k) return NQT_ERR_ARG;
  if (k > INT32_MAX - 7) return NQT_ERR_UNSUPPORTED;  // whole vectors of 8
  if (m == 0) return NQT_OK;  // tensors without elements have no address
  if (!x || !q || !scale || !aligned(x, 2) || !aligned(scale, 4)) return NQT_ERR_ARG;
  return run_quantize(x, ldx, m, k, q, ldq, scale, as_stream(stream));
}

extern "C" int nqt_gemm_int8(const void* xq, int64_t ldxq, const float* xscale, const void* w, int64_t ldw,
                             const float* wscale, const void* bias, void* y, int64_t ldy, int m, int n, int cols,
                             int k, int epilogue, int32_t* status, void* stream) {
  const int rc = check_gemm(true, xq, ldxq, xscale, w, ldw, wscale, bias, y, ldy, m, n, cols, k, epilogue);
  if (rc != NQT_OK) return rc;
  if (m == 0) return NQT_OK;
  if (takes_gemv(m, k))
    return run_gemv(gemv_args(nullptr, 0, xq, ldxq, xscale, w, ldw, wscale, bias, y, ldy, m, n, cols, k, epilogue),
                    as_stream(stream));
  return run_gemm(xq, ldxq, xscale, w, ldw, wscale, bias, y, ldy, m, n, cols, k, epilogue, 0, status,
                  as_stream(stream));
}

extern "C" int nqt_linear_int8_launches(int m, int k) { return m < 1 || k < 1 ? 0 : (takes_gemv(m, k) ? 1 : 2); }

extern "C" int nqt_linear_int8(const void* x, int64_t ldx, void* xq, int64_t ldxq, float* xscale, const void* w,
                               int64_t ldw, const float* wscale, const void* bias, void* y, int64_t ldy, int m, int n,
                               int cols, int k, int epilogue, int32_t* status, void* stream) {
  const int rc = check_gemm(nqt_linear_int8_launches(m, k) == 2, xq, ldxq, xscale, w, ldw, wscale, bias, y, ldy, m, n,
                            cols, k, epilogue);
  if (rc != NQT_OK) return rc;
  if (!x || ldx < k || !aligned(x, 2)) return NQT_ERR_ARG;
  if (m == 0) return NQT_OK;
  cudaStream_t s = as_stream(stream);
  if (takes_gemv(m, k))
    return run_gemv(gemv_args(x, ldx, nullptr, 0, nullptr, w, ldw, wscale, bias, y, ldy, m, n, cols, k, epilogue), s);
  const int rq = run_quantize(x, ldx, m, k, xq, ldxq, xscale, s);
  if (rq != NQT_OK) return rq;
  // the product starts when the quantiser has seen all earlier kernels finish, so it may read the weights at once
  return run_gemm(xq, ldxq, xscale, w, ldw, wscale, bias, y, ldy, m, n, cols, k, epilogue, 1, status, s);
}
