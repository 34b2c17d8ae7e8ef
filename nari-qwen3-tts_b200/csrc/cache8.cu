// Writing and reading the 8-bit paged KV cache (layout and codes: cache8.cuh).
//
// The write takes a step's packed q, k, v and does what a decoder layer does
// between its QKV projection and its attention: q and k are RMS-normalised
// per head and rotated, k and v are quantised into their pages.  All of it is
// fp32; the only roundings are q to bf16 and k, v to codes.
//
// Quantisation.  The tokens that one call writes into a block of 16 share the
// block's new scale.  With need = (largest magnitude of the group) / top code:
//   the group starts the block (its first offset is 0):  s' = need
//   the block has tokens already:  s' = s * 2^k, the least k >= 0 with
//   s' >= need (s = 0: s' = need), and the codes of the tokens before the
//   group are rounded again to code * s / s'.
// Growing by powers of two bounds what the re-rounding costs: a code that is
// rounded k times is off by at most s' (1/2 + 1/4 + ...) < s' in all, where
// following the maximum exactly would cost half a step for every new maximum.
// Codes behind the group are left as they are: they belong to no token.
//
// Angles.  position * theta^(-2i/D) is taken in turns as a 64-bit fraction,
// position * round(2^64 theta^(-2i/D) / 2 pi) mod 2^64, so whole turns drop
// out exactly and far positions lose nothing; then sincospi in fp32.
//
// Work.  One warp owns one unit: a query head of one token, or K or V of one
// KV head of one block group, whose up to 16 tokens stay in registers between
// the maximum and the rounding (a lane owns the rotation pairs (2l, 2l + 1)
// and their partners, so loads are 4-byte and the rotation needs no shuffle).
// The group is led by its first token; the warps of the others leave at once.
// Bound by latency for a decode step and by HBM for a prefill.
#include "cache8.cuh"

#include <float.h>
#include <math.h>
#include <string.h>

namespace nqt {
namespace {

using namespace c8;

struct Write8Args {
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  const __nv_bfloat16 *qw, *kw;
  const int64_t *pos, *pages, *offsets;
  uint8_t* cache;
  float* scales;
  int32_t* status;
  int tokens, hq, hkv, page_size, total_pages;
  int vec;  // every row of q, k, v, out and the weights is 4-byte aligned
  float eps;
  uint64_t turns[64];  // round(2^64 theta^(-2i/D) / (2 pi)), i < D / 2
};

// Two neighbouring elements as floats.
__device__ __forceinline__ float2 load_pair(const __nv_bfloat16* p, int vec) {
  if (vec) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
  return make_float2(__bfloat162float(p[0]), __bfloat162float(p[1]));
}

// RMSNorm and rotation of one head row.  A lane holds the J pairs of elements x[2j], x[2j + 1] = first halves
// (dims J lane ..) and y[...] their partners D / 2 further.
template <int D>
__device__ __forceinline__ void norm_rope(float (&x)[D / 64], float (&y)[D / 64], const float (&wx)[D / 64],
                                          const float (&wy)[D / 64], const uint64_t (&turn)[D / 64], int64_t pos,
                                          float eps) {
  constexpr int J = D / 64;
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) ss += x[j] * x[j] + y[j] * y[j];
  ss = warp_sum(ss);
  const float inv = 1.0f / sqrtf(ss / static_cast<float>(D) + eps);
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const float a = x[j] * inv * wx[j];
    const float b = y[j] * inv * wy[j];
    // the fraction of a turn, rounded to the nearest 2^-32 turn in [-1/2, 1/2), times two for sincospi
    const uint64_t t = static_cast<uint64_t>(pos) * turn[j] + 0x80000000ull;
    const float half_turns = static_cast<float>(static_cast<int32_t>(t >> 32)) * 4.656612873077393e-10f;  // 2^-31
    float s, c;
    sincospif(half_turns, &s, &c);
    x[j] = a * c - b * s;
    y[j] = b * c + a * s;
  }
}

// The lane's elements of one head row: D = 128: dims 2l, 2l + 1 and 64 + the same; D = 64: dims l and 32 + l.
template <int D>
__device__ __forceinline__ void load_row(const __nv_bfloat16* row, int lane, int vec, float (&x)[D / 64],
                                         float (&y)[D / 64]) {
  if constexpr (D == 128) {
    const float2 a = load_pair(row + 2 * lane, vec), b = load_pair(row + 64 + 2 * lane, vec);
    x[0] = a.x;
    x[1] = a.y;
    y[0] = b.x;
    y[1] = b.y;
  } else {
    x[0] = __bfloat162float(row[lane]);
    y[0] = __bfloat162float(row[32 + lane]);
  }
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(256) write8_kernel(const __grid_constant__ Write8Args a) {
  constexpr int J = D / 64;
  constexpr int H = D / 2;
  // a decode launch queued behind this one with NQT_DECODE_OVERLAP_KV_WRITE may read the page table and the
  // blocks that this call does not write; it waits for this grid before q and each row's last block
  grid_dependents_launch();
  const int unit = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (unit >= a.hq + 2 * a.hkv) return;
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31;

  uint64_t turn[J];
  if (unit < a.hq + a.hkv) {
#pragma unroll
    for (int j = 0; j < J; ++j) turn[j] = a.turns[J * lane + j];
  }

  if (unit < a.hq) {
    float x[J], y[J], wx[J], wy[J];
    load_row<D>(a.q + t * a.q_st + unit * a.q_sh, lane, a.vec, x, y);
    load_row<D>(a.qw, lane, a.vec, wx, wy);
    norm_rope<D>(x, y, wx, wy, turn, a.pos[t], a.eps);
    __nv_bfloat16* dst = a.out + t * a.o_st + unit * a.o_sh;
    if (D == 128 && a.vec) {
      *reinterpret_cast<__nv_bfloat162*>(dst + J * lane) = __floats2bfloat162_rn(x[0], x[J - 1]);
      *reinterpret_cast<__nv_bfloat162*>(dst + H + J * lane) = __floats2bfloat162_rn(y[0], y[J - 1]);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        dst[J * lane + j] = __float2bfloat16_rn(x[j]);
        dst[H + J * lane + j] = __float2bfloat16_rn(y[j]);
      }
    }
    return;
  }

  // ---- K or V of one head of the block group that starts at token t
  const int kind = unit < a.hq + a.hkv ? 0 : 1;
  const int head = unit - a.hq - kind * a.hkv;
  // lane i < 17 looks at token t - 1 + i: lane 0 at the one before
  int64_t page = -1, off = -1;
  const int tt = t - 1 + lane;
  if (lane <= kBlock && tt >= 0 && tt < a.tokens) {
    page = a.pages[tt];
    off = a.offsets[tt];
  }
  const int64_t p_page = __shfl_up_sync(kFull, page, 1), p_off = __shfl_up_sync(kFull, off, 1);
  const bool ok_here = page >= 0 && page < a.total_pages && off >= 0 && off < a.page_size;
  // this token continues the group of the one before it
  const bool cont = lane >= 1 && lane <= kBlock && ok_here && p_page == page && p_off >= 0 &&
                    (p_off / kBlock) == (off / kBlock) && p_off < off;
  const unsigned conts = __ballot_sync(kFull, cont);
  const unsigned oks = __ballot_sync(kFull, ok_here);
  if (!(oks & 2u)) {
    if (lane == 0) report(a.status, NQT_DEV_BAD_PAGE);
    return;
  }
  if (conts & 2u) return;                      // not the group's first token
  const int n = __ffs(~(conts >> 2));          // tokens t .. t + n - 1, n <= 16
  const int64_t pg = __shfl_sync(kFull, page, 1);
  const int off0 = static_cast<int>(__shfl_sync(kFull, off, 1));
  const int blk = off0 / kBlock, o = off0 % kBlock;
  const int my_off = static_cast<int>(off);    // lane i + 1: offset of the group's token i

  float x[kBlock][J], y[kBlock][J];
  float amax = 0.f;
  {
    const __nv_bfloat16* src = kind == 0 ? a.k + t * a.k_st + head * a.k_sh : a.v + t * a.v_st + head * a.v_sh;
    const int64_t st = kind == 0 ? a.k_st : a.v_st;
#pragma unroll
    for (int i = 0; i < kBlock; ++i)
      if (i < n) load_row<D>(src + i * st, lane, a.vec, x[i], y[i]);
    if (kind == 0) {
      float wx[J], wy[J];
      load_row<D>(a.kw, lane, a.vec, wx, wy);
#pragma unroll
      for (int i = 0; i < kBlock; ++i)
        if (i < n) norm_rope<D>(x[i], y[i], wx, wy, turn, a.pos[t + i], a.eps);
    }
#pragma unroll
    for (int i = 0; i < kBlock; ++i)
      if (i < n) {
#pragma unroll
        for (int j = 0; j < J; ++j) amax = fmaxf(amax, fmaxf(fabsf(x[i][j]), fabsf(y[i][j])));
      }
  }
  amax = fminf(warp_max(amax), FLT_MAX);
  const float need = __fdiv_rn(amax, top_code<E4M3>());

  const int64_t row = static_cast<int64_t>(a.hkv) * D;
  uint8_t* block = a.cache + ((pg * 2 + kind) * a.page_size + blk * kBlock) * row + static_cast<int64_t>(head) * D;
  float* sp = a.scales + ((pg * 2 + kind) * (a.page_size / kBlock) + blk) * a.hkv + head;
  float s = need;
  if (o != 0) {
    const float old = *sp;
    if (old > 0.f) {
      const float ratio = __fdiv_rn(need, old);
      s = ratio <= 1.f ? old : (ratio <= FLT_MAX ? scalbnf(old, fp8::ceil_log2(ratio)) : need);
    }
    if (s != old && s > 0.f) {
      // the codes of the block's earlier tokens follow the scale (all zero if there was none)
      const float f = old > 0.f ? __fdiv_rn(old, s) : 0.f;
      for (int i = 0; i < o; ++i) {
        uint8_t* r = block + i * row + lane * (D / 32);
        if constexpr (D == 128) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(r);
          uint32_t u = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) u |= f32_to_code<E4M3>(code_to_f32<E4M3>(w, b) * f) << (8 * b);
          *reinterpret_cast<uint32_t*>(r) = u;
        } else {
          const uint32_t w = *reinterpret_cast<const uint16_t*>(r);
          const uint32_t u = f32_to_code<E4M3>(code_to_f32<E4M3>(w, 0) * f) |
                             (f32_to_code<E4M3>(code_to_f32<E4M3>(w, 1) * f) << 8);
          *reinterpret_cast<uint16_t*>(r) = static_cast<uint16_t>(u);
        }
      }
    }
    __syncwarp();  // every lane has read the old scale
  }
  if (lane == 0) *sp = s;
#pragma unroll
  for (int i = 0; i < kBlock; ++i) {
    if (i >= n) continue;
    const int oi = __shfl_sync(kFull, my_off, i + 1) % kBlock;
    uint8_t* r = block + oi * row;
    uint32_t cx[J], cy[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      cx[j] = s > 0.f ? f32_to_code<E4M3>(__fdiv_rn(x[i][j], s)) : 0u;
      cy[j] = s > 0.f ? f32_to_code<E4M3>(__fdiv_rn(y[i][j], s)) : 0u;
    }
    if constexpr (D == 128) {
      *reinterpret_cast<uint16_t*>(r + 2 * lane) = static_cast<uint16_t>(cx[0] | (cx[J - 1] << 8));
      *reinterpret_cast<uint16_t*>(r + H + 2 * lane) = static_cast<uint16_t>(cy[0] | (cy[J - 1] << 8));
    } else {
      r[lane] = static_cast<uint8_t>(cx[0]);
      r[H + lane] = static_cast<uint8_t>(cy[0]);
    }
  }
}

// Pages back to bf16: one thread per 16 codes (one 16-byte load, two 16-byte stores).
template <bool E4M3>
__global__ void __launch_bounds__(256) read8_kernel(const uint8_t* cache, const float* scales, int total_pages,
                                                    int page_size, int hkv, int d, const int64_t* pages, int64_t total,
                                                    __nv_bfloat16* out, int32_t* status) {
  const int64_t i = blockIdx.x * static_cast<int64_t>(256) + threadIdx.x;
  if (i >= total) return;
  const int vecs = d / 16;                                  // 16-code vectors of a row
  const int64_t row = i / vecs;                             // [page, kind, token, head]
  const int head = static_cast<int>(row % hkv);
  const int64_t tok = row / hkv;                            // [page, kind, token]
  const int in_page = static_cast<int>(tok % page_size);
  const int64_t pk = tok / page_size;
  const int kind = static_cast<int>(pk & 1);
  const int64_t page = pages[pk >> 1];
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  float s = 0.f;
  if (page >= 0 && page < total_pages) {
    const int64_t src = ((page * 2 + kind) * page_size + in_page) * hkv + head;
    w = *reinterpret_cast<const uint4*>(cache + src * d + (i % vecs) * 16);
    s = scales[((page * 2 + kind) * (page_size / kBlock) + in_page / kBlock) * hkv + head];
  } else {
    report(status, NQT_DEV_BAD_PAGE);
  }
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[2 * e] = pack_bf16x2(code_to_f32<E4M3>(ws[e], 0) * s, code_to_f32<E4M3>(ws[e], 1) * s);
    o[2 * e + 1] = pack_bf16x2(code_to_f32<E4M3>(ws[e], 2) * s, code_to_f32<E4M3>(ws[e], 3) * s);
  }
  uint4* dst = reinterpret_cast<uint4*>(out + i * 16);
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// The rotation's turns per position.  The table depends on (head_dim, theta) alone and costs tens of microseconds to
// make, so the thread's last one is kept.
void turn_table(uint64_t* out, int head_dim, float theta) {
  static thread_local float last_theta = 0.f;
  static thread_local int last_dim = 0;
  static thread_local uint64_t last[64];
  if (last_dim != head_dim || last_theta != theta) {
    const long double ln_theta = logl(static_cast<long double>(theta));
    const long double full = 18446744073709551616.0L;  // 2^64
    for (int i = 0; i < head_dim / 2; ++i) {
      const long double f = expl(-ln_theta * (2.0L * i / head_dim)) / 6.283185307179586476925286766559L * full;
      last[i] = static_cast<uint64_t>(fmodl(roundl(f), full));
    }
    last_dim = head_dim;
    last_theta = theta;
  }
  memcpy(out, last, sizeof(uint64_t) * (head_dim / 2));
}

bool pairs_aligned(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 3) == 0 && st % 2 == 0 && sh % 2 == 0;
}

}  // namespace
}  // namespace nqt

using namespace nqt;

extern "C" int nqt_qk_norm_rope_paged_cache8(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k, int64_t k_stride_tok,
    int64_t k_stride_head, const void* v, int64_t v_stride_tok, int64_t v_stride_head, const void* q_weight,
    const void* k_weight, const int64_t* position_ids, const int64_t* write_pages, const int64_t* write_offsets,
    void* q_out, int64_t out_stride_tok, int64_t out_stride_head, void* layer_cache, float* layer_scales,
    int total_pages, int page_size, int tokens, int num_qo_heads, int num_kv_heads, int head_dim, float eps,
    float rope_theta, int code, int32_t* status, void* stream) {
  const int rc = c8::check_layer(layer_cache, layer_scales, total_pages, page_size, num_kv_heads, head_dim, code);
  if (rc != NQT_OK) return rc;
  if (!q || !k || !v || !q_weight || !k_weight || !position_ids || !write_pages || !write_offsets || !q_out)
    return NQT_ERR_ARG;
  if (tokens < 0 || num_qo_heads < 1 || !(rope_theta > 0.f)) return NQT_ERR_ARG;
  if (tokens == 0) return NQT_OK;
  const int units = num_qo_heads + 2 * num_kv_heads;
  if ((units + 7) / 8 > 65535) return NQT_ERR_UNSUPPORTED;
  Write8Args a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.k_st = k_stride_tok;
  a.k_sh = k_stride_head;
  a.v_st = v_stride_tok;
  a.v_sh = v_stride_head;
  a.out = static_cast<__nv_bfloat16*>(q_out);
  a.o_st = out_stride_tok;
  a.o_sh = out_stride_head;
  a.qw = static_cast<const __nv_bfloat16*>(q_weight);
  a.kw = static_cast<const __nv_bfloat16*>(k_weight);
  a.pos = position_ids;
  a.pages = write_pages;
  a.offsets = write_offsets;
  a.cache = static_cast<uint8_t*>(layer_cache);
  a.scales = layer_scales;
  a.status = status;
  a.tokens = tokens;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.page_size = page_size;
  a.total_pages = total_pages;
  a.eps = eps;
  a.vec = pairs_aligned(q, q_stride_tok, q_stride_head) && pairs_aligned(k, k_stride_tok, k_stride_head) &&
          pairs_aligned(v, v_stride_tok, v_stride_head) && pairs_aligned(q_out, out_stride_tok, out_stride_head) &&
          pairs_aligned(q_weight, 0, 0) && pairs_aligned(k_weight, 0, 0);
  turn_table(a.turns, head_dim, rope_theta);
  const dim3 grid(tokens, (units + 7) / 8);
  cudaStream_t s = as_stream(stream);
  const bool e4m3 = code == NQT_E4M3;
  if (head_dim == 128) {
    if (e4m3) write8_kernel<128, true><<<grid, 256, 0, s>>>(a);
    else write8_kernel<128, false><<<grid, 256, 0, s>>>(a);
  } else {
    if (e4m3) write8_kernel<64, true><<<grid, 256, 0, s>>>(a);
    else write8_kernel<64, false><<<grid, 256, 0, s>>>(a);
  }
  return check_launch("qk_norm_rope_paged_cache8");
}

extern "C" int nqt_read_paged_cache8(const void* layer_cache, const float* layer_scales, int total_pages,
                                     int page_size, int num_kv_heads, int head_dim, int code, const int64_t* pages,
                                     int count, void* out, int32_t* status, void* stream) {
  const int rc = c8::check_layer(layer_cache, layer_scales, total_pages, page_size, num_kv_heads, head_dim, code);
  if (rc != NQT_OK) return rc;
  if (!pages || !out || count < 0 || (reinterpret_cast<uintptr_t>(out) & 15)) return NQT_ERR_ARG;
  if (count == 0) return NQT_OK;
  const int64_t total = static_cast<int64_t>(count) * 2 * page_size * num_kv_heads * (head_dim / 16);
  const int64_t blocks = (total + 255) / 256;
  if (blocks > 0x7fffffff) return NQT_ERR_UNSUPPORTED;
  cudaStream_t s = as_stream(stream);
  if (code == NQT_E4M3)
    read8_kernel<true><<<static_cast<unsigned>(blocks), 256, 0, s>>>(
        static_cast<const uint8_t*>(layer_cache), layer_scales, total_pages, page_size, num_kv_heads, head_dim, pages,
        total, static_cast<__nv_bfloat16*>(out), status);
  else
    read8_kernel<false><<<static_cast<unsigned>(blocks), 256, 0, s>>>(
        static_cast<const uint8_t*>(layer_cache), layer_scales, total_pages, page_size, num_kv_heads, head_dim, pages,
        total, static_cast<__nv_bfloat16*>(out), status);
  return check_launch("read_paged_cache8");
}
