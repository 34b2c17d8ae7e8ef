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
// Work.  A CTA owns a window of consecutive tokens and a share of the units (query heads, K heads, V heads); its
// warps take turns at (unit, token) rows of q and at (unit, group) of K and V, where a group belongs to the window
// that holds its first token.  The rotations of the window's tokens are computed once into shared memory and serve
// every head.  Eight lanes share a row (a lane owns D / 16 neighbouring elements of the first half and their partners,
// so loads and stores are wide, the rotation needs no shuffle and a sum three), a warp takes four rows at a time.  K
// and V are read twice, once for the maximum and once (from L1) to be rounded; between the two only the rows' norms
// are kept.  Few tokens: windows of one token and up to one unit per warp, for latency.  Many: windows of 16, the
// groups of an aligned prefill.  Bound by latency for a decode step, by instruction issue for a prefill.  One B200, 16
// query and 8 KV heads of 128, captured graphs: 200 tokens 9.6 us, 4893 tokens 31 us (70 MB), 16384 tokens 87 us (2.7
// TB/s).  The page read: 307 pages 8.1 us, 1025 pages 22 us (4.6 TB/s).
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
  int vec;  // every row of q, k, v, out and the weights is 16-byte aligned
  float eps;
  uint64_t turns[64];  // round(2^64 theta^(-2i/D) / (2 pi)), i < D / 2
};

constexpr int kLanes = 8;  // lanes of a row

// The lane's elements of one head row: E = D / 16 from E l of the first half (x), and the same of the second (y).
template <int D>
__device__ __forceinline__ void load_half(const __nv_bfloat16* p, int vec, float (&x)[D / 16]) {
  constexpr int E = D / 16;
  if (vec) {
    uint32_t w[E / 2];
    if constexpr (E == 8) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x;
      w[1] = v.y;
      w[E / 2 - 2] = v.z;
      w[E / 2 - 1] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x;
      w[1] = v.y;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = __bfloat162float(p[i]);
  }
}
template <int D>
__device__ __forceinline__ void load_row(const __nv_bfloat16* row, int l8, int vec, float (&x)[D / 16],
                                         float (&y)[D / 16]) {
  load_half<D>(row + l8 * (D / 16), vec, x);
  load_half<D>(row + D / 2 + l8 * (D / 16), vec, y);
}

__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// 1 / RMS of one head row.
template <int D>
__device__ __forceinline__ float inv_rms(const float (&x)[D / 16], const float (&y)[D / 16], float eps) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) ss += x[j] * x[j] + y[j] * y[j];
  return rsqrtf(row_sum(ss) * (1.0f / D) + eps);  // within 2 ulp
}

// The row's norm `inv` and weights applied, and its rotation by the token's (cos, sin) pairs `cs`.
template <int D>
__device__ __forceinline__ void norm_rope(float (&x)[D / 16], float (&y)[D / 16], const float (&wx)[D / 16],
                                          const float (&wy)[D / 16], const float2* cs, int l8, float inv) {
  constexpr int E = D / 16;
#pragma unroll
  for (int j = 0; j < E; j += 2) {
    const float4 r = *reinterpret_cast<const float4*>(cs + E * l8 + j);
    const float a0 = x[j] * inv * wx[j], b0 = y[j] * inv * wy[j];
    const float a1 = x[j + 1] * inv * wx[j + 1], b1 = y[j + 1] * inv * wy[j + 1];
    x[j] = a0 * r.x - b0 * r.y;
    y[j] = b0 * r.x + a0 * r.y;
    x[j + 1] = a1 * r.z - b1 * r.w;
    y[j + 1] = b1 * r.z + a1 * r.w;
  }
}

template <int D>
__device__ __forceinline__ void store_half(__nv_bfloat16* p, int vec, const float (&x)[D / 16]) {
  constexpr int E = D / 16;
  if (vec) {
    if constexpr (E == 8)
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                                pack_bf16x2(x[E - 4], x[E - 3]), pack_bf16x2(x[E - 2], x[E - 1]));
    else
      *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) p[i] = __float2bfloat16_rn(x[i]);
  }
}

// Codes of x / s, E in a row at r, as x times the rounded 1 / s: within 2^-23 of the quotient, relative, so a code is not
// the quotient's only where that lies within 2^-16 steps of the middle between two codes.
template <int D, bool E4M3>
__device__ __forceinline__ void store_codes(uint8_t* r, const float (&x)[D / 16], float s, float inv) {
  constexpr int E = D / 16;
  uint32_t w[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      // 1 / s overflows for subnormal scales only; s = 0 stands for a block of zeros (and of what is NaN: 0 x)
      v[j] = x[4 * i + j] * (inv <= FLT_MAX ? inv : 0.f);
    if (inv > FLT_MAX && s > 0.f)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __fdiv_rn(x[4 * i + j], s);
    w[i] = codes_of_pair<E4M3>(v[0], v[1]) | static_cast<uint32_t>(codes_of_pair<E4M3>(v[2], v[3])) << 16;
  }
  if constexpr (E == 8) *reinterpret_cast<uint2*>(r) = make_uint2(w[0], w[E / 4 - 1]);
  else *reinterpret_cast<uint32_t*>(r) = w[0];
}

constexpr int kWindow = 16;   // tokens of a window when there are many
constexpr int kWarps8 = 8;

// W: tokens of a window, 1 or kWindow.
template <int D, bool E4M3, int W>
__global__ void __launch_bounds__(kWarps8 * 32, 4) write8_kernel(const __grid_constant__ Write8Args a) {
  constexpr int E = D / 16;
  constexpr int H = D / 2;
  // a decode launch queued behind this one with NQT_DECODE_OVERLAP_KV_WRITE may read the page table and the
  // blocks that this call does not write; it waits for this grid before q and each row's last block
  grid_dependents_launch();
  extern __shared__ float smem8[];
  // rotations of the window's tokens and of the up to 15 that its last group has behind it
  constexpr int kTok = W + kBlock - 1;
  float2* s_cs = reinterpret_cast<float2*>(smem8);                      // [kTok][H]
  __shared__ int s_first[W], s_count[W], s_groups, s_end;  // groups: first token (in the window), tokens; end of the last
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.x * W;
  const int live = min(W, a.tokens - t0);

  // the groups whose first token lies in the window: lane i of warp 0 looks at token t0 - 1 + i
  if (warp == 0) {
    int64_t page = -1, off = -1;
    const int t = t0 - 1 + lane;
    if (lane <= kTok && t >= 0 && t < a.tokens) {
      page = a.pages[t];
      off = a.offsets[t];
    }
    const int64_t p_page = __shfl_up_sync(kFull, page, 1), p_off = __shfl_up_sync(kFull, off, 1);
    const bool ok = page >= 0 && page < a.total_pages && off >= 0 && off < a.page_size;
    // the token continues the group of the one before it
    const bool cont = lane >= 1 && ok && p_page == page && p_off >= 0 && p_off / kBlock == off / kBlock && p_off < off;
    const bool mine = lane >= 1 && lane <= live;
    if (mine && !ok) report(a.status, NQT_DEV_BAD_PAGE);
    const unsigned conts = __ballot_sync(kFull, cont);
    const unsigned firsts = __ballot_sync(kFull, mine && ok && !cont);
    if (mine && ok && !cont) {
      const int g = __popc(firsts & ((1u << lane) - 1u));
      s_first[g] = lane - 1;  // lane <= W < 31
      s_count[g] = min(__ffs(~(conts >> (lane + 1))), kBlock);
    }
    if (lane == 0) {
      s_groups = __popc(firsts);
      if (firsts == 0u) s_end = 0;
    }
    if (firsts != 0u && lane == 31 - __clz(firsts)) s_end = lane - 1 + min(__ffs(~(conts >> (lane + 1))), kBlock);
  }
  // rotations: position * turns as a 64-bit fraction of a turn, rounded to the nearest 2^-32 turn in [-1/2, 1/2)
  const int d = threadIdx.x % H;
  const uint64_t turns = a.turns[d];
  auto rotations = [&](int from, int to) {
    for (int t = from + threadIdx.x / H; t < to; t += kWarps8 * 32 / H) {
      const uint64_t turn = static_cast<uint64_t>(a.pos[t0 + t]) * turns + 0x80000000ull;
      const float half_turns = static_cast<float>(static_cast<int32_t>(turn >> 32)) * 4.656612873077393e-10f;  // 2^-31
      float s, c;
      sincospif(half_turns, &s, &c);
      s_cs[t * H + d] = make_float2(c, s);
    }
  };
  rotations(0, live);
  __syncthreads();
  if (s_end > live) {  // the last group goes on behind the window (the same for every thread)
    rotations(live, s_end);
    __syncthreads();
  }

  // this CTA's units: query heads, then K heads, then V heads; the dearer K and V start first (4893 tokens, 16 and 8
  // heads of 128: 31 us, against 34 the other way round, and 46 with the kinds mixed in every CTA)
  const int units = a.hq + 2 * a.hkv;
  const int per = (units + gridDim.y - 1) / gridDim.y;
  const int u0 = (gridDim.y - 1 - blockIdx.y) * per, u1 = min(units, u0 + per);

  const int sub = lane / kLanes, l8 = lane % kLanes;  // row of the warp's four, place in it
  {
    float wx[E], wy[E];
    load_row<D>(a.qw, l8, a.vec, wx, wy);
    const int rows = (min(u1, a.hq) - u0) * W;
#pragma unroll 2
    for (int i = warp * 4 + sub; i < (rows + 3) / 4 * 4; i += kWarps8 * 4) {  // whole warps: the sums shuffle
      const int head = u0 + i / W, t = i % W;
      const bool on = i < rows && t < live;
      float x[E], y[E];
      load_row<D>(a.q + (t0 + (on ? t : 0)) * a.q_st + (on ? head : u0) * a.q_sh, l8, a.vec, x, y);
      norm_rope<D>(x, y, wx, wy, s_cs + (on ? t : 0) * H, l8, inv_rms<D>(x, y, a.eps));
      if (on) {
        __nv_bfloat16* dst = a.out + (t0 + t) * a.o_st + head * a.o_sh + l8 * E;
        store_half<D>(dst, a.vec, x);
        store_half<D>(dst + H, a.vec, y);
      }
    }
  }

  const int groups = s_groups;
  const int kv0 = max(u0, a.hq);
  const int64_t row = static_cast<int64_t>(a.hkv) * D;
  for (int w = warp; w < (u1 - kv0) * groups; w += kWarps8) {
    const int unit = kv0 + w / groups, g = w % groups;
    const int kind = unit < a.hq + a.hkv ? 0 : 1;
    const int head = unit - a.hq - kind * a.hkv;
    const int first = s_first[g], n = s_count[g], t = t0 + first;
    const int64_t page = a.pages[t];
    const int off0 = static_cast<int>(a.offsets[t]);
    const int blk = off0 / kBlock, o = off0 % kBlock;
    const __nv_bfloat16* src = kind == 0 ? a.k + t * a.k_st + head * a.k_sh : a.v + t * a.v_st + head * a.v_sh;
    const int64_t st = kind == 0 ? a.k_st : a.v_st;

    float wx[E], wy[E];
    load_row<D>(a.kw, l8, a.vec, wx, wy);
    float amax = 0.f;
    float inv_of[4];  // 1 / RMS of the lane's rows (K)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 4 + sub;
      inv_of[i] = 0.f;
      if (i * 4 < n) {  // the same for the whole warp
        float x[E], y[E];
        load_row<D>(src + (r < n ? r : 0) * st, l8, a.vec, x, y);  // a row that is not there repeats the first
        if (kind == 0) {
          inv_of[i] = inv_rms<D>(x, y, a.eps);
          norm_rope<D>(x, y, wx, wy, s_cs + (first + (r < n ? r : 0)) * H, l8, inv_of[i]);
        }
#pragma unroll
        for (int j = 0; j < E; ++j) amax = fmaxf(amax, fmaxf(fabsf(x[j]), fabsf(y[j])));
      }
    }
    amax = fminf(warp_max(amax), FLT_MAX);
    const float need = __fdiv_rn(amax, top_code<E4M3>());

    uint8_t* block = a.cache + ((page * 2 + kind) * a.page_size + blk * kBlock) * row + static_cast<int64_t>(head) * D;
    float* sp = a.scales + ((page * 2 + kind) * (a.page_size / kBlock) + blk) * a.hkv + head;
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
#pragma unroll 1
        for (int i = sub; i < o; i += 4) {
          uint32_t* r = reinterpret_cast<uint32_t*>(block + i * row) + l8 * (D / 32);
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const uint32_t c = r[j];
            const uint32_t lo = codes_of_pair<E4M3>(code_to_f32<E4M3>(c, 0) * f, code_to_f32<E4M3>(c, 1) * f);
            const uint32_t hi = codes_of_pair<E4M3>(code_to_f32<E4M3>(c, 2) * f, code_to_f32<E4M3>(c, 3) * f);
            r[j] = lo | hi << 16;
          }
        }
      }
      __syncwarp();  // every lane has read the old scale
    }
    if (lane == 0) *sp = s;
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 4 + sub;
      if (r >= n) continue;
      float x[E], y[E];
      load_row<D>(src + r * st, l8, a.vec, x, y);
      if (kind == 0) norm_rope<D>(x, y, wx, wy, s_cs + (first + r) * H, l8, inv_of[i]);
      uint8_t* dst = block + static_cast<int>(a.offsets[t + r]) % kBlock * row + l8 * E;
      store_codes<D, E4M3>(dst, x, s, inv);
      store_codes<D, E4M3>(dst + H, y, s, inv);
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

template <int D, bool E4M3, int W>
int launch_window(const Write8Args& a, int slices, cudaStream_t s) {
  constexpr int kSmem = (W + kBlock - 1) * (D / 2) * 8;
  write8_kernel<D, E4M3, W><<<dim3((a.tokens + W - 1) / W, slices), kWarps8 * 32, kSmem, s>>>(a);
  return check_launch("qk_norm_rope_paged_cache8");
}

template <int D, bool E4M3>
int launch_write8(const Write8Args& a, cudaStream_t s) {
  const int units = a.hq + 2 * a.hkv;
  const int sms = num_sms();
  // Windows of one token and a warp per unit until those CTAs fill the GPU twice over; then windows of 16 tokens,
  // their units sliced only as far as that fills it.
  const int fine = (units + kWarps8 - 1) / kWarps8;
  if (static_cast<int64_t>(a.tokens) * fine <= 4 * sms) return launch_window<D, E4M3, 1>(a, fine, s);
  const int windows = (a.tokens + kWindow - 1) / kWindow;
  int slices = (8 * sms + windows - 1) / windows;
  slices = slices < 1 ? 1 : (slices > fine ? fine : slices);
  return launch_window<D, E4M3, kWindow>(a, slices, s);
}

bool rows_aligned(const void* p, int64_t st, int64_t sh) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && st % 8 == 0 && sh % 8 == 0;
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
  if (tokens < 0 || num_qo_heads < 1 || !(rope_theta > 0.f && rope_theta <= FLT_MAX)) return NQT_ERR_ARG;
  if (tokens == 0) return NQT_OK;
  const int units = num_qo_heads + 2 * num_kv_heads;
  if ((units + kWarps8 - 1) / kWarps8 > 65535) return NQT_ERR_UNSUPPORTED;
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
  a.vec = rows_aligned(q, q_stride_tok, q_stride_head) && rows_aligned(k, k_stride_tok, k_stride_head) &&
          rows_aligned(v, v_stride_tok, v_stride_head) && rows_aligned(q_out, out_stride_tok, out_stride_head) &&
          rows_aligned(q_weight, 0, 0) && rows_aligned(k_weight, 0, 0);
  turn_table(a.turns, head_dim, rope_theta);
  cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return code == NQT_E4M3 ? launch_write8<128, true>(a, s) : launch_write8<128, false>(a, s);
  return code == NQT_E4M3 ? launch_write8<64, true>(a, s) : launch_write8<64, false>(a, s);
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
