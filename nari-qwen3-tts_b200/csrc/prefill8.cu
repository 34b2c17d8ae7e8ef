// Ragged causal prefill attention over an 8-bit paged KV cache (layout and codes: cache8.cuh), tcgen05.
//
//   out[i, h] = softmax(q[i, h] . K[:, h / G]^T * sm_scale) V[:, h / G],  query i of a chunk of n queries sees
//   the keys <= kv_len - n + i of its row.
//
// Mathematics.  With codes k, v and block scales a, c, in log2 units and with a running reference M:
//   x = a sm_scale log2(e) (q . k),  y = x + log2 c,  p' = 2^(y - M + 8),  O += p' v,  l += p' / c,  out = O / l
// so a key's scale is one factor of a score and a value's scale one summand of an exponent: neither costs an
// instruction per element.  q . k runs on the tensor cores in bf16 (q as it is, codes exact), p' v in fp16 (codes
// exact, p' rounded to 11 bits), both with fp32 accumulation; sums are fp32.  M follows the maximum of y, the weight
// with which a key's codes enter the output, and moves only when that grows by more than 7, so p' lies below 2^15
// and fp16 reaches down to 2^-32 of the largest weight.  Scales below 2^-80 count as 2^-80.
//
// A CTA owns two 128-row query tiles of one row and KV head (a tile row is a token x query head of the group) and
// walks over blocks of 64 keys:
//   warp 0        Q loader and TMEM owner; warps 1 and 2: MMA issuers of tile A and B
//   warp 3        brings the codes of a block by TMA (one box of 16 tokens, K and V, per lane) into a raw ring, and
//                 the scale factors of four blocks at a time
//   warps 4..7    converters: raw codes to 16 bits in the operands' 128-byte-swizzled layout
//   warps 8..23   softmax (8..15 tile A, 16..23 tile B), half of a query row's keys per thread
// TMEM: S double-buffered per tile, p' over its own S buffer, O per tile.  The two tiles share every converted
// block, which halves the conversions per product.  setmaxnreg gives the softmax warps the registers that the
// others do not need; every role runs to its own end, with no code in common behind the split.
//
// When the query tiles are too few for the GPU (late chunks of long prompts) a cluster of up to 8 CTAs shares one
// pair of tiles, each walking over a part of its keys; the parts are joined in the cluster's shared memory in CTA
// order, so there is no workspace and nothing depends on timing.
#include "cache8.cuh"
#include "gemm_common.cuh"
#include "tcgen05.cuh"

namespace nqt {
namespace {

using namespace c8;

namespace p8 {
constexpr int kM = 128;       // rows per tile
constexpr int kTiles = 2;     // tiles per CTA
constexpr int kN = 64;        // keys per block
constexpr int kStages = 3;     // converted blocks
constexpr int kRaw = 3;        // raw blocks
constexpr int kScaleRing = 4;  // groups of four blocks whose scale factors are kept
constexpr int kThreads = 768;
constexpr int kPages = 1024;  // page ids of the row staged in shared memory
constexpr int kRows = 512;    // rows of the batch whose tiles are put in order, longest first
constexpr uint32_t kColO = 256;
}  // namespace p8

template <int D>
struct P8Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kQBytes = p8::kM * D * 2;               // [half][128 rows][128 B]
  static constexpr int kHalf = p8::kN * 128;                   // [64 tokens][128 B]
  static constexpr int kKV = 2 * kHalves * kHalf;              // K halves, V halves
  static constexpr int kRawBytes = 2 * p8::kN * D;             // [tile][K, V][16 tokens][D]
  static constexpr int kBars = 512;
  static constexpr int kScales = p8::kScaleRing * 4 * 4 * 3 * 4;  // [block][tile][score factor, log2 c, 1 / c]
  static constexpr int kRowState = 3 * p8::kTiles * p8::kM * 4;  // of every row: log2-sum-exp, for the join; its halves' exchange
  static constexpr int kSmem =
      1024 + p8::kTiles * kQBytes + p8::kStages * kKV + p8::kRaw * kRawBytes + kBars + kScales + kRowState + 4 * p8::kPages;
  static_assert(p8::kStages * kKV + p8::kRaw * kRawBytes >= p8::kTiles * p8::kM * D * 4, "the join stages O over them");
};

struct Prefill8Args {
  const float* scales;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  const int32_t *qo_indptr, *kv_indptr, *indices, *last_len;
  int32_t* status;
  int batch, hq, hkv, group, page_size, total_pages;
  float scale_log2;
  int tma_out;  // full tiles leave through a TMA store
  int out16;    // output rows allow 16-byte stores
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t pk2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t pk2(float lo, float hi) { return pk2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpk2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Whether `v` holds in any of the barrier's threads.
__device__ __forceinline__ bool bar_any(int id, int n, bool v) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %3, 0;\n\tbarrier.cta.red.or.pred p, %1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"(id), "r"(n), "r"(static_cast<uint32_t>(v))
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_addr(src)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Four codes -> two bf16x2 in order.  int8: behind 0x43 a byte's low seven bits are the bf16 number 128 + b, and
// its sign bit turns 128 into 256 in the number to subtract.  e4m3: through the exact fp16 and fp32.
template <bool E4M3>
__device__ __forceinline__ void codes_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    const uint32_t a = e4m3x2_to_f16x2(static_cast<uint16_t>(w)), b = e4m3x2_to_f16x2(static_cast<uint16_t>(w >> 16));
    const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
    const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
    lo = pack_bf16x2(fa.x, fa.y);
    hi = pack_bf16x2(fb.x, fb.y);
  } else {
    const uint32_t p = __byte_perm(w, 0x43434343u, 0x4140), q = __byte_perm(w, 0x43434343u, 0x4342);
    const uint32_t pa = p & 0xff7fff7fu, pb = p & 0xff80ff80u, qa = q & 0xff7fff7fu, qb = q & 0xff80ff80u;
    const __nv_bfloat162 x = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pa),
                                     *reinterpret_cast<const __nv_bfloat162*>(&pb));
    const __nv_bfloat162 y = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&qa),
                                     *reinterpret_cast<const __nv_bfloat162*>(&qb));
    lo = *reinterpret_cast<const uint32_t*>(&x);
    hi = *reinterpret_cast<const uint32_t*>(&y);
  }
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Instruction descriptor, kind::f16 with fp16 operands (formats 0) and fp32 accumulation, B MN-major.
__host__ __device__ constexpr uint32_t idesc_f16_f32_bmn(int m, int n) {
  return (1u << 4) | (1u << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// (row, tile) of tile index `want`, by the whole CTA: rows with the longest keys first (their last tiles first), so
// that the first wave starts the most expensive tiles and the cheap ones fill its tail; beyond kRows rows the
// batch's own order.  `tpc`: query tokens of a CTA.  `stage`: scratch of kRows int2.  found = {row or -1, tile}.
__device__ void find_tile(const Prefill8Args& p, int tpc, int want, int2* stage, int* found) {
  const int tid = threadIdx.x;
  auto geometry = [&](int b) -> int2 {  // (keys, tiles)
    const int qo = p.qo_indptr[b + 1] - p.qo_indptr[b];
    const int np = p.kv_indptr[b + 1] - p.kv_indptr[b];
    int ll = p.last_len[b];
    ll = ll < 1 ? 1 : (ll > p.page_size ? p.page_size : ll);
    return make_int2(np > 0 ? (np - 1) * p.page_size + ll : 0, qo > 0 ? (qo + tpc - 1) / tpc : 0);
  };
  if (tid == 0) found[0] = -1;
  if (p.batch <= p8::kRows) {
    int2 mine = make_int2(0, 0);
    if (tid < p.batch) stage[tid] = mine = geometry(tid);
    __syncthreads();
    if (tid < p.batch && mine.y > 0) {
      int first = 0;
      for (int o = 0; o < p.batch; ++o) {
        const int2 g = stage[o];
        if (g.x > mine.x || (g.x == mine.x && o < tid)) first += g.y;
      }
      if (want >= first && want < first + mine.y) {
        found[0] = tid;
        found[1] = mine.y - 1 - (want - first);
      }
    }
  } else {
    // thread i sums the tiles of its share of rows, one thread finds the share, then the row
    const int per = (p.batch + p8::kThreads - 1) / p8::kThreads;
    int sum = 0;
    for (int b = tid * per; b < min(p.batch, (tid + 1) * per); ++b) sum += geometry(b).y;
    stage[tid].x = sum;
    __syncthreads();
    if (tid == 0) {
      int first = 0, i = 0;
      while (i < p8::kThreads && first + stage[i].x <= want) first += stage[i++].x;
      if (i < p8::kThreads)
        for (int b = i * per; b < min(p.batch, (i + 1) * per); ++b) {
          const int n = geometry(b).y;
          if (want < first + n) {
            found[0] = b;
            found[1] = want - first;
            break;
          }
          first += n;
        }
    }
  }
  __syncthreads();
}

template <int D, bool E4M3>
__global__ void __launch_bounds__(p8::kThreads, 1)
    prefill8_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kvmap,
                    const __grid_constant__ CUtensorMap omap, const __grid_constant__ Prefill8Args p) {
  using namespace p8;
  using Cfg = P8Cfg<D>;
  constexpr int kHalves = Cfg::kHalves;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + kTiles * Cfg::kQBytes;
  uint8_t* sRaw = sKV + kStages * Cfg::kKV;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sRaw + kRaw * Cfg::kRawBytes);
  uint64_t* raw_full = q_full + 1;
  uint64_t* raw_empty = raw_full + kRaw;
  uint64_t* sc_full = raw_empty + kRaw;            // [group of the scale ring]
  uint64_t* kv_full = sc_full + kScaleRing;
  uint64_t* kv_empty = kv_full + kStages;          // [tile][stage]
  uint64_t* s_full = kv_empty + kTiles * kStages;  // [tile][S buffer]
  uint64_t* p_full = s_full + 2 * kTiles;
  uint64_t* o_done = p_full + 2 * kTiles;          // [tile][parity of the block]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_done + 2 * kTiles);
  int* found = reinterpret_cast<int*>(tmem_slot + 1);
  float* s_scale = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(q_full) + Cfg::kBars);  // [block][4][3]
  float* s_lse = s_scale + kScaleRing * 4 * 4 * 3;
  float* s_half = s_lse + kTiles * kM;  // [tile][half][row]
  int32_t* s_pages = reinterpret_cast<int32_t*>(s_half + 2 * kTiles * kM);

  const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
  const int S = gridDim.y, part = blockIdx.y;
  // KV head fastest: the heaviest tiles of every head start in the first wave
  const int kvh = blockIdx.x % p.hkv;
  const int G = p.group;
  const int tpt = kM / G;  // tokens per tile
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kRaw; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int s = 0; s < kScaleRing; ++s) mbar_init(&sc_full[s], 1);
    for (int s = 0; s < kStages; ++s) mbar_init(&kv_full[s], 4);
    for (int s = 0; s < kTiles * kStages; ++s) mbar_init(&kv_empty[s], 1);
    for (int b = 0; b < 2 * kTiles; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 8);
      mbar_init(&o_done[b], 1);
    }
    fence_barrier_init();
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kvmap);
  }
  if (warp == 0) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  find_tile(p, kTiles * tpt, static_cast<int>(blockIdx.x) / p.hkv, reinterpret_cast<int2*>(sKV), found);
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const int row = found[0];

  // blocks that each tile needs in all, and those of this CTA's part: [j0, j0 + nbt)
  int nbt[kTiles] = {0, 0};
  int q0 = 0, qo_len = 0, n_pages = 0, kv_len = 0, t_first = 0, shift = 0, j0 = 0;
  const int32_t* pages_g = p.indices;
  if (row >= 0) {
    q0 = p.qo_indptr[row];
    qo_len = p.qo_indptr[row + 1] - q0;
    n_pages = p.kv_indptr[row + 1] - p.kv_indptr[row];
    pages_g += p.kv_indptr[row];
    int ll = p.last_len[row];
    ll = ll < 1 ? 1 : (ll > p.page_size ? p.page_size : ll);
    kv_len = n_pages > 0 ? (n_pages - 1) * p.page_size + ll : 0;
    t_first = found[1] * kTiles * tpt;
    shift = kv_len - qo_len;
    int all = 0;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      const int f = t_first + t * tpt;
      const int t_last = min(qo_len, f + tpt) - 1;
      const int hi = min(kv_len, shift + t_last + 1);
      nbt[t] = t_last >= f && hi > 0 ? (hi + kN - 1) / kN : 0;
      all = max(all, nbt[t]);
    }
    const int per = (all + S - 1) / S;
    j0 = part * per;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) nbt[t] = max(0, min(nbt[t], j0 + per) - j0);
  }
  const int nb = max(nbt[0], nbt[1]);
  const bool have[kTiles] = {row >= 0 && t_first < qo_len, row >= 0 && t_first + tpt < qo_len};

  if (warp < 4) {
    reg_dec<40>();
    if (warp == 0) {
      if (lane == 0 && nb > 0) {
        const int nq = nbt[1] > 0 ? kTiles : 1;
        mbar_arrive_expect_tx(q_full, nq * tpt * G * D * 2);
        for (int t = 0; t < nq; ++t)
          for (int half = 0; half < kHalves; ++half)
            tma_load_3d(sQ + t * Cfg::kQBytes + half * (kM * 128), &qmap, q_full, half * 64, kvh * G,
                        q0 + t_first + t * tpt);
      }
    } else if (warp <= 2) {
      // ------------------------------------------------------------ MMA issuers
      // Per tile: S(0), S(1), then for every block j PV(j), S(j + 2); one thread's MMAs run in order, so S(j + 2)
      // overwrites p'(j) only after PV(j) has read it.
      // The whole warp runs the loop and one elected lane issues, so descriptors stay in uniform registers.
      const int t = warp - 1;
      const int nbx = nbt[t];
      if (nbx > 0) {
        constexpr uint32_t kIdescS = tc::idesc_bf16_f32(kM, kN, false, false);
        constexpr uint32_t kIdescPV = idesc_f16_f32_bmn(kM, D);
        const bool lead = tc::elect_one();
        auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
          const bool ok = __all_sync(kFull, mbar_wait(bar, parity, p.status));
          tc::fence_after_sync();
          return ok;
        };
        bool ok = wait(q_full, 0);
        const uint64_t q_desc = tc::smem_desc_sw128(smem_addr(sQ + t * Cfg::kQBytes), 16, 1024);
        const uint64_t k_desc = tc::smem_desc_sw128(smem_addr(sKV), 16, 1024);
        const uint64_t v_desc = tc::smem_desc_sw128(smem_addr(sKV + kHalves * Cfg::kHalf), Cfg::kHalf, 1024);
        const uint32_t s_cols = tmem + t * 128, o_cols = tmem + kColO + t * 128;
        int ss = 0, ps = 0;  // stages of the next S and PV
        uint32_t s_phase = 0;
        auto issue_s = [&](int j) {
          ok = wait(&kv_full[ss], s_phase);
          if (!ok) return;
          if (lead) {
            const uint64_t kd = k_desc + static_cast<uint32_t>((ss * Cfg::kKV) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t qo = ((kk >> 2) * (kM * 128) + (kk & 3) * 32) >> 4;
              const uint32_t ko = ((kk >> 2) * Cfg::kHalf + (kk & 3) * 32) >> 4;
              tc::mma_f16_ss(s_cols + (j & 1) * kN, q_desc + qo, kd + ko, kIdescS, kk > 0 ? 1u : 0u);
            }
            tc::commit(&s_full[2 * t + (j & 1)]);
          }
          if (++ss == kStages) {
            ss = 0;
            s_phase ^= 1u;
          }
        };
        auto issue_pv = [&](int j) {
          const int sb = j & 1;
          ok = wait(&p_full[2 * t + sb], (j >> 1) & 1);
          if (!ok) return;
          if (lead) {
            const uint64_t vd = v_desc + static_cast<uint32_t>((ps * Cfg::kKV) >> 4);
#pragma unroll
            for (int ks = 0; ks < kN / 16; ++ks)
              tc::mma_f16_ts(o_cols, s_cols + sb * kN + (ks >> 1) * 32 + (ks & 1) * 8, vd + ((ks * 2048) >> 4), kIdescPV,
                             (j > 0 || ks > 0) ? 1u : 0u);
            tc::commit(&o_done[2 * t + sb]);
            tc::commit(&kv_empty[t * kStages + ps]);
          }
          if (++ps == kStages) ps = 0;
        };
        for (int j = 0; j < 2 && j < nbx && ok; ++j) issue_s(j);
        for (int j = 0; j < nbx && ok; ++j) {
          issue_pv(j);
          if (ok && j + 2 < nbx) issue_s(j + 2);
        }
      }
    } else if (nb > 0) {
      // ------------------------------------------------------------ codes and scales
      const int tpp = p.page_size / kBlock;
      const uint32_t inv_tpp = static_cast<uint32_t>(0xffffffffu / static_cast<uint32_t>(tpp)) + 1u;  // tpp = 1: 0
      auto page_index = [&](int tile) -> int {
        return tpp == 1 ? tile : static_cast<int>(__umulhi(static_cast<uint32_t>(tile), inv_tpp));
      };
      const int first_page = page_index(j0 * 4);
      const int used = min(n_pages, page_index((j0 + nb) * 4 - 1) + 1) - first_page;
      const bool staged = used <= kPages;
      if (staged)
        for (int i = lane; i < used; i += 32) s_pages[i] = pages_g[first_page + i];
      __syncwarp();
      // page and block in it of 16-token tile `tile` of the row; total_pages where there is none
      auto locate = [&](int tile, int& blk) -> int {
        blk = 0;
        if (tile * kBlock >= kv_len) return p.total_pages;
        const int pi = page_index(tile);
        blk = tile - pi * tpp;
        const int page = staged ? s_pages[pi - first_page] : pages_g[pi];
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.total_pages)) {
          report(p.status, NQT_DEV_BAD_PAGE);
          return p.total_pages;
        }
        return page;
      };
      // lane: block lane / 8 of a group of four, tile (lane / 2) % 4, K (even) or V (odd)
      auto load_scale = [&](int group) -> float {
        const int in = group * 16 + (lane >> 1);  // tile of this CTA's part
        if (in >= nb * 4) return 0.f;
        int blk;
        const int page = locate(j0 * 4 + in, blk);
        if (page >= p.total_pages) return 0.f;
        return __ldg(p.scales + ((static_cast<int64_t>(page) * 2 + (lane & 1)) * tpp + blk) * p.hkv + kvh);
      };
      float sc = load_scale(0);
      bool ok = true;
      int issued = 0;
      for (int j = 0; j < nb; ++j) {
        const int s = j % kRaw;
        if (j >= kRaw) ok = mbar_wait(&raw_empty[s], ((j / kRaw) - 1) & 1, p.status);
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&raw_full[s], Cfg::kRawBytes);
        __syncwarp();
        if (lane < 4) {
          int blk;
          const int page = locate((j0 + j) * 4 + lane, blk);
          tma_load_4d(sRaw + s * Cfg::kRawBytes + lane * (2 * kBlock * D), &kvmap, &raw_full[s], 0, kvh, blk * kBlock,
                      page * 2);
        }
        issued = j + 1;
        if ((j & 3) == 0) {
          // the ring holds 16 blocks; this warp is at most kRaw + kStages + 1 ahead of the softmax
          const int group = j >> 2;
          float* f = s_scale + (((group % kScaleRing) * 16 + (lane >> 1)) * 3);
          if (lane & 1) {
            const float c = fmaxf(sc, 8.271806e-25f);  // 2^-80
            f[1] = log2f(c);
            f[2] = __fdiv_rn(1.f, c);
          } else {
            f[0] = fmaxf(sc * p.scale_log2, 1.17549435e-38f);  // a masked -inf times it stays -inf
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[group % kScaleRing]);
          if (j + 4 < nb) sc = load_scale(group + 1);
        }
      }
      // the last copies have landed before the CTA leaves, also when a wait gave up
      for (int j = max(0, issued - kRaw); j < issued; ++j) mbar_wait(&raw_full[j % kRaw], (j / kRaw) & 1, p.status);
    }
    if (S > 1) {  // the join's two barriers belong to every thread of the cluster
      gemm_detail::cluster_arrive();
      gemm_detail::cluster_wait();
      gemm_detail::cluster_arrive();
      gemm_detail::cluster_wait();
    }
    __syncwarp();
    tc::fence_before_sync();
    bar_sync(0, kThreads);
    if (warp == 0) {
      tc::fence_after_sync();
      tc::tmem_dealloc(tmem, 512);
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------ converters
    reg_inc<88>();
    {
      const int ct = threadIdx.x - 128;
      constexpr int kChunks = D / 16;       // 16-code chunks of a row
      constexpr int kStep = 128 / kChunks;  // tokens that the 128 threads cover at once
      constexpr int kIter = kN / kStep;
      const int chunk = ct % kChunks, tok0 = ct / kChunks;
      // Where the thread's chunk lies in a raw tile pair, and its two 16-byte pieces in the token's 128-byte line,
      // swizzled by the token (kStep is a multiple of 8, so the same for all of its tokens).  The two halves of a row
      // write their pieces in opposite order, so that a quarter-warp's stores meet no bank twice.
      const uint32_t raw0 = (tok0 / kBlock) * (2 * kBlock * D) + (tok0 % kBlock) * D + chunk * 16;
      const int c = (chunk & 3) * 2, flip = (chunk >> 2) & 1;
      const uint32_t line = (chunk >> 2) * Cfg::kHalf + tok0 * 128;
      const uint32_t at0 = line + (((c + flip) ^ (tok0 & 7)) << 4), at1 = line + (((c + 1 - flip) ^ (tok0 & 7)) << 4);
      bool ok = true;
      for (int j = 0; j < nb && ok; ++j) {
        const int rs = j % kRaw, s = j % kStages;
        ok = mbar_wait(&raw_full[rs], (j / kRaw) & 1, p.status);
        if (j >= kStages) {
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            if (j - kStages < nbt[t] && !mbar_wait(&kv_empty[t * kStages + s], ((j / kStages) - 1) & 1, p.status))
              ok = false;
        }
        ok = __all_sync(kFull, ok);
        if (!ok) break;
        const uint8_t* raw = sRaw + rs * Cfg::kRawBytes + raw0;
        uint4 k[kIter], v[kIter];
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
          k[i] = *reinterpret_cast<const uint4*>(raw + i * (kStep * 2 * D));
          v[i] = *reinterpret_cast<const uint4*>(raw + i * (kStep * 2 * D) + kBlock * D);
        }
        const int left = kv_len - (j0 + j) * kN;  // tokens of the block that exist
        if (E4M3 && left < kN) {  // what lies behind them may be NaN codes, which no probability of 0 silences
#pragma unroll
          for (int i = 0; i < kIter; ++i)
            if (tok0 + i * kStep >= left) v[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        uint8_t* st = sKV + s * Cfg::kKV;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
          uint32_t o[8];
          codes_to_bf16<E4M3>(k[i].x, o[0], o[1]);
          codes_to_bf16<E4M3>(k[i].y, o[2], o[3]);
          codes_to_bf16<E4M3>(k[i].z, o[4], o[5]);
          codes_to_bf16<E4M3>(k[i].w, o[6], o[7]);
          *reinterpret_cast<uint4*>(st + at0 + i * (kStep * 128)) = flip ? make_uint4(o[4], o[5], o[6], o[7]) : make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(st + at1 + i * (kStep * 128)) = flip ? make_uint4(o[0], o[1], o[2], o[3]) : make_uint4(o[4], o[5], o[6], o[7]);
        }
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
          uint32_t o[8];
          codes_to_f16_rows<E4M3>(v[i].x, o[0], o[1]);
          codes_to_f16_rows<E4M3>(v[i].y, o[2], o[3]);
          codes_to_f16_rows<E4M3>(v[i].z, o[4], o[5]);
          codes_to_f16_rows<E4M3>(v[i].w, o[6], o[7]);
          uint8_t* sv = st + kHalves * Cfg::kHalf + i * (kStep * 128);
          *reinterpret_cast<uint4*>(sv + at0) = flip ? make_uint4(o[4], o[5], o[6], o[7]) : make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(sv + at1) = flip ? make_uint4(o[0], o[1], o[2], o[3]) : make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&raw_empty[rs]);
          mbar_arrive(&kv_full[s]);
        }
      }
    }
    if (S > 1) {  // the join's two barriers belong to every thread of the cluster
      gemm_detail::cluster_arrive();
      gemm_detail::cluster_wait();
      gemm_detail::cluster_arrive();
      gemm_detail::cluster_wait();
    }
    bar_sync(0, kThreads);
  } else {
    // ------------------------------------------------------------ softmax
    reg_inc<88>();
    const int t = (warp - 8) >> 3, h = ((warp - 8) >> 2) & 1;
    const int nbx = nbt[t];
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // tile row = TMEM lane
    const int pair = 5 + t * 4 + quarter;  // barrier of the two warps that share 32 rows
    const uint32_t t_row = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t col_s = t * 128 + h * 32, col_o = kColO + t * 128 + h * (D / 2);
    uint64_t* sfull = s_full + 2 * t;
    uint64_t* pfull = p_full + 2 * t;
    uint64_t* odone = o_done + 2 * t;
    float* mine = s_half + (t * 2 + h) * kM + r;
    const float* other = s_half + (t * 2 + 1 - h) * kM + r;
    const int lim = min(shift + t_first + t * tpt + r / G, kv_len - 1);  // last key that this row sees
    const float NEG_INF = -__int_as_float(0x7f800000);
    float m_used = NEG_INF, l = 0.f;
    bool ok = true;
    // a warp whose wait gave up goes on to the barriers that its partner waits in
    for (int j = 0; j < nbx; ++j) {
      const int sb = j & 1, s = j % (4 * kScaleRing);
      if (ok && (j & 3) == 0) ok = mbar_wait(&sc_full[(j >> 2) % kScaleRing], ((j >> 2) / kScaleRing) & 1, p.status);
      if (ok) ok = mbar_wait(&sfull[sb], (j >> 1) & 1, p.status);
      ok = __all_sync(kFull, ok);
      tc::fence_after_sync();
      uint32_t sr[32];
      tc::ld_32x32b_x32(t_row + col_s + sb * kN, sr);
      float fk[2], fe[2], fv[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float* f = s_scale + (s * 4 + h * 2 + g) * 3;
        fk[g] = f[0];
        fe[g] = f[1];
        fv[g] = f[2];
      }
      tc::wait_ld();
      const int last = lim - (j0 + j) * kN - h * 32;  // columns behind it are hidden
      if (last < 31) {
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if (c > last) sr[c] = __float_as_uint(NEG_INF);
      }
      float mx = NEG_INF;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint32_t* x = sr + g * 16;
        float a = max3(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
        float b = max3(__uint_as_float(x[3]), __uint_as_float(x[4]), __uint_as_float(x[5]));
        a = max3(a, __uint_as_float(x[6]), __uint_as_float(x[7]));
        b = max3(b, __uint_as_float(x[8]), __uint_as_float(x[9]));
        a = max3(a, __uint_as_float(x[10]), __uint_as_float(x[11]));
        b = max3(b, __uint_as_float(x[12]), __uint_as_float(x[13]));
        a = max3(a, __uint_as_float(x[14]), __uint_as_float(x[15]));
        mx = fmaxf(mx, fmaf(fmaxf(a, b), fk[g], fe[g]));
      }
      // the reference moves where either half of a row asks for it; until it has one, at the first key
      if (bar_any(pair, 64, ok && mx > m_used + 7.f)) {
        *mine = mx;
        bar_sync(pair, 64);
        const float m_new = fmaxf(m_used, fmaxf(mx, *other));
        const bool move = m_new > m_used + 7.f;
        // rescale this warp's half of the O rows once PV(j - 1) has landed
        if (j > 0) {
          if (ok) ok = mbar_wait(&odone[(j - 1) & 1], ((j - 1) >> 1) & 1, p.status);
          ok = __all_sync(kFull, ok);
          tc::fence_after_sync();
          const float alpha = move ? ex2(m_used - m_new) : 1.f;
#pragma unroll
          for (int ch = 0; ch < D / 32; ++ch) {
            uint32_t o[16];
            tc::ld_32x32b_x16(t_row + col_o + ch * 16, o);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tc::st_32x32b_x16(t_row + col_o + ch * 16, o);
          }
          tc::wait_st();
          l *= alpha;
        }
        if (move) m_used = m_new;
      }
      const float ref = m_used == NEG_INF ? 0.f : m_used;  // a row that has seen no key yet
      uint32_t pk[16];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint64_t c2 = pk2(fk[g], fk[g]);
        const float off = fe[g] - ref + 8.f;
        const uint64_t o2 = pk2(off, off);
        uint64_t sum = pk2(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 8; q += 4) {
          float pv[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = g * 16 + 2 * (q + e);
            float lo, hi;
            unpk2(fma2(pk2(sr[i], sr[i + 1]), c2, o2), lo, hi);
            pv[2 * e] = ex2(lo);
            pv[2 * e + 1] = ex2(hi);
            pk[i / 2] = pack_f16x2(pv[2 * e], pv[2 * e + 1]);
          }
          sum = add2(sum, add2(add2(pk2(pv[0], pv[1]), pk2(pv[2], pv[3])), add2(pk2(pv[4], pv[5]), pk2(pv[6], pv[7]))));
        }
        float lo, hi;
        unpk2(sum, lo, hi);
        l = fmaf(lo + hi, fv[g], l);
      }
      tc::st_32x32b_x16(t_row + col_s + sb * kN, pk);
      tc::wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0 && ok) mbar_arrive(&pfull[sb]);
    }
    // epilogue: O / l
    ok = nbx > 0 && ok && mbar_wait(&odone[(nbx - 1) & 1], ((nbx - 1) >> 1) & 1, p.status);
    ok = __all_sync(kFull, ok);
    tc::fence_after_sync();
    bar_sync(pair, 64);  // the exchange's last readers
    *mine = l;
    bar_sync(pair, 64);
    l = h == 0 ? l + *other : *other + l;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (S == 1) {
      if (have[t]) {
        // bf16 into the tile's own Q buffer (its last reader, S(nbx - 1), is done) in the Q box layout; a tile with
        // all its tokens leaves through one TMA store per 64 dims, a ragged one row by row
        uint8_t* sO = sQ + t * Cfg::kQBytes;
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
          uint32_t o[32];
          tc::ld_32x32b_x32(t_row + col_o + ch * 32, o);
          tc::wait_ld();
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (ok && inv != 0.f) {
              w.x = pack_bf16x2(__uint_as_float(o[v * 8 + 0]) * inv, __uint_as_float(o[v * 8 + 1]) * inv);
              w.y = pack_bf16x2(__uint_as_float(o[v * 8 + 2]) * inv, __uint_as_float(o[v * 8 + 3]) * inv);
              w.z = pack_bf16x2(__uint_as_float(o[v * 8 + 4]) * inv, __uint_as_float(o[v * 8 + 5]) * inv);
              w.w = pack_bf16x2(__uint_as_float(o[v * 8 + 6]) * inv, __uint_as_float(o[v * 8 + 7]) * inv);
            }
            const int c = h * (D / 16) + ch * 4 + v;  // 16-byte piece of the row
            *reinterpret_cast<uint4*>(sO + (c >> 3) * (kM * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = w;
          }
        }
        const bool full = p.tma_out && t_first + (t + 1) * tpt <= qo_len;
        if (full) fence_proxy_async_smem();
        bar_sync(2 + t, 256);
        if (full) {
          if (h == 0 && quarter == 0 && lane == 0) {
            for (int half = 0; half < kHalves; ++half)
              tma_store_3d(&omap, sO + half * (kM * 128), half * 64, kvh * G, q0 + t_first + t * tpt);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          }
        } else {
          constexpr int kC = D / 8;  // 16-byte pieces of an output row
          for (int i = h * kM + r; i < kM * kC; i += 2 * kM) {
            const int rr = i / kC, c = i % kC;
            const int tok = t_first + t * tpt + rr / G;
            if (rr < tpt * G && tok < qo_len) {
              const uint4 v = *reinterpret_cast<const uint4*>(sO + (c >> 3) * (kM * 128) + rr * 128 +
                                                              (((c & 7) ^ (rr & 7)) << 4));
              __nv_bfloat16* dst = p.out + static_cast<int64_t>(q0 + tok) * p.o_st +
                                   static_cast<int64_t>(kvh * G + rr % G) * p.o_sh + c * 8;
              if (p.out16) {
                *reinterpret_cast<uint4*>(dst) = v;
              } else {
                const uint16_t* e = reinterpret_cast<const uint16_t*>(&v);
#pragma unroll
                for (int x = 0; x < 8; ++x) reinterpret_cast<uint16_t*>(dst)[x] = e[x];
              }
            }
          }
        }
      }
    } else {
      // the row's part: normalised O in fp32 over the KV stages (every reader of them is done once both tiles'
      // last products are: bar 4) and its log2-sum-exp; -inf for a part that saw no key
      bar_sync(4, 512);
      uint8_t* sO = sKV + t * (kM * D * 4);
      const bool any = ok && inv != 0.f;
      if (h == 0) s_lse[t * kM + r] = any ? m_used - 8.f + log2f(l) : NEG_INF;
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch) {
        uint32_t o[32];
        tc::ld_32x32b_x32(t_row + col_o + ch * 32, o);
        tc::wait_ld();
#pragma unroll
        for (int f = 0; f < 8; ++f) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (any)
            v = make_float4(__uint_as_float(o[f * 4]) * inv, __uint_as_float(o[f * 4 + 1]) * inv,
                            __uint_as_float(o[f * 4 + 2]) * inv, __uint_as_float(o[f * 4 + 3]) * inv);
          *reinterpret_cast<float4*>(sO + r * (D * 4) + (((h * (D / 8) + ch * 8 + f) ^ (r & 7)) << 4)) = v;
        }
      }
      // join: CTA `part` finishes every S-th slice of the 256 rows
      gemm_detail::cluster_arrive();
      gemm_detail::cluster_wait();
      constexpr int kF = D / 4;
      const int rows = kTiles * kM / S;
      for (int i = static_cast<int>(threadIdx.x) - 256; i < rows * kF; i += 512) {
        const int rr = part * rows + i / kF, f = i % kF;
        const int jt = rr / kM, jr = rr % kM;
        const int tok = t_first + jt * tpt + jr / G;
        if (row < 0 || jr >= tpt * G || tok >= qo_len) continue;
        const uint32_t lse_a = smem_addr(s_lse + rr);
        const uint32_t o_a = smem_addr(sKV + jt * (kM * D * 4) + jr * (D * 4) + ((f ^ (jr & 7)) << 4));
        float top = NEG_INF;
        for (int c = 0; c < S; ++c) top = fmaxf(top, ld_cluster_f32(gemm_detail::map_rank(lse_a, c)));
        const float ref = top == NEG_INF ? 0.f : top;
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < S; ++c) {
          const float w = exp2f(ld_cluster_f32(gemm_detail::map_rank(lse_a, c)) - ref);
          const float4 v = ld_cluster_f4(gemm_detail::map_rank(o_a, c));
          sum += w;
          acc.x = fmaf(w, v.x, acc.x);
          acc.y = fmaf(w, v.y, acc.y);
          acc.z = fmaf(w, v.z, acc.z);
          acc.w = fmaf(w, v.w, acc.w);
        }
        const float norm = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        __nv_bfloat16* dst = p.out + static_cast<int64_t>(q0 + tok) * p.o_st +
                             static_cast<int64_t>(kvh * G + jr % G) * p.o_sh + f * 4;
        const uint32_t lo = pack_bf16x2(acc.x * norm, acc.y * norm), hi = pack_bf16x2(acc.z * norm, acc.w * norm);
        if (p.out16) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
        } else {
          uint16_t* d = reinterpret_cast<uint16_t*>(dst);
          d[0] = static_cast<uint16_t>(lo);
          d[1] = static_cast<uint16_t>(lo >> 16);
          d[2] = static_cast<uint16_t>(hi);
          d[3] = static_cast<uint16_t>(hi >> 16);
        }
      }
      gemm_detail::cluster_arrive();  // nobody's shared memory goes away while it is read
      gemm_detail::cluster_wait();
    }
    tc::fence_before_sync();
    bar_sync(0, kThreads);
  }
}

// Rows of q (or out) as {D, heads, tokens} in boxes of 64 dims x G heads x (128 / G) tokens.
int encode_rows(CUtensorMap* map, const void* q, int64_t st, int64_t sh, int tokens, int hq, int group, int d) {
  auto encode = c8::get_encode();
  if (encode == nullptr) return NQT_ERR_CUDA;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(hq), static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(st) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(p8::kM / group)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? NQT_OK : NQT_ERR_CUDA;
}

// The layer's codes as {D, Hkv, P, pages x 2} in boxes of one head x 16 tokens x K and V, rows as they are.
int encode_codes(CUtensorMap* map, const void* layer, int total_pages, int page_size, int hkv, int d) {
  auto encode = c8::get_encode();
  if (encode == nullptr) return NQT_ERR_CUDA;
  const cuuint64_t D = static_cast<cuuint64_t>(d);
  cuuint64_t dims[4] = {D, static_cast<cuuint64_t>(hkv), static_cast<cuuint64_t>(page_size),
                        static_cast<cuuint64_t>(total_pages) * 2};
  cuuint64_t strides[3] = {D, static_cast<cuuint64_t>(hkv) * D, static_cast<cuuint64_t>(page_size) * hkv * D};
  cuuint32_t box[4] = {static_cast<cuuint32_t>(d), 1, kBlock, 2};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(layer), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? NQT_OK : NQT_ERR_CUDA;
}

template <int D, bool E4M3>
int launch_prefill8(const CUtensorMap& qmap, const CUtensorMap& kvmap, const CUtensorMap& omap,
                    const Prefill8Args& a, int total_q, cudaStream_t s) {
  using Cfg = P8Cfg<D>;
  static DeviceOnce once;
  once([] {
    cudaFuncSetAttribute(prefill8_kernel<D, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  });
  const int tokens_per_cta = p8::kTiles * (p8::kM / a.group);
  // an upper bound of the tiles: a row's last one may be ragged (empty rows have none)
  const int rows = a.batch < total_q ? a.batch : total_q;
  const int64_t tiles = (total_q + tokens_per_cta - 1) / tokens_per_cta + rows - 1;
  if (tiles * a.hkv > 0x7fffffff) return NQT_ERR_UNSUPPORTED;
  // few tiles: share each among a cluster, as long as the cluster's CTAs still find SMs
  int split = 1;
  while (split < 8 && tiles * a.hkv * split * 2 <= num_sms()) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.hkv), split);
  cfg.blockDim = dim3(p8::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1;
  attr.val.clusterDim.y = split;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, prefill8_kernel<D, E4M3>, qmap, kvmap, omap, a);
  if (err != cudaSuccess) {
    set_last_error("prefill_attention8", err);
    return NQT_ERR_CUDA;
  }
  return NQT_OK;
}

}  // namespace
}  // namespace nqt

using namespace nqt;

extern "C" int nqt_prefill_attention8(const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                                      const void* layer_cache, const float* layer_scales, int total_pages,
                                      int page_size, const int32_t* qo_indptr, const int32_t* kv_indptr,
                                      const int32_t* kv_indices, const int32_t* last_page_len, int batch,
                                      int total_q_tokens, int num_qo_heads, int num_kv_heads, int head_dim,
                                      float sm_scale, int code, void* out, int64_t out_stride_tok,
                                      int64_t out_stride_head, int32_t* status, void* stream) {
  int rc = c8::check_layer(layer_cache, layer_scales, total_pages, page_size, num_kv_heads, head_dim, code);
  if (rc != NQT_OK) return rc;
  if (!q || !qo_indptr || !kv_indptr || !kv_indices || !last_page_len || !out) return NQT_ERR_ARG;
  if (batch < 1 || total_q_tokens < 0 || num_qo_heads < 1 || num_qo_heads % num_kv_heads) return NQT_ERR_ARG;
  if (!(sm_scale >= 0.f)) return NQT_ERR_ARG;
  const int group = num_qo_heads / num_kv_heads;
  if (group > 8) return NQT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || q_stride_tok % 8 || q_stride_head % 8) return NQT_ERR_ARG;
  if (total_q_tokens == 0) return NQT_OK;
  CUtensorMap qmap, kvmap, omap{};
  rc = encode_rows(&qmap, q, q_stride_tok, q_stride_head, total_q_tokens, num_qo_heads, group, head_dim);
  if (rc == NQT_OK) rc = encode_codes(&kvmap, layer_cache, total_pages, page_size, num_kv_heads, head_dim);
  if (rc != NQT_OK) {
    set_last_message("prefill_attention8: cuTensorMapEncodeTiled failed");
    return rc;
  }
  Prefill8Args a{};
  a.scales = layer_scales;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.o_st = out_stride_tok;
  a.o_sh = out_stride_head;
  a.qo_indptr = qo_indptr;
  a.kv_indptr = kv_indptr;
  a.indices = kv_indices;
  a.last_len = last_page_len;
  a.status = status;
  a.batch = batch;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.group = group;
  a.page_size = page_size;
  a.total_pages = total_pages;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.out16 = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && out_stride_tok % 8 == 0 && out_stride_head % 8 == 0;
  a.tma_out = a.out16 && encode_rows(&omap, out, out_stride_tok, out_stride_head, total_q_tokens, num_qo_heads, group,
                                     head_dim) == NQT_OK;
  cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return code == NQT_E4M3 ? launch_prefill8<128, true>(qmap, kvmap, omap, a, total_q_tokens, s)
                            : launch_prefill8<128, false>(qmap, kvmap, omap, a, total_q_tokens, s);
  return code == NQT_E4M3 ? launch_prefill8<64, true>(qmap, kvmap, omap, a, total_q_tokens, s)
                          : launch_prefill8<64, false>(qmap, kvmap, omap, a, total_q_tokens, s);
}
