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
// An item of work is two 128-row query tiles of one row and KV head (a tile row is a token x query head of the group),
// which walk over blocks of 64 keys:
//   warp 0        items and their queries; owner of the TMEM.  Warps 1 and 2: MMA issuers of tile A and B
//   warp 3        brings the codes of a block by TMA (one box of 16 tokens, K and V, per lane) into a raw ring, and
//                 the scale factors of four blocks at a time
//   warps 4..7    converters: raw codes to 16 bits in the operands' 128-byte-swizzled layout
//   warps 8..23   softmax (8..15 tile A, 16..23 tile B), half of a query row's keys per thread
// TMEM: S double-buffered per tile, p' over its own S buffer, O per tile.  The two tiles share every converted
// block, which halves the conversions per product.  setmaxnreg gives the converters and softmax warps the registers
// that the others do not need; every role runs to its own end, with no code in common behind the split.
//
// The grid has a CTA per item, those with the most keys first.  A running CTA takes over the next one that has not
// started (cluster launch control), so barriers, TMEM and the tile order are set up once per SM, the next item's keys
// and first scores run under the last one's end, and the work stays balanced.
//
// When the items are too few for the GPU (late chunks of long prompts) a cluster of up to 8 CTAs shares one, each
// walking over a part of its keys; the parts are joined in the cluster's shared memory in CTA order, so there is no
// workspace and nothing depends on timing.
//
// Bound by the softmax warps: for a block the tensor pipe and MUFU each need about 1024 clocks and are busy 35 to 42 % of
// the time; 54 % of the issue slots are used, and the warps wait for TMEM loads, fixed latencies and one another.  On one
// B200 (16 query and 8 KV heads of 128), one call among others and in a captured graph: eight prompts of 2048 tokens 201
// and 186 us, eight first chunks of 128 to 1024 55 and 53, two chunks of 301 to 515 behind 9000 to 16001 tokens 172 and
// 166.
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
constexpr int kKStages = 3;   // converted blocks of keys
constexpr int kVStages = 4;   // and of values, which are needed longer
constexpr int kRaw = 2;       // raw blocks
constexpr int kScaleRing = 8;  // groups of up to four blocks whose scale factors are kept
constexpr int kThreads = 768;
constexpr int kPages = 1024;  // page ids of the row staged in shared memory
constexpr int kRows = 512;    // rows of the batch whose tiles are put in order
constexpr int kItems = 4;     // items that are set up or in work; the issuers look two ahead
constexpr int kUsers = 23;    // warps that read an item
constexpr uint32_t kColO = 256;
}  // namespace p8

template <int D>
struct P8Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kQBytes = p8::kM * D * 2;               // [half][128 rows][128 B]
  static constexpr int kHalf = p8::kN * 128;                   // [64 tokens][128 B]
  static constexpr int kBlockBytes = kHalves * kHalf;          // of K or V
  static constexpr int kKV = (p8::kKStages + p8::kVStages) * kBlockBytes;
  static constexpr int kRawBytes = 2 * p8::kN * D;             // [tile][K, V][16 tokens][D]
  static constexpr int kBars = 640;
  static constexpr int kScales = p8::kScaleRing * 4 * 4 * 3 * 4;  // [block][tile][score factor, log2 c, 1 / c]
  static constexpr int kTable = 8 * p8::kRows;                 // keys and tiles of every row
  static constexpr int kRowState = 5 * p8::kTiles * p8::kM * 4;  // log2-sum-exp, for the join; the halves' exchanges
  static constexpr int kSmem =
      1024 + p8::kTiles * kQBytes + kKV + p8::kRaw * kRawBytes + kBars + kScales + kRowState + kTable + 4 * p8::kPages;
  static_assert(kSmem <= 227 * 1024, "one CTA takes the SM's shared memory");
  static_assert(kKV + p8::kRaw * kRawBytes >= p8::kTiles * p8::kM * D * 4, "the join stages O over them");
};

struct Prefill8Args {
  const float* scales;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  const int32_t *qo_indptr, *kv_indptr, *indices, *last_len;
  int32_t* status;
  int batch, hq, hkv, group, page_size, total_pages;
  float scale_log2;
  int out_vec;  // bytes of a store that the output's rows allow: 32, 16 or 2
};

// A piece of work: two query tiles of one row and KV head, and the part of the keys that this CTA walks over.
struct Item {
  int row;  // -1: none
  int kvh, q0, qo_len, kv_len, n_pages, t_first;
  int j0, nbt[2];  // first block, and how many from there each tile needs
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

// Cluster launch control: ask for the index of a CTA of this grid that has not started yet (`result`: 16 bytes, 16-byte
// aligned, written asynchronously with 16 bytes on `bar`), and read the answer: its blockIdx.x, or -1 when none is left.
__device__ __forceinline__ void steal_cta(void* result, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_addr(result)),
               "r"(smem_addr(bar))
               : "memory");
}
__device__ __forceinline__ int stolen_cta(const void* result) {
  int x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\tld.shared.b128 h, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tmov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n\t}"
      : "=r"(x)
      : "r"(smem_addr(result))
      : "memory");
  return x;
}
__device__ __forceinline__ void store_32(void* dst, uint4 a, uint4 b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(a.x), "r"(a.y), "r"(a.z),
               "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
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

// The order of the tiles: those with the most keys first, so that the cheap ones fill the tail.  A row of L keys has
// tiles that see about L, L - tpc, L - 2 tpc, ... of them (`tpc`: query tokens of a CTA's tiles).  Beyond kRows rows the
// batch's own order.  make_table, by the whole CTA: table[i] = {keys, tiles} of row i, or, beyond kRows rows,
// {first tile, tiles} of the i-th share of the rows.
__device__ __forceinline__ int2 row_geometry(const Prefill8Args& p, int tpc, int b) {  // (keys, tiles)
  const int qo = p.qo_indptr[b + 1] - p.qo_indptr[b];
  const int np = p.kv_indptr[b + 1] - p.kv_indptr[b];
  int ll = p.last_len[b];
  ll = ll < 1 ? 1 : (ll > p.page_size ? p.page_size : ll);
  return make_int2(np > 0 ? (np - 1) * p.page_size + ll : 0, qo > 0 ? (qo + tpc - 1) / tpc : 0);
}

__device__ __forceinline__ int warp_prefix(int n) {  // sum over this and the lower lanes
  const int lane = threadIdx.x & 31;
  int sum = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, sum, o);
    if (lane >= o) sum += v;
  }
  return sum;
}

__device__ void make_table(const Prefill8Args& p, int tpc, int2* table) {
  const int tid = threadIdx.x;
  if (p.batch <= p8::kRows) {
    if (tid < p.batch) table[tid] = row_geometry(p, tpc, tid);
    __syncthreads();
    return;
  }
  const int per = (p.batch + p8::kRows - 1) / p8::kRows;
  if (tid < p8::kRows) {
    int tiles = 0;
    for (int b = tid * per; b < min(p.batch, (tid + 1) * per); ++b) tiles += row_geometry(p, tpc, b).y;
    table[tid].y = tiles;
  }
  __syncthreads();
  if (tid < 32) {
    int first = 0;
    for (int i = tid; i < p8::kRows; i += 32) {
      const int n = table[i].y, sum = warp_prefix(n);
      table[i].x = first + sum - n;
      first += __shfl_sync(kFull, sum, 31);
    }
  }
  __syncthreads();
}

// (row, tile) of tile `want` in that order, by one warp; row -1 where there is none.
__device__ int2 find_tile(const Prefill8Args& p, int tpc, int want, const int2* table) {
  const int lane = threadIdx.x & 31;
  if (p.batch <= p8::kRows) {
    // tiles that see at least e keys; the last one has that many more than `left` keys beyond a multiple of tpc
    auto count = [&](int e) -> int {
      int n = 0;
      for (int i = lane; i < p.batch; i += 32) {
        const int2 g = table[i];
        if (g.x >= e) n += min(g.y, (g.x - e) / tpc + 1);
      }
      return __reduce_add_sync(kFull, n);
    };
    int lo = INT32_MIN / 2, hi = 0;  // count(lo) > want >= count(hi)
    for (int i = lane; i < p.batch; i += 32) hi = max(hi, table[i].x);
    hi = __reduce_max_sync(kFull, hi) + 1;
    if (count(lo) <= want) return make_int2(-1, 0);
    for (int step = tpc; count(hi - step) <= want; step *= 2) hi -= step;
    lo = hi;
    for (int step = tpc; count(lo) <= want; step *= 2) lo -= step;
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      (count(mid) > want ? lo : hi) = mid;
    }
    int left = want - count(hi);  // of the tiles that see exactly lo keys, in the order of their rows
    for (int i0 = 0; i0 < p.batch; i0 += 32) {
      const int2 g = i0 + lane < p.batch ? table[i0 + lane] : make_int2(0, 0);
      const int back = (g.x - lo) / tpc;
      const uint32_t in = __ballot_sync(kFull, g.x >= lo && (g.x - lo) % tpc == 0 && back < g.y);
      if (left < __popc(in)) {
        const int src = __fns(in, 0, left + 1);
        return make_int2(i0 + src, __shfl_sync(kFull, g.y - 1 - back, src));
      }
      left -= __popc(in);
    }
    return make_int2(-1, 0);
  }
  int2 hit = make_int2(-1, 0);
  for (int i = lane; i < p8::kRows; i += 32) {
    const int2 e = table[i];
    if (want >= e.x && want < e.x + e.y) hit = make_int2(i, want - e.x);
  }
  const uint32_t who = __ballot_sync(kFull, hit.x >= 0);
  if (who == 0) return make_int2(-1, 0);
  const int per = (p.batch + p8::kRows - 1) / p8::kRows;
  const int src = __ffs(who) - 1, share = __shfl_sync(kFull, hit.x, src);
  const int end = min(p.batch, (share + 1) * per);
  int left = __shfl_sync(kFull, hit.y, src);
  for (int b0 = share * per; b0 < end; b0 += 32) {
    const int n = b0 + lane < end ? row_geometry(p, tpc, b0 + lane).y : 0;
    const int sum = warp_prefix(n);
    const uint32_t in = __ballot_sync(kFull, left < sum);
    if (in != 0) {
      const int w = __ffs(in) - 1;
      return make_int2(b0 + w, left - __shfl_sync(kFull, sum - n, w));
    }
    left -= __shfl_sync(kFull, sum, 31);
  }
  return make_int2(-1, 0);
}

// JOIN: a cluster of CTAs shares the keys of one item; else a CTA takes further items.
template <int D, bool E4M3, bool JOIN>
__global__ void __launch_bounds__(p8::kThreads, 1)
    prefill8_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kvmap,
                    const __grid_constant__ Prefill8Args p) {
  using namespace p8;
  using Cfg = P8Cfg<D>;
  constexpr int kHalves = Cfg::kHalves;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + kTiles * Cfg::kQBytes;
  uint8_t* sV = sKV + kKStages * Cfg::kBlockBytes;
  uint8_t* sRaw = sKV + Cfg::kKV;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sRaw + kRaw * Cfg::kRawBytes);  // [tile]
  uint64_t* q_empty = q_full + kTiles;             // (its last S is done)
  uint64_t* raw_full = q_empty + kTiles;
  uint64_t* raw_empty = raw_full + kRaw;
  uint64_t* sc_full = raw_empty + kRaw;            // [group of the scale ring]
  uint64_t* kv_full = sc_full + kScaleRing;        // [K stage], K and V of a block
  uint64_t* k_empty = kv_full + kKStages;          // of both tiles, as is v_empty
  uint64_t* v_empty = k_empty + kKStages;
  uint64_t* s_full = v_empty + kVStages;           // [tile][S buffer]
  uint64_t* p_full = s_full + 2 * kTiles;
  uint64_t* o_done = p_full + 2 * kTiles;          // [tile][S buffer]
  uint64_t* item_full = o_done + 2 * kTiles;       // [item % kItems]
  uint64_t* item_empty = item_full + kItems;
  uint64_t* steal_bar = item_empty + kItems;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(steal_bar + 1);
  uint8_t* s_steal = reinterpret_cast<uint8_t*>(q_full) + 400;                     // 16 bytes
  Item* s_item = reinterpret_cast<Item*>(reinterpret_cast<uint8_t*>(q_full) + 416);  // [kItems]
  static_assert((8 * kTiles + 2 * kRaw + kScaleRing + 2 * kKStages + kVStages + 2 * kItems + 1) * 8 + 4 <= 400, "barriers");
  static_assert(416 + kItems * sizeof(Item) <= Cfg::kBars, "items");
  float* s_scale = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(q_full) + Cfg::kBars);  // [block][4][3]
  float* s_lse = s_scale + kScaleRing * 4 * 4 * 3;
  float* s_half = s_lse + kTiles * kM;  // [tile][half][row]
  float* s_sum = s_half + 2 * kTiles * kM;
  int2* s_table = reinterpret_cast<int2*>(s_sum + 2 * kTiles * kM);
  int32_t* s_pages = reinterpret_cast<int32_t*>(s_table + kRows);

  const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
  const int S = JOIN ? gridDim.y : 1, part = JOIN ? blockIdx.y : 0;
  const int G = p.group;
  const int tpt = kM / G;  // tokens per tile
  if (threadIdx.x == 0) {
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
    }
    for (int s = 0; s < kRaw; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int s = 0; s < kScaleRing; ++s) mbar_init(&sc_full[s], 1);
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(&kv_full[s], 4);
      mbar_init(&k_empty[s], kTiles);
    }
    for (int s = 0; s < kVStages; ++s) mbar_init(&v_empty[s], kTiles);
    for (int b = 0; b < 2 * kTiles; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&p_full[b], 8);
      mbar_init(&o_done[b], 1);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kUsers);
    }
    mbar_init(steal_bar, 1);
    fence_barrier_init();
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kvmap);
  }
  if (warp == 0) {
    tc::tmem_alloc(tmem_slot, 512);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  make_table(p, kTiles * tpt, s_table);
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  // The next item, copied out of its slot; ok: false when the wait gave up.  Whole warps.
  auto next_item = [&](int it, bool& ok) -> Item {
    ok = __all_sync(kFull, mbar_wait(&item_full[it % kItems], (it / kItems) & 1, p.status));
    Item item = s_item[it % kItems];
    if (!ok) item.row = -1;
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[it % kItems]);
    return item;
  };

  if (warp < 4) {
    reg_dec<40>();
    if (warp == 0) {
      // ------------------------------------------------------------ items and queries
      int uses[kTiles] = {0, 0};
      int index = static_cast<int>(blockIdx.x);
      bool ok = true;
      for (int it = 0, steals = 0; ok;) {
        const bool more = !JOIN && index >= 0;
        Item item{};
        item.row = -1;
        if (index >= 0) {
          item.kvh = index % p.hkv;  // KV head fastest: the heaviest tiles of every head come first
          const int2 at = find_tile(p, kTiles * tpt, index / p.hkv, s_table);
          item.row = at.x;
          if (at.x >= 0) {
            item.q0 = p.qo_indptr[at.x];
            item.qo_len = p.qo_indptr[at.x + 1] - item.q0;
            item.n_pages = p.kv_indptr[at.x + 1] - p.kv_indptr[at.x];
            int ll = p.last_len[at.x];
            ll = ll < 1 ? 1 : (ll > p.page_size ? p.page_size : ll);
            item.kv_len = item.n_pages > 0 ? (item.n_pages - 1) * p.page_size + ll : 0;
            item.t_first = at.y * kTiles * tpt;
            int all = 0;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
              const int f = item.t_first + t * tpt;
              const int t_last = min(item.qo_len, f + tpt) - 1;
              const int hi = min(item.kv_len, item.kv_len - item.qo_len + t_last + 1);
              item.nbt[t] = t_last >= f && hi > 0 ? (hi + kN - 1) / kN : 0;
              all = max(all, item.nbt[t]);
            }
            const int per = (all + S - 1) / S;
            item.j0 = part * per;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) item.nbt[t] = max(0, min(item.nbt[t], item.j0 + per) - item.j0);
          }
        }
        // an index behind the last tile has no item; the end (row -1) is passed on when none is left to ask for
        if (item.row >= 0 || !more) {
          if (it >= kItems) ok = __all_sync(kFull, mbar_wait(&item_empty[it % kItems], ((it / kItems) - 1) & 1, p.status));
          if (ok && lane == 0) {
            s_item[it % kItems] = item;
            mbar_arrive(&item_full[it % kItems]);
          }
          ++it;
        }
        for (int t = 0; t < kTiles && ok; ++t) {
          if (item.row < 0 || item.nbt[t] == 0) continue;
          if (uses[t] > 0) ok = __all_sync(kFull, mbar_wait(&q_empty[t], (uses[t] - 1) & 1, p.status));
          if (ok && lane == 0) {
            mbar_arrive_expect_tx(&q_full[t], tpt * G * D * 2);
            for (int half = 0; half < kHalves; ++half)
              tma_load_3d(sQ + t * Cfg::kQBytes + half * (kM * 128), &qmap, &q_full[t], half * 64, item.kvh * G,
                          item.q0 + item.t_first + t * tpt);
          }
          ++uses[t];
        }
        const bool last = item.row < 0 && !more;
        if (more && ok) {
          // One item ahead: asked for when this one's queries are on their way.  (Eight prompts of 2048: 186 us, against
          // 212 when it is asked for with this one's last keys, and 245 with one item per CTA.)
          if (lane == 0) {
            mbar_arrive_expect_tx(steal_bar, 16);
            steal_cta(s_steal, steal_bar);
          }
          // also after a wait that gave up: the answer lands before the CTA leaves
          const bool answered = __all_sync(kFull, mbar_wait(steal_bar, steals++ & 1, p.status));
          ok = ok && answered;
          index = answered ? stolen_cta(s_steal) : -1;
          __syncwarp();
          fence_proxy_async_smem();  // the answer is read before the next one is written
        } else {
          index = -1;
        }
        if (last) break;
      }
    } else if (warp <= 2) {
      // ------------------------------------------------------------ MMA issuers
      // Per tile: S(0), S(1), then for every block j PV(j), S(j + 2); one thread's MMAs run in order, so S(j + 2)
      // overwrites p'(j) only after PV(j) has read it.  An item's first PV overwrites O; it has to wait for p', which the
      // softmax warps store after they have read the last item's O.
      // The whole warp runs the loop and one elected lane issues, so descriptors stay in uniform registers.
      const int t = warp - 1;
      constexpr uint32_t kIdescS = tc::idesc_bf16_f32(kM, kN, false, false);
      constexpr uint32_t kIdescPV = idesc_f16_f32_bmn(kM, D);
      const bool lead = tc::elect_one();
      auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        const bool ok = __all_sync(kFull, mbar_wait(bar, parity, p.status));
        tc::fence_after_sync();
        return ok;
      };
      const uint64_t q_desc = tc::smem_desc_sw128(smem_addr(sQ + t * Cfg::kQBytes), 16, 1024);
      const uint64_t k_desc = tc::smem_desc_sw128(smem_addr(sKV), 16, 1024);
      const uint64_t v_desc = tc::smem_desc_sw128(smem_addr(sV), Cfg::kHalf, 1024);
      const uint32_t s_cols = tmem + t * 128, o_cols = tmem + kColO + t * 128;
      int ss = 0, ps = 0;  // stages of the next S and PV
      uint32_t s_phase = 0;
      int cs = 0, cp = 0;  // S and PV of this tile so far: their buffer and its turn
      int uses = 0;
      bool ok = true;
      // The blocks of all items are one stream, in which S is two blocks ahead of PV.  find_s waits for the next block and
      // says what it is: 1 used by this tile, 2 its item's first, 4 its last; -1: no more.
      int it = 0, s_j = 0, s_nb = 0, s_nbx = 0;
      auto find_s = [&]() -> int {
        while (s_j == s_nb) {
          const Item item = next_item(it++, ok);
          if (item.row < 0) return -1;
          s_j = 0;
          s_nbx = item.nbt[t];
          s_nb = max(item.nbt[0], item.nbt[1]);
        }
        const int j = s_j++;
        if (j == 0 && s_nbx > 0) ok = wait(&q_full[t], uses++ & 1);
        if (ok) ok = wait(&kv_full[ss], s_phase);
        return j >= s_nbx ? 0 : 1 | (j == 0 ? 2 : 0) | (j == s_nbx - 1 ? 4 : 0);
      };
      auto issue_s = [&](int block) {
        if (block & 1) {
          if (lead) {
            const uint64_t kd = k_desc + static_cast<uint32_t>((ss * Cfg::kBlockBytes) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint32_t qo = ((kk >> 2) * (kM * 128) + (kk & 3) * 32) >> 4;
              const uint32_t ko = ((kk >> 2) * Cfg::kHalf + (kk & 3) * 32) >> 4;
              tc::mma_f16_ss(s_cols + (cs & 1) * kN, q_desc + qo, kd + ko, kIdescS, kk > 0 ? 1u : 0u);
            }
            tc::commit(&s_full[2 * t + (cs & 1)]);
            tc::commit(&k_empty[ss]);
            if (block & 4) tc::commit(&q_empty[t]);
          }
          ++cs;
        } else if (lane == 0) {
          mbar_arrive(&k_empty[ss]);  // only the other tile needs this block
        }
        if (++ss == kKStages) {
          ss = 0;
          s_phase ^= 1u;
        }
      };
      auto issue_pv = [&](int block) {
        if (block & 1) {
          const int sb = cp & 1;
          ok = wait(&p_full[2 * t + sb], (cp >> 1) & 1);
          if (!ok) return;
          if (lead) {
            const uint64_t vd = v_desc + static_cast<uint32_t>((ps * Cfg::kBlockBytes) >> 4);
#pragma unroll
            for (int ks = 0; ks < kN / 16; ++ks)
              tc::mma_f16_ts(o_cols, s_cols + sb * kN + (ks >> 1) * 32 + (ks & 1) * 8, vd + ((ks * 2048) >> 4), kIdescPV,
                             !(block & 2) || ks > 0 ? 1u : 0u);
            tc::commit(&v_empty[ps]);
            tc::commit(&o_done[2 * t + sb]);
          }
          ++cp;
        } else if (lane == 0) {
          mbar_arrive(&v_empty[ps]);
        }
        if (++ps == kVStages) ps = 0;
      };
      int a = find_s();
      if (a >= 0 && ok) issue_s(a);
      int b = a >= 0 && ok ? find_s() : -1;
      if (b >= 0 && ok) issue_s(b);
      while (a >= 0 && ok) {
        issue_pv(a);
        if (!ok) break;
        const int next = b >= 0 ? find_s() : -1;
        if (!ok) break;
        if (next >= 0) issue_s(next);
        a = b;
        b = next;
      }
    } else {
      // ------------------------------------------------------------ codes and scales
      const int tpp = p.page_size / kBlock;
      const uint32_t inv_tpp = static_cast<uint32_t>(0xffffffffu / static_cast<uint32_t>(tpp)) + 1u;  // tpp = 1: 0
      auto page_index = [&](int tile) -> int {
        return tpp == 1 ? tile : static_cast<int>(__umulhi(static_cast<uint32_t>(tile), inv_tpp));
      };
      int s = 0, issued = 0, group = 0;  // raw slot; blocks and groups so far
      uint32_t phase = 1;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const Item item = next_item(it, ok);
        if (!ok || item.row < 0) break;
        const int nb = max(item.nbt[0], item.nbt[1]);
        if (nb == 0) continue;
        const int32_t* pages_g = p.indices + p.kv_indptr[item.row];
        const int first_page = page_index(item.j0 * 4);
        const int used = min(item.n_pages, page_index((item.j0 + nb) * 4 - 1) + 1) - first_page;
        const bool staged = used <= kPages;
        __syncwarp();
        if (staged)
          for (int i = lane; i < used; i += 32) s_pages[i] = pages_g[first_page + i];
        __syncwarp();
        // page and block in it of 16-token tile `tile` of the row; total_pages where there is none
        auto locate = [&](int tile, int& blk) -> int {
          blk = 0;
          if (tile * kBlock >= item.kv_len) return p.total_pages;
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
        auto load_scale = [&](int j) -> float {
          const int in = j * 4 + (lane >> 1);  // tile of this CTA's part
          if (in >= nb * 4) return 0.f;
          int blk;
          const int page = locate(item.j0 * 4 + in, blk);
          if (page >= p.total_pages) return 0.f;
          return __ldg(p.scales + ((static_cast<int64_t>(page) * 2 + (lane & 1)) * tpp + blk) * p.hkv + item.kvh);
        };
        float sc = load_scale(0);
        for (int j = 0; j < nb; ++j) {
          if (issued >= kRaw) ok = __all_sync(kFull, mbar_wait(&raw_empty[s], phase, p.status));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&raw_full[s], Cfg::kRawBytes);
          __syncwarp();
          if (lane < 4) {
            int blk;
            const int page = locate((item.j0 + j) * 4 + lane, blk);
            tma_load_4d(sRaw + s * Cfg::kRawBytes + lane * (2 * kBlock * D), &kvmap, &raw_full[s], 0, item.kvh,
                        blk * kBlock, page * 2);
          }
          ++issued;
          if (++s == kRaw) {
            s = 0;
            phase ^= 1u;
          }
          if ((j & 3) == 0) {
            // a group's factors are read before its slot comes round: this warp is at most kRaw + kVStages blocks ahead
            float* f = s_scale + (((group % kScaleRing) * 16 + (lane >> 1)) * 3);
            if (lane & 1) {
              const float c = sc < 8.271806e-25f ? 8.271806e-25f : sc;  // 2^-80; NaN stays NaN
              f[1] = log2f(c);
              f[2] = __fdiv_rn(1.f, c);
            } else {
              const float k = sc * p.scale_log2;
              f[0] = k < 1.17549435e-38f ? 1.17549435e-38f : k;  // a masked -inf times it stays -inf
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_full[group % kScaleRing]);
            ++group;
            if (j + 4 < nb) sc = load_scale(j + 4);
          }
        }
      }
      // the last copies have landed before the CTA leaves, also when a wait gave up
      for (int j = max(0, issued - kRaw); j < issued; ++j) mbar_wait(&raw_full[j % kRaw], (j / kRaw) & 1, p.status);
    }
    if (JOIN) {  // the join's two barriers belong to every thread of the cluster
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
      int rs = 0, ks = 0, vs = 0, done = 0;  // raw slot, stages; blocks so far
      uint32_t r_phase = 0, k_phase = 1, v_phase = 1;
      bool ok = true;
      for (int it = 0; ok; ++it) {
        const Item item = next_item(it, ok);
        if (!ok || item.row < 0) break;
        const int nb = max(item.nbt[0], item.nbt[1]);
        for (int j = 0; j < nb; ++j) {
          ok = mbar_wait(&raw_full[rs], r_phase, p.status);
          if (done >= kKStages) ok = mbar_wait(&k_empty[ks], k_phase, p.status) && ok;
          if (done >= kVStages) ok = mbar_wait(&v_empty[vs], v_phase, p.status) && ok;
          ok = __all_sync(kFull, ok);
          if (!ok) break;
          const uint8_t* raw = sRaw + rs * Cfg::kRawBytes + raw0;
          uint4 k[kIter], v[kIter];
#pragma unroll
          for (int i = 0; i < kIter; ++i) {
            const uint2 k0 = *reinterpret_cast<const uint2*>(raw + i * (kStep * 2 * D) + flip * 8);
            const uint2 k1 = *reinterpret_cast<const uint2*>(raw + i * (kStep * 2 * D) + 8 - flip * 8);
            const uint2 v0 = *reinterpret_cast<const uint2*>(raw + i * (kStep * 2 * D) + kBlock * D + flip * 8);
            const uint2 v1 = *reinterpret_cast<const uint2*>(raw + i * (kStep * 2 * D) + kBlock * D + 8 - flip * 8);
            k[i] = make_uint4(k0.x, k0.y, k1.x, k1.y);
            v[i] = make_uint4(v0.x, v0.y, v1.x, v1.y);
          }
          const int left = item.kv_len - (item.j0 + j) * kN;  // tokens of the block that exist
          if (E4M3 && left < kN) {  // what lies behind them may be NaN codes, which no probability of 0 silences
#pragma unroll
            for (int i = 0; i < kIter; ++i)
              if (tok0 + i * kStep >= left) v[i] = make_uint4(0u, 0u, 0u, 0u);
          }
          uint8_t* st = sKV + ks * Cfg::kBlockBytes;
#pragma unroll
          for (int i = 0; i < kIter; ++i) {
            uint32_t o[8];
            codes_to_bf16<E4M3>(k[i].x, o[0], o[1]);
            codes_to_bf16<E4M3>(k[i].y, o[2], o[3]);
            codes_to_bf16<E4M3>(k[i].z, o[4], o[5]);
            codes_to_bf16<E4M3>(k[i].w, o[6], o[7]);
            *reinterpret_cast<uint4*>(st + at0 + i * (kStep * 128)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(st + at1 + i * (kStep * 128)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
#pragma unroll
          for (int i = 0; i < kIter; ++i) {
            uint32_t o[8];
            codes_to_f16_rows<E4M3>(v[i].x, o[0], o[1]);
            codes_to_f16_rows<E4M3>(v[i].y, o[2], o[3]);
            codes_to_f16_rows<E4M3>(v[i].z, o[4], o[5]);
            codes_to_f16_rows<E4M3>(v[i].w, o[6], o[7]);
            uint8_t* sv = sV + vs * Cfg::kBlockBytes + i * (kStep * 128);
            *reinterpret_cast<uint4*>(sv + at0) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(sv + at1) = make_uint4(o[4], o[5], o[6], o[7]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&raw_empty[rs]);
            mbar_arrive(&kv_full[ks]);
          }
          ++done;
          if (++rs == kRaw) {
            rs = 0;
            r_phase ^= 1u;
          }
          if (++ks == kKStages) {
            ks = 0;
            k_phase ^= 1u;
          }
          if (++vs == kVStages) {
            vs = 0;
            v_phase ^= 1u;
          }
        }
      }
    }
    if (JOIN) {  // the join's two barriers belong to every thread of the cluster
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
    float* my_sum = s_sum + (t * 2 + h) * kM + r;
    const float* other_sum = s_sum + (t * 2 + 1 - h) * kM + r;
    const int r_tok = r / G, r_head = r % G;
    const float NEG_INF = -__int_as_float(0x7f800000);
    int c = 0, group0 = 0;  // blocks of this tile and groups of scale factors so far
    bool ok = true;
    for (int it = 0;; ++it) {
      ok = mbar_wait(&item_full[it % kItems], (it / kItems) & 1, p.status) && ok;
      const Item& item = s_item[it % kItems];  // given back after the epilogue
      // the two warps of a row leave together: one that gave up would be missed in their barriers
      const bool none = bar_any(pair, 64, !ok || item.row < 0);
      if (none && !JOIN) break;
      const int nbx = none ? 0 : item.nbt[t];
      const int t_first = item.t_first + t * tpt;
      // the last key that this row sees, from this part's first
      const int lim = min(item.kv_len - item.qo_len + t_first + r_tok, item.kv_len - 1) - item.j0 * kN - h * 32;
      float m_used = NEG_INF, l = 0.f;
      // a warp whose wait gave up goes on to the barriers that its partner waits in
      for (int j = 0; j < nbx; ++j, ++c) {
        const int sb = c & 1, group = group0 + (j >> 2), s = group % kScaleRing * 4 + (j & 3);
        if (ok) ok = mbar_wait(&sfull[sb], (c >> 1) & 1, p.status);
        __syncwarp();
        // (after the scores: this tile may have passed over groups, and then only they say that the ring has come round)
        if (ok && (j & 3) == 0) ok = mbar_wait(&sc_full[group % kScaleRing], (group / kScaleRing) & 1, p.status);
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
        const int last = lim - j * kN;  // columns behind it are hidden
        if (last < 31) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (e > last) sr[e] = __float_as_uint(NEG_INF);
          // a NaN scale is for those who see one of its keys
#pragma unroll
          for (int g = 0; g < 2; ++g)
            if (last < g * 16) {
              fk[g] = 1.f;
              fe[g] = fv[g] = 0.f;
            }
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
            if (ok) ok = mbar_wait(&odone[(c - 1) & 1], ((c - 1) >> 1) & 1, p.status);
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
      group0 += (max(item.nbt[0], item.nbt[1]) + 3) >> 2;
      if (ok && nbx > 0) ok = mbar_wait(&odone[(c - 1) & 1], ((c - 1) >> 1) & 1, p.status);
      ok = __all_sync(kFull, ok);
      tc::fence_after_sync();
      *my_sum = l;
      bar_sync(pair, 64);
      l = h == 0 ? l + *other_sum : *other_sum + l;
      const bool any = ok && nbx > 0 && (l > 0.f || l != l);
      const float inv = any ? 1.f / l : 0.f;
      if constexpr (!JOIN) {
        const int tok = t_first + r_tok;
        __nv_bfloat16* dst = p.out + static_cast<int64_t>(item.q0 + tok) * p.o_st +
                             static_cast<int64_t>(item.kvh * G + r_head) * p.o_sh + h * (D / 2);
        const bool live = r < tpt * G && tok < item.qo_len;
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
          uint32_t o[32];
          tc::ld_32x32b_x32(t_row + col_o + ch * 32, o);
          tc::wait_ld();
          if (live) {
#pragma unroll
            for (int v = 0; v < 4; v += 2) {
              uint4 w[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t* x = o + (v + i) * 8;
                w[i] = make_uint4(0u, 0u, 0u, 0u);
                if (any)
                  w[i] = make_uint4(pack_bf16x2(__uint_as_float(x[0]) * inv, __uint_as_float(x[1]) * inv),
                                    pack_bf16x2(__uint_as_float(x[2]) * inv, __uint_as_float(x[3]) * inv),
                                    pack_bf16x2(__uint_as_float(x[4]) * inv, __uint_as_float(x[5]) * inv),
                                    pack_bf16x2(__uint_as_float(x[6]) * inv, __uint_as_float(x[7]) * inv));
              }
              __nv_bfloat16* to = dst + ch * 32 + v * 8;
              if (p.out_vec == 32) {
                store_32(to, w[0], w[1]);
              } else if (p.out_vec == 16) {
                *reinterpret_cast<uint4*>(to) = w[0];
                *reinterpret_cast<uint4*>(to + 8) = w[1];
              } else {
                const uint16_t* e = reinterpret_cast<const uint16_t*>(w);
#pragma unroll
                for (int i = 0; i < 16; ++i) reinterpret_cast<uint16_t*>(to)[i] = e[i];
              }
            }
          }
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&item_empty[it % kItems]);
      } else {
        // the row's part: normalised O in fp32 over the KV stages (every reader of them is done once both tiles'
        // last products are: bar 4) and its log2-sum-exp; -inf for a part that saw no key
        bar_sync(4, 512);
        uint8_t* sO = sKV + t * (kM * D * 4);
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
          const int tok = item.t_first + jt * tpt + jr / G;
          if (none || jr >= tpt * G || tok >= item.qo_len) continue;
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
          __nv_bfloat16* dst = p.out + static_cast<int64_t>(item.q0 + tok) * p.o_st +
                               static_cast<int64_t>(item.kvh * G + jr % G) * p.o_sh + f * 4;
          const uint32_t lo = pack_bf16x2(acc.x * norm, acc.y * norm), hi = pack_bf16x2(acc.z * norm, acc.w * norm);
          if (p.out_vec >= 16) {
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
        break;
      }
    }
    tc::fence_before_sync();
    bar_sync(0, kThreads);
  }
}

// Rows of q as {D, heads, tokens} in boxes of 64 dims x G heads x (128 / G) tokens.
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

template <int D, bool E4M3, bool JOIN>
int run_prefill8(const CUtensorMap& qmap, const CUtensorMap& kvmap, const Prefill8Args& a, int items, int split,
                 cudaStream_t s) {
  using Cfg = P8Cfg<D>;
  static DeviceOnce once;
  once([] {
    cudaFuncSetAttribute(prefill8_kernel<D, E4M3, JOIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items), split);
  cfg.blockDim = dim3(p8::kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1;
  attr.val.clusterDim.y = split;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = JOIN ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, prefill8_kernel<D, E4M3, JOIN>, qmap, kvmap, a);
  if (err != cudaSuccess) {
    set_last_error("prefill_attention8", err);
    return NQT_ERR_CUDA;
  }
  return NQT_OK;
}

template <int D, bool E4M3>
int launch_prefill8(const CUtensorMap& qmap, const CUtensorMap& kvmap, const Prefill8Args& a, int total_q,
                    cudaStream_t s) {
  const int tokens_per_cta = p8::kTiles * (p8::kM / a.group);
  // an upper bound of the tiles: a row's last one may be ragged (empty rows have none)
  const int rows = a.batch < total_q ? a.batch : total_q;
  const int64_t tiles = (total_q + tokens_per_cta - 1) / tokens_per_cta + rows - 1;
  if (tiles * a.hkv > 0x7fffffff) return NQT_ERR_UNSUPPORTED;
  const int items = static_cast<int>(tiles * a.hkv);
  // few tiles: share each among a cluster, as long as the cluster's CTAs still find SMs
  int split = 1;
  while (split < 8 && static_cast<int64_t>(items) * split * 2 <= num_sms()) split *= 2;
  return split > 1 ? run_prefill8<D, E4M3, true>(qmap, kvmap, a, items, split, s)
                   : run_prefill8<D, E4M3, false>(qmap, kvmap, a, items, 1, s);
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
  if (q_stride_tok <= 0 || q_stride_head <= 0) return NQT_ERR_ARG;
  if (total_q_tokens == 0) return NQT_OK;
  CUtensorMap qmap, kvmap;
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
  const auto rows_allow = [&](int bytes) {
    return reinterpret_cast<uintptr_t>(out) % bytes == 0 && out_stride_tok * 2 % bytes == 0 && out_stride_head * 2 % bytes == 0;
  };
  a.out_vec = rows_allow(32) ? 32 : rows_allow(16) ? 16 : 2;
  cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return code == NQT_E4M3 ? launch_prefill8<128, true>(qmap, kvmap, a, total_q_tokens, s)
                            : launch_prefill8<128, false>(qmap, kvmap, a, total_q_tokens, s);
  return code == NQT_E4M3 ? launch_prefill8<64, true>(qmap, kvmap, a, total_q_tokens, s)
                          : launch_prefill8<64, false>(qmap, kvmap, a, total_q_tokens, s);
}
