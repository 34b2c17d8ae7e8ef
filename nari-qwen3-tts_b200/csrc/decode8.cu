// Paged GQA decode attention over an 8-bit KV cache (layout and codes: cache8.cuh).
//
//   out[b, h] = softmax(q[b, h] . K[b, :, h / G]^T * sm_scale) V[b, :, h / G]
//
// over the (n_pages - 1) * P + last_page_len tokens of row b, one query per row.
//
// Mathematics.  With codes k_t, v_t and block scales a, c (16 tokens each), in log2 units and with a running
// reference M:
//   x_t = a sm_scale log2(e) (q . k_t),  y_t = x_t + log2 c,  p'_t = 2^(y_t - M + 8),
//   O = sum_t p'_t v_t,  l = sum_t p'_t / c,  out = O / l
// so a value's scale is a summand of an exponent.  q . k and p' v are fp16 tensor-core tiles with fp32
// accumulation: codes are exact in fp16; q is brought to [1, 2) by the power of two of its row maximum, which is
// exact for every element above 2^-14 of it; p' is rounded to fp16's 11 bits.  M follows the maximum of y, the
// weight with which a token's codes enter the output, and moves only when that grows by more than 7: p' lies below
// 2^15, fp16 reaches down to 2^-32 of the largest weight, and the accumulators are rarely rescaled.  Scales below
// 2^-80 count as 2^-80.
//
// Work split.  The KV of one KV-head group is a flat list of 16-token tiles;
// CTA c of n streams tiles [T c / n, T (c + 1) / n) across sequence borders, so
// every CTA moves the same bytes whatever the lengths are.  Where that makes no range
// much longer the rows are cut one by one instead: no CTA then loads a second query
// or joins twice.  The tile prefix is
// computed by every CTA from the row lengths (one read and a scan, which costs
// no more than reading a prefix that a plan kernel left), so the call is one
// launch.  A row that several CTAs cover leaves fp32 partials in the workspace.
// They are joined in two steps, 16 CTAs at a time: the warp that completes the
// ticket of 16 neighbours joins their parts into one, the warp that completes
// the row's ticket joins those.  One warp never reads more than 16 + n / 16
// parts, whatever the length, and the order is that of the CTAs: the result
// does not depend on which warp comes last.  No CTA waits for another.
//
// Data path.  A producer warp keeps STAGES tiles in flight with TMA boxes
// {one head, or two of 64 dims, 16 tokens, K and V}.  Four consumer warps: one for each of
// four KV heads, or two or four for each of fewer, which then take turns and
// join their states in shared memory at the end of a row.  A warp takes two
// tiles at a time: their products are independent, and the maximum's shuffles
// and the reference's check are paid once for both.
// Rows of 128 (64) bytes use the 128-byte (64-byte) swizzle, so ldmatrix reads
// eight rows without bank conflicts.  ldmatrix moves 16-bit units: as an A
// operand K's bytes 4t..4t+3 of a row become two fp16 pairs, and since a dot
// product does not mind the order of its terms q's fragments are loaded in that
// order; for V the transposing form delivers bytes (token, token + 1) x (dim,
// dim + 1), and one byte permutation sorts them into the fragments of two dims.
// P goes from the accumulator layout to the B layout with movmatrix.
//
// Bound by HBM for large batches and by a chain of dependent trips (row lengths,
// page ids, TMA, tickets: about 6 us) for small ones.  One B200, one call among others
// and in a captured graph: 1 row of 300 tokens 9.4 and 9.1 us; 64 rows of 64 to 2048
// tokens (16 query and 8 KV heads of 128) 35.9 and 35.5, 144 MB; 240 rows of 32 to 4096
// 176 to 191 and 172 to 176, 5.6 to 6.2 TB/s; five rows of 20001 to 98765 tokens (14 and
// 2 heads of 64) 30 and 30, 81 MB.
#include "cache8.cuh"

namespace nqt {
namespace {

using namespace c8;

constexpr int kMaxCtas = 1184;     // split CTAs of all head groups (8 per SM on 148 SMs)
constexpr int kMaxHpc = 4;         // KV heads of a CTA at most
constexpr int kMaxRows8 = 8192;    // rows whose prefix a CTA holds in shared memory
constexpr int kFewRows8 = 255;     // up to here the shared memory is sized alike, so its occupancy is asked for once
constexpr int kGroup8 = 16;        // CTAs whose parts are joined at once
constexpr int kMinTiles8 = 4;      // tiles of a CTA at least: shorter parts cost more to join than they save

constexpr size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// The workspace: tickets, zero between launches, then the split rows' parts.  A ticket belongs to a part's slot and KV
// head: those of a row's groups of CTAs to each group's first slot, the row's own to the row's first slot.  A launch has
// up to kMaxCtas CTAs of up to kMaxHpc KV heads with two slots each, so the tickets take the same bytes whatever the
// call's rows, heads and head size are, and no call's parts lie where another call's tickets do.
constexpr size_t kTickets8 = static_cast<size_t>(2) * kMaxCtas * kMaxHpc;

struct Ws8 {
  size_t groups, lse, o, total;  // the rows' tickets are at 0
};

constexpr Ws8 ws8_layout(int hq, int d) {
  Ws8 w{};
  w.groups = 4 * kTickets8;
  w.lse = up256(2 * w.groups);
  w.o = up256(w.lse + 4 * static_cast<size_t>(2 * kMaxCtas) * hq);
  w.total = up256(w.o + 4 * static_cast<size_t>(2 * kMaxCtas) * hq * d);
  return w;
}

struct Decode8Args {
  const __nv_bfloat16* q;
  int64_t q_st, q_sh;
  __nv_bfloat16* out;
  int64_t o_st, o_sh;
  const float* scales;
  const int32_t *indptr, *indices, *last_len;
  int32_t *tickets, *group_tickets;
  float *part_lse, *part_o;
  int32_t* status;
  int batch, hq, hkv, group, page_size, total_pages, n_ctas;
  int early;   // NQT_DECODE_OVERLAP_KV_WRITE
  int by_row;  // few rows: they may be cut one by one
  float scale_log2;
  uint64_t wait_ns;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 matrix of 16-bit elements held one row per quad.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int head, int tok, int pk,
                                         uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(0), "r"(head), "r"(tok), "r"(pk), "l"(policy)
      : "memory");
}

// Bounded pipeline wait; with NQT_DECODE_SHORT_WAIT (limit 0) one look at the barrier.
__device__ __forceinline__ bool pipe_wait(uint64_t* bar, uint32_t parity, const Decode8Args& p) {
  return mbar_wait_ns(bar, parity, p.status, p.wait_ns);
}

__device__ __forceinline__ int atomic_inc_acq_rel(int32_t* addr) {
  int32_t old;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(addr) : "memory");
  return old;
}

// First tile of CTA c of n, and the CTA that owns tile t.
__device__ __forceinline__ int64_t first_tile(int64_t total, int c, int n) { return total * c / n; }
__device__ __forceinline__ int tile_owner(int64_t total, int n, int64_t t) {
  return static_cast<int>(((t + 1) * n + total - 1) / total) - 1;
}

// Row that owns flat tile t: the last b with prefix[b] <= t.
__device__ __forceinline__ int row_of_tile(const int32_t* prefix, int batch, int64_t t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A CTA has at most two split rows: the one of its first tile leaves its part in slot 2c, one that starts later (and
// goes on behind the range) in slot 2c + 1.  `late`: the row starts inside its first CTA's range.
__device__ __forceinline__ int part_slot(int c, int ca, bool late) { return c == ca && late ? 2 * c + 1 : 2 * c; }

// Counts the warp in on a ticket (release of its stores, acquire of the others'); true for the one that completes
// it with `others` before, which leaves it at zero for the next launch.
__device__ __forceinline__ bool count_in(int32_t* ticket, int others, int lane) {
  int arrived = 0;
  if (lane == 0) {
    arrived = atomic_inc_acq_rel(ticket);
    if (arrived == others) *ticket = 0;
  }
  const bool last = __shfl_sync(kFull, arrived, 0) == others;
  __syncwarp();  // what lane 0 acquired is there for all
  return last;
}

// Joins `count` parts of one row and KV head: sum_i 2^(lse_i - M) O_i / sum_i 2^(lse_i - M) for every query head of
// the group, by WARPS warps of which this is number `sub`.  slot(i): the slot of part i.  Goes to `out` (last) or to slot
// `dst`, which may be slot(0), as a part.  The loads of two sets of heads and eight parts are in flight at once: a join is a chain of trips to
// L2.
template <int D, int WARPS, typename Slot>
__device__ __forceinline__ void join_parts(const Decode8Args& p, int row, int kvh, int count, Slot slot, bool last,
                                           int dst, int sub, int lane) {
  constexpr int QD = D / 4;    // float4 of a head
  constexpr int HP = 32 / QD;  // heads of a set: the warp's lanes
  constexpr int kBatch = 8;
  const float NEG_INF = -__int_as_float(0x7f800000);
  const int col = lane % QD;
  for (int g0 = 2 * HP * sub; g0 < p.group; g0 += 2 * HP * WARPS) {
    int head[2];
    bool live[2];
    float m[2], sum[2];
    float4 acc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int g = g0 + u * HP + lane / QD;
      live[u] = g < p.group;
      head[u] = kvh * p.group + (live[u] ? g : 0);
      m[u] = NEG_INF;
      sum[u] = 0.f;
      acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i0 = 0; i0 < count; i0 += kBatch) {
      float lse[2][kBatch];
      float4 v[2][kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          lse[u][k] = NEG_INF;
          v[u][k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i0 + k < count && live[u]) {
            const int64_t r = static_cast<int64_t>(slot(i0 + k)) * p.hq + head[u];
            lse[u][k] = __ldcg(p.part_lse + r);
            v[u][k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + r * D) + col);
          }
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float nm = m[u];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) nm = fmaxf(nm, lse[u][k]);
        const float ref = nm == NEG_INF ? 0.f : nm;
        const float a = ex2(m[u] - ref);
        m[u] = nm;
        sum[u] *= a;
        acc[u].x *= a;
        acc[u].y *= a;
        acc[u].z *= a;
        acc[u].w *= a;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (i0 + k >= count) continue;
          const float w = ex2(lse[u][k] - ref);
          sum[u] += w;
          acc[u].x = fmaf(w, v[u][k].x, acc[u].x);
          acc[u].y = fmaf(w, v[u][k].y, acc[u].y);
          acc[u].z = fmaf(w, v[u][k].z, acc[u].z);
          acc[u].w = fmaf(w, v[u][k].w, acc[u].w);
        }
      }
    }
    __syncwarp();  // slot `dst` may be one of the parts, and another lane may still be reading its log2-sum-exp
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!live[u]) continue;
      const float inv = 1.f / sum[u];
      if (last) {
        __nv_bfloat16* o = p.out + row * p.o_st + static_cast<int64_t>(head[u]) * p.o_sh + col * 4;
        *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(acc[u].x * inv, acc[u].y * inv);
        *reinterpret_cast<__nv_bfloat162*>(o + 2) = __floats2bfloat162_rn(acc[u].z * inv, acc[u].w * inv);
      } else {
        const int64_t r = static_cast<int64_t>(dst) * p.hq + head[u];
        __stcg(reinterpret_cast<float4*>(p.part_o + r * D) + col,
               make_float4(acc[u].x * inv, acc[u].y * inv, acc[u].z * inv, acc[u].w * inv));
        if (col == 0) __stcg(p.part_lse + r, m[u] + log2f(sum[u]));
      }
    }
  }
}

template <int D, int HPC, int STAGES>
struct Cfg8 {
  static constexpr int kWarps = 4;               // consumer warps
  static constexpr int kPerHead = kWarps / HPC;  // of one KV head
  static constexpr int kBoxHeads = D == 64 && HPC > 1 ? 2 : 1;  // heads of a TMA box: rows of 128 bytes if it can be
  static constexpr int kBoxRow = kBoxHeads * D;
  static constexpr int kBox = 2 * kBlock * kBoxRow;  // K then V of 16 tokens
  static constexpr int kBoxes = HPC / kBoxHeads;
  static constexpr int kStage = kBoxes * kBox;
  static constexpr int kThreads = (kWarps + 1) * 32;
  static constexpr int kState = 32 * (D / 4 + 4) * 4;  // a warp's O, m and l
  static constexpr int kJoin = HPC * (kPerHead - 1) * kState;
  static __host__ __device__ constexpr int smem(int rows) {
    return STAGES * kStage + 1024 + 2 * STAGES * 8 + kJoin + 4 * ((rows <= kFewRows8 ? 3 : 2) * (rows + 1)) + (rows + 3) / 4 * 4;
  }
};

template <int D, int HPC, int STAGES, bool E4M3>
__global__ void __launch_bounds__(160, 3) decode8_kernel(const __grid_constant__ CUtensorMap tmap,
                                                      const __grid_constant__ Decode8Args p) {
  using Cfg = Cfg8<D, HPC, STAGES>;
  constexpr int CH = D / 16;  // 16-byte chunks of a row
  constexpr int kWarps = Cfg::kWarps, kPerHead = Cfg::kPerHead;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::kStage);
  uint64_t* empty = full + STAGES;
  float* s_join = reinterpret_cast<float*>(empty + STAGES);  // [head][warp - 1][O, m, l][lane]
  int32_t* s_prefix = reinterpret_cast<int32_t*>(s_join + Cfg::kJoin / 4);  // [batch + 1] first tile of every row
  int32_t* s_base = s_prefix + p.batch + 1;       // [batch + 1] kv_indptr
  int32_t* s_first = s_base + p.batch + 1;        // [batch + 1] first CTA of every row (by_row)
  uint8_t* s_valid = reinterpret_cast<uint8_t*>(s_first + (p.by_row ? p.batch + 1 : 0));  // [batch] tokens of the row's last tile
  __shared__ int s_warp_sum[kWarps + 1];
  __shared__ int s_issued;
  __shared__ int s_progress[kWarps];
  __shared__ int s_fix[HPC][2];  // what a head's first warp tells the others

  // see nqt_decode_attention_ex: by default everything waits for the previous grid; with `early` only q, each
  // row's last tile and its scales, the workspace and all writes do
  if (!p.early) grid_dependency_wait();
  grid_dependents_launch();

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tpp = p.page_size / kBlock;

  // exclusive scan over the batch by the whole CTA; its sum
  auto scan = [&](auto value, int32_t* prefix) -> int {
    int carry = 0;
    for (int b0 = 0; b0 < p.batch; b0 += Cfg::kThreads) {
      const int b = b0 + threadIdx.x;
      const int mine = b < p.batch ? value(b) : 0;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) s_warp_sum[warp] = incl;
      __syncthreads();
      int before = carry, sum = 0;
#pragma unroll
      for (int w = 0; w < kWarps + 1; ++w) {
        if (w < warp) before += s_warp_sum[w];
        sum += s_warp_sum[w];
      }
      if (b < p.batch) prefix[b] = before + incl - mine;
      carry += sum;
      __syncthreads();
    }
    if (threadIdx.x == 0) prefix[p.batch] = carry;
    return carry;
  };
  // the rows' first tiles
  const int64_t total = scan(
      [&](int b) -> int {
        const int i0 = p.indptr[b], np = p.indptr[b + 1] - i0;
        int tiles = 0, valid = 0;
        if (np > 0) {
          int ll = p.last_len[b];
          ll = ll < 1 ? 1 : (ll > p.page_size ? p.page_size : ll);
          tiles = (np - 1) * tpp + (ll + kBlock - 1) / kBlock;
          valid = ll - (ll - 1) / kBlock * kBlock;
        }
        s_base[b] = i0;
        s_valid[b] = static_cast<uint8_t>(valid);
        return tiles;
      },
      s_prefix);
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], HPC);
    }
    fence_barrier_init();
  }
  __syncthreads();

  const int c = blockIdx.x;
  const int kv0 = blockIdx.y * HPC;
  // rows without a page are zeros (this CTA's heads of rows c, c + n_ctas, ...)
  for (int b = c; b < p.batch; b += p.n_ctas) {
    if (s_valid[b] != 0) continue;
    if (p.early) grid_dependency_wait();
    for (int i = threadIdx.x; i < HPC * p.group * D; i += Cfg::kThreads)
      p.out[b * p.o_st + static_cast<int64_t>(kv0 * p.group + i / D) * p.o_sh + i % D] = __float2bfloat16_rn(0.f);
  }
  // few tiles: fewer CTAs, so that each has some; every range is non-empty (n <= total)
  int n;
  int64_t t_begin, t_end;
  // Rows cut one by one make the longest range up to total / (n - rows) tiles, total * rows / (n (n - rows)) more than a
  // cut across rows, at some 0.5 us each, and save 3 us.  (One B200, 64 rows: of 33 to 100 tokens 11.9 us against 15.5,
  // of 333 to 1000 26.9 against 27.5, of 1000 to 3000 57.4 against 52.9.)
  const bool by_row = p.by_row && total * p.batch <= 5ll * p.n_ctas * (p.n_ctas - p.batch);
  if (by_row) {
    int per = static_cast<int>((total + p.n_ctas - p.batch - 1) / (p.n_ctas - p.batch));
    per = per < kMinTiles8 ? kMinTiles8 : per;
    n = scan([&](int b) -> int { return (s_prefix[b + 1] - s_prefix[b] + per - 1) / per; }, s_first);
    __syncthreads();
    if (c >= n) return;  // uniform over the block
    const int r = row_of_tile(s_first, p.batch, c);
    t_begin = s_prefix[r] + static_cast<int64_t>(c - s_first[r]) * per;
    t_end = t_begin + per < s_prefix[r + 1] ? t_begin + per : s_prefix[r + 1];
  } else {
    const int64_t want = (total + kMinTiles8 - 1) / kMinTiles8;
    n = want < p.n_ctas ? static_cast<int>(want) : p.n_ctas;
    if (c >= n) return;
    t_begin = first_tile(total, c, n);
    t_end = first_tile(total, c + 1, n);
  }
  // the CTAs of a row, and whether it starts inside the first one's range
  auto owners = [&](int row, int& ca, int& cb) -> bool {
    if (by_row) {
      ca = s_first[row];
      cb = s_first[row + 1] - 1;
      return false;
    }
    const int64_t t0 = s_prefix[row], t1 = s_prefix[row + 1];
    ca = tile_owner(total, n, t0);
    cb = tile_owner(total, n, t1 - 1);
    return first_tile(total, ca, n) < t0;
  };
  const int n_tiles = static_cast<int>(t_end - t_begin);

  if (warp == kWarps) {
    // ---------------------------------------------------------- producer
    // lane l looks up the page of tile 32 k + l of the range: one search and one load for 32 tiles, a chunk ahead
    auto look_up = [&](int i, int& page, int& tok) -> bool {  // whether the tile is its row's last
      page = p.total_pages;  // a box outside the map: TMA fills zeros
      tok = 0;
      if (i >= n_tiles) return false;
      const int64_t t = t_begin + i;
      const int r = row_of_tile(s_prefix, p.batch, t);
      const int in_row = static_cast<int>(t - s_prefix[r]);
      const int pl = in_row / tpp;
      tok = (in_row - pl * tpp) * kBlock;
      page = p.indices[s_base[r] + pl];
      return t == s_prefix[r + 1] - 1;
    };
    int page_n, tok_n;
    bool last_n = look_up(lane, page_n, tok_n);
    if (lane == 0) prefetch_tensormap(&tmap);
    uint64_t evict_first;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(evict_first));
    bool met = !p.early;
    int issued = 0;
    bool ready = true;
    for (int i0 = 0; i0 < n_tiles && ready; i0 += 32) {
      int page_c = page_n;
      const int tok_c = tok_n;
      const unsigned lasts = __ballot_sync(kFull, last_n);
      if (i0 + lane < n_tiles && static_cast<unsigned>(page_c) >= static_cast<unsigned>(p.total_pages)) {
        report(p.status, NQT_DEV_BAD_PAGE);
        page_c = p.total_pages;
      }
      last_n = look_up(i0 + 32 + lane, page_n, tok_n);
      for (int u = 0; u < 32 && i0 + u < n_tiles; ++u) {
        const int i = i0 + u, s = i % STAGES;
        if (!met && (lasts >> u & 1u)) {  // a row's last tile may come from the previous grid
          grid_dependency_wait();
          met = true;
        }
        if (i >= STAGES) ready = pipe_wait(&empty[s], ((i / STAGES) - 1) & 1, p);
        ready = __all_sync(kFull, ready);
        if (!ready) break;
        const int page = __shfl_sync(kFull, page_c, u), tok = __shfl_sync(kFull, tok_c, u);
        if (lane == 0) mbar_arrive_expect_tx(&full[s], Cfg::kStage);
        __syncwarp();
        if (lane < Cfg::kBoxes)
          tma_tile(smem + s * Cfg::kStage + lane * Cfg::kBox, &tmap, &full[s], kv0 / Cfg::kBoxHeads + lane, tok,
                   page * 2, evict_first);
        issued = i + 1;
      }
    }
    if (lane == 0) s_issued = issued;
  } else {
    // ------------------------------------------------------------ consumers
    const int hw = warp / kPerHead, sub = warp % kPerHead;  // head in the CTA, place among the head's warps
    const int kvh = kv0 + hw;
    const int g = lane >> 2, t4 = lane & 3;
    const int lm_j = lane >> 3, lm_r = lane & 7;
    const int group = p.group;
    const float NEG_INF = -__int_as_float(0x7f800000);

    // scales of up to 32 tiles ahead, one per lane; the page ids are a chunk further ahead
    auto tile_page = [&](int i) -> int {  // page of this lane's tile i, -1 past the range
      if (i >= n_tiles) return -1;
      const int r = row_of_tile(s_prefix, p.batch, t_begin + i);
      return p.indices[s_base[r] + static_cast<int>(t_begin + i - s_prefix[r]) / tpp];
    };
    auto tile_scales = [&](int i, int page, float& ks, float& vs) {
      ks = 0.f;
      vs = 1.f;  // a page outside the pool: keys and values of zeros
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.total_pages)) return;
      const int r = row_of_tile(s_prefix, p.batch, t_begin + i);
      const int blk = static_cast<int>(t_begin + i - s_prefix[r]) % tpp;
      const float* sp = p.scales + (static_cast<int64_t>(page) * 2 * tpp + blk) * p.hkv + kvh;
      ks = __ldcg(sp);  // from L2: the previous grid may have written neighbouring scales
      vs = __ldcg(sp + static_cast<int64_t>(tpp) * p.hkv);
    };
    // what a tile needs of its scales, per lane of the chunk: score factor, log2 c, 1 / c
    float ks_c, lc_c, rc_c;
    auto take = [&](float ks, float vs) {
      const float c = vs < 8.271806e-25f ? 8.271806e-25f : vs;  // 2^-80; NaN stays NaN
      ks_c = ks;
      lc_c = log2f(c);
      rc_c = __frcp_rn(c);
    };
    // query heads of the group: lane (g, t4) holds elements 16 ch + 4 t4 .. + 3 of head g
    auto load_q = [&](int r, uint32_t (&qf)[CH][2]) {
      const __nv_bfloat16* qrow = p.q + r * p.q_st + static_cast<int64_t>(kvh * group + g) * p.q_sh;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        qf[ch][0] = qf[ch][1] = 0u;
        if (g < group) {
          qf[ch][0] = *reinterpret_cast<const uint32_t*>(qrow + ch * 16 + 4 * t4);
          qf[ch][1] = *reinterpret_cast<const uint32_t*>(qrow + ch * 16 + 4 * t4 + 2);
        }
      }
    };
    int row = row_of_tile(s_prefix, p.batch, t_begin);
    uint32_t qf[CH][2];

    int chunk = 0;  // the 32 tiles whose factors are in ks_c, lc_c, rc_c; the next 32 scales are in ks_n, vs_n
    float ks_n, vs_n;
    int page_nx = tile_page(lane);
    if (p.early) grid_dependency_wait();  // q, the last tiles' scales, the parts and tickets of the last launch
    load_q(row, qf);
    bool q_ready = true;
    tile_scales(lane, page_nx, ks_n, vs_n);
    page_nx = tile_page(32 + lane);
    take(ks_n, vs_n);
    tile_scales(32 + lane, page_nx, ks_n, vs_n);
    page_nx = tile_page(64 + lane);
    auto factors_of = [&](int i, float& ks, float& lc, float& rc) {  // i does not fall
      while (chunk < (i >> 5)) {
        ++chunk;
        take(ks_n, vs_n);
        tile_scales((chunk + 1) * 32 + lane, page_nx, ks_n, vs_n);
        page_nx = tile_page((chunk + 2) * 32 + lane);
      }
      ks = __shfl_sync(kFull, ks_c, i & 31);
      lc = __shfl_sync(kFull, lc_c, i & 31);
      rc = __shfl_sync(kFull, rc_c, i & 31);
    };

    const int tok = ((lm_j & 1) << 3) + lm_r;  // ldmatrix row of this lane
    const int sw = Cfg::kBoxRow == 128 ? (tok & 7) : ((tok >> 1) & 3);
    const uint32_t box0 = smem_addr(smem) + hw / Cfg::kBoxHeads * Cfg::kBox + tok * Cfg::kBoxRow;
    uint32_t at[CH / 2];  // the lane's 16-byte chunk of each chunk pair, swizzled
#pragma unroll
    for (int i = 0; i < CH / 2; ++i)
      at[i] = static_cast<uint32_t>((hw % Cfg::kBoxHeads * CH + 2 * i + (lm_j >> 1)) ^ sw) << 4;
    int fix_a = -1, fix_b = -1;  // split rows whose group's ticket this warp completed
    int stop = n_tiles;          // first tile of this warp that was not consumed
    bool dead = false;           // a wait gave up: the rows are still gone through, so that every ticket completes

    for (int i0 = 0; i0 < n_tiles; ++row) {
      const int row_t0 = s_prefix[row], row_t1 = s_prefix[row + 1];
      const int i1 = static_cast<int>(row_t1 - t_begin < n_tiles ? row_t1 - t_begin : n_tiles);
      if (i1 <= i0) continue;  // a row without pages
      const bool ends = row_t1 - t_begin == i1;
      const int valid_last = ends ? s_valid[row] : kBlock;

      // the row's query heads of the group, as B fragments in K's byte order, scaled to a maximum in [1, 2)
      if (!q_ready) load_q(row, qf);
      q_ready = false;
      float f0, f1;  // score factors of heads 2 t4, 2 t4 + 1: q's power of two, sm_scale, log2 e
      {
        float amax = 0.f;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[ch][h]));
            amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(kFull, amax, 2));
        int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
        e = (amax == 0.f || e > 127) ? 0 : min(max(e, -126), 126);
        const float down = fp8::exp2_int(-e);
#pragma unroll
        for (int ch = 0; ch < CH; ++ch)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[ch][h]));
            qf[ch][h] = pack_f16x2(v.x * down, v.y * down);
          }
        f0 = fp8::exp2_int(__shfl_sync(kFull, e, 8 * t4)) * p.scale_log2;
        f1 = fp8::exp2_int(__shfl_sync(kFull, e, 8 * t4 + 4)) * p.scale_log2;
      }
      float o[CH][4];
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) o[ch][0] = o[ch][1] = o[ch][2] = o[ch][3] = 0.f;
      float m0 = NEG_INF, m1 = NEG_INF, l0 = 0.f, l1 = 0.f;  // references and sums of heads 2 t4, 2 t4 + 1

      for (int i = i0 + 2 * sub; i < i1 && !dead; i += 2 * kPerHead) {
        const bool two = i + 1 < i1;
        const int sA = i % STAGES, sB = (i + 1) % STAGES;
        float ksA, lcA, rcA, ksB = 0.f, lcB = 0.f, rcB = 0.f;
        factors_of(i, ksA, lcA, rcA);
        if (two) factors_of(i + 1, ksB, lcB, rcB);
        bool ok = pipe_wait(&full[sA], (i / STAGES) & 1, p);
        if (two) ok = pipe_wait(&full[sB], ((i + 1) / STAGES) & 1, p) && ok;
        if (!__all_sync(kFull, ok)) {
          dead = true;
          stop = i;
          break;
        }
        const uint32_t rowA = box0 + sA * Cfg::kStage, rowB = box0 + sB * Cfg::kStage;

        // S^T[tok][head] = sum_d K[tok][d] Q[head][d]
        auto scores = [&](uint32_t krow, float (&s)[4]) {
          float x[4] = {0.f, 0.f, 0.f, 0.f};
          s[0] = s[1] = s[2] = s[3] = 0.f;
#pragma unroll
          for (int cc = 0; cc < CH; cc += 2) {
            uint32_t r0, r1, r2, r3, a0, a1, a2, a3;
            ldmatrix_x4(r0, r1, r2, r3, krow + at[cc / 2]);
            codes_to_f16_rows<E4M3>(r0, a0, a2);
            codes_to_f16_rows<E4M3>(r1, a1, a3);
            mma_f16_16816(s, a0, a1, a2, a3, qf[cc][0], qf[cc][1]);
            codes_to_f16_rows<E4M3>(r2, a0, a2);
            codes_to_f16_rows<E4M3>(r3, a1, a3);
            mma_f16_16816(x, a0, a1, a2, a3, qf[cc + 1][0], qf[cc + 1][1]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] += x[e];
        };
        float sa[4], sb[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
        scores(rowA, sa);
        if (two) scores(rowB, sb);

        // online softmax (log2): the lane holds heads 2 t4 (0, 2) and 2 t4 + 1 (1, 3) of tokens g and g + 8
        const int validA = !two && i + 1 == i1 ? valid_last : kBlock;
        const int validB = two ? (i + 2 == i1 ? valid_last : kBlock) : 0;
        {
          const float c0 = ksA * f0, c1 = ksA * f1;
          sa[0] = g < validA ? fmaf(sa[0], c0, lcA) : NEG_INF;
          sa[1] = g < validA ? fmaf(sa[1], c1, lcA) : NEG_INF;
          sa[2] = g + 8 < validA ? fmaf(sa[2], c0, lcA) : NEG_INF;
          sa[3] = g + 8 < validA ? fmaf(sa[3], c1, lcA) : NEG_INF;
        }
        if (two) {
          const float c0 = ksB * f0, c1 = ksB * f1;
          sb[0] = g < validB ? fmaf(sb[0], c0, lcB) : NEG_INF;
          sb[1] = g < validB ? fmaf(sb[1], c1, lcB) : NEG_INF;
          sb[2] = g + 8 < validB ? fmaf(sb[2], c0, lcB) : NEG_INF;
          sb[3] = g + 8 < validB ? fmaf(sb[3], c1, lcB) : NEG_INF;
        }
        float x0 = fmaxf(fmaxf(sa[0], sa[2]), fmaxf(sb[0], sb[2]));
        float x1 = fmaxf(fmaxf(sa[1], sa[3]), fmaxf(sb[1], sb[3]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          x0 = fmaxf(x0, __shfl_xor_sync(kFull, x0, off));
          x1 = fmaxf(x1, __shfl_xor_sync(kFull, x1, off));
        }
        if (__any_sync(kFull, x0 > m0 + 7.f || x1 > m1 + 7.f)) {  // always on a row's first tiles (m = -inf)
          const float n0 = x0 > m0 + 7.f ? x0 : m0, n1 = x1 > m1 + 7.f ? x1 : m1;
          const float a0 = n0 == m0 ? 1.f : ex2(m0 - n0), a1 = n1 == m1 ? 1.f : ex2(m1 - n1);
          l0 *= a0;
          l1 *= a1;
          m0 = n0;
          m1 = n1;
#pragma unroll
          for (int ch = 0; ch < CH; ++ch) {
            o[ch][0] *= a0;
            o[ch][1] *= a1;
            o[ch][2] *= a0;
            o[ch][3] *= a1;
          }
        }
        const float r0 = m0 - 8.f, r1 = m1 - 8.f;

        // O^T[d][head] += sum_tok V[tok][d] P'[head][tok]; rows g and g + 8 of a chunk are its dims 2g and 2g + 1
        auto add_values = [&](uint32_t vrow, const float (&s)[4], float rc, int valid) {
          const float p0 = ex2(s[0] - r0), p1 = ex2(s[1] - r1), p2 = ex2(s[2] - r0), p3 = ex2(s[3] - r1);
          l0 = fmaf(p0 + p2, rc, l0);
          l1 = fmaf(p1 + p3, rc, l1);
          const uint32_t b0 = movmatrix_trans(pack_f16x2(p0, p1)), b1 = movmatrix_trans(pack_f16x2(p2, p3));
          // e4m3 codes behind the row's end may be NaN codes: they count as zeros
          uint32_t k0 = 0xffffffffu, k1 = 0xffffffffu;
          if (E4M3) {
            k0 = (2 * t4 < valid ? 0xffffu : 0u) | (2 * t4 + 1 < valid ? 0xffff0000u : 0u);
            k1 = (2 * t4 + 8 < valid ? 0xffffu : 0u) | (2 * t4 + 9 < valid ? 0xffff0000u : 0u);
          }
#pragma unroll
          for (int cc = 0; cc < CH; cc += 2) {
            uint32_t v0, v1, v2, v3, a0, a1, a2, a3;
            ldmatrix_x4_trans(v0, v1, v2, v3, vrow + at[cc / 2]);
            codes_to_f16_cols<E4M3>(v0, a0, a1);
            codes_to_f16_cols<E4M3>(v1, a2, a3);
            mma_f16_16816(o[cc], a0 & k0, a1 & k0, a2 & k1, a3 & k1, b0, b1);
            codes_to_f16_cols<E4M3>(v2, a0, a1);
            codes_to_f16_cols<E4M3>(v3, a2, a3);
            mma_f16_16816(o[cc + 1], a0 & k0, a1 & k0, a2 & k1, a3 & k1, b0, b1);
          }
        };
        add_values(rowA + kBlock * Cfg::kBoxRow, sa, rcA, validA);
        if (two) add_values(rowB + kBlock * Cfg::kBoxRow, sb, rcB, validB);
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&empty[sA]);
          if (two) mbar_arrive(&empty[sB]);
        }
      }

      if (kPerHead > 1) {
        // the head's other warps hand their states over; lane by lane they are the same elements
        float* mine = s_join + (hw * (kPerHead - 1) + (sub > 0 ? sub - 1 : 0)) * (Cfg::kState / 4) + lane;
        if (sub > 0) {
#pragma unroll
          for (int ch = 0; ch < CH; ++ch)
#pragma unroll
            for (int x = 0; x < 4; ++x) mine[(ch * 4 + x) * 32] = o[ch][x];
          mine[(CH * 4) * 32] = m0;
          mine[(CH * 4 + 1) * 32] = m1;
          mine[(CH * 4 + 2) * 32] = l0;
          mine[(CH * 4 + 3) * 32] = l1;
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + hw), "n"(kPerHead * 32) : "memory");
        if (sub == 0) {
#pragma unroll 1
          for (int w = 0; w < kPerHead - 1; ++w) {
            const float* s = mine + w * (Cfg::kState / 4);
            const float om0 = s[(CH * 4) * 32], om1 = s[(CH * 4 + 1) * 32];
            const float n0 = fmaxf(m0, om0), n1 = fmaxf(m1, om1);
            const float z0 = n0 == NEG_INF ? 0.f : n0, z1 = n1 == NEG_INF ? 0.f : n1;
            const float a0 = ex2(m0 - z0), a1 = ex2(m1 - z1), b0 = ex2(om0 - z0), b1 = ex2(om1 - z1);
            l0 = l0 * a0 + s[(CH * 4 + 2) * 32] * b0;
            l1 = l1 * a1 + s[(CH * 4 + 3) * 32] * b1;
            m0 = n0;
            m1 = n1;
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
              o[ch][0] = o[ch][0] * a0 + s[(ch * 4) * 32] * b0;
              o[ch][1] = o[ch][1] * a1 + s[(ch * 4 + 1) * 32] * b1;
              o[ch][2] = o[ch][2] * a0 + s[(ch * 4 + 2) * 32] * b0;
              o[ch][3] = o[ch][3] * a1 + s[(ch * 4 + 3) * 32] * b1;
            }
          }
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + hw), "n"(kPerHead * 32) : "memory");
      }

      if (sub == 0) {
        float t0 = l0, t1 = l1;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          t0 += __shfl_xor_sync(kFull, t0, off);
          t1 += __shfl_xor_sync(kFull, t1, off);
        }
        const float v0 = 1.f / t0, v1 = 1.f / t1;
        const int ha = kvh * group + 2 * t4;
        const bool has0 = 2 * t4 < group, has1 = 2 * t4 + 1 < group;
        if (t_begin <= row_t0 && ends) {
          __nv_bfloat16* ob = p.out + row * p.o_st + static_cast<int64_t>(ha) * p.o_sh + 2 * g;
#pragma unroll
          for (int ch = 0; ch < CH; ++ch) {
            if (has0)
              *reinterpret_cast<__nv_bfloat162*>(ob + ch * 16) = __floats2bfloat162_rn(o[ch][0] * v0, o[ch][2] * v0);
            if (has1)
              *reinterpret_cast<__nv_bfloat162*>(ob + p.o_sh + ch * 16) =
                  __floats2bfloat162_rn(o[ch][1] * v1, o[ch][3] * v1);
          }
        } else {
          int ca, cb;
          const bool late = owners(row, ca, cb);
          const int slot = part_slot(c, ca, late);
          float* po = p.part_o + (static_cast<int64_t>(slot) * p.hq + ha) * D + 2 * g;
          float* pl = p.part_lse + static_cast<int64_t>(slot) * p.hq + ha;
#pragma unroll
          for (int ch = 0; ch < CH; ++ch) {
            if (has0) __stcg(reinterpret_cast<float2*>(po + ch * 16), make_float2(o[ch][0] * v0, o[ch][2] * v0));
            if (has1) __stcg(reinterpret_cast<float2*>(po + D + ch * 16), make_float2(o[ch][1] * v1, o[ch][3] * v1));
          }
          if (g == 0) {
            if (has0) __stcg(pl, m0 - 8.f + log2f(t0));
            if (has1) __stcg(pl + 1, m1 - 8.f + log2f(t1));
          }
          __syncwarp();
          const int lo = c - (c - ca) % kGroup8, hi = min(cb, lo + kGroup8 - 1);  // the CTAs joined with this one
          if (count_in(p.group_tickets + part_slot(lo, ca, late) * p.hkv + kvh, hi - lo, lane)) {
            if (fix_a < 0) fix_a = row;  // only a range's first and last rows can be split
            else fix_b = row;
          }
        }
      }
      i0 = i1;
    }

    // joins, behind the tile loop: its accumulators are dead here; a head's warps share the query heads
    auto head_sync = [&]() {
      if (kPerHead > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + hw), "n"(kPerHead * 32) : "memory");
      else __syncwarp();
    };
    if (kPerHead > 1) {
      if (sub == 0 && lane == 0) {
        s_fix[hw][0] = fix_a;
        s_fix[hw][1] = fix_b;
      }
      head_sync();
      fix_a = s_fix[hw][0];
      fix_b = s_fix[hw][1];
    }
    for (int f = 0; f < 2; ++f) {
      const int r = f == 0 ? fix_a : fix_b;
      if (r < 0) continue;
      int ca, cb;
      const bool late = owners(r, ca, cb);
      const int lo = c - (c - ca) % kGroup8, hi = min(cb, lo + kGroup8 - 1);
      const int groups = (cb - ca) / kGroup8;  // less one
      join_parts<D, kPerHead>(p, r, kvh, hi - lo + 1, [&](int i) { return part_slot(lo + i, ca, late); }, groups == 0,
                              part_slot(lo, ca, late), sub, lane);
      if (groups == 0) continue;
      head_sync();
      int32_t* ticket = p.tickets + part_slot(ca, ca, late) * p.hkv + kvh;
      bool whole;
      if (kPerHead > 1) {
        if (sub == 0) {
          const bool w = count_in(ticket, groups, lane);
          if (lane == 0) s_fix[hw][f] = w;
        }
        head_sync();
        whole = s_fix[hw][f] != 0;
      } else {
        whole = count_in(ticket, groups, lane);
      }
      if (whole)
        join_parts<D, kPerHead>(
            p, r, kvh, groups + 1, [&](int i) { return part_slot(ca + i * kGroup8, ca, late); }, true, 0, sub, lane);
    }
    if (lane == 0) s_progress[warp] = stop;
  }
  // When a wait gave up, copies that were issued but not consumed may still land: wait for them before leaving.
  __syncthreads();
  if (threadIdx.x == 0) {
    int lo = n_tiles;
    for (int w = 0; w < kWarps; ++w) lo = s_progress[w] < lo ? s_progress[w] : lo;
    for (int j = lo; j < s_issued; ++j) mbar_wait(&full[j % STAGES], (j / STAGES) & 1, p.status);
  }
}

// The layer as {bytes of `heads` heads, groups of heads, P, pages x 2} in boxes of one group x 16 tokens x K and V.
int encode_tiles(CUtensorMap* map, const void* layer, int total_pages, int page_size, int hkv, int d, int heads) {
  auto encode = c8::get_encode();
  if (encode == nullptr) return NQT_ERR_CUDA;
  const cuuint64_t row = static_cast<cuuint64_t>(heads) * d;
  cuuint64_t dims[4] = {row, static_cast<cuuint64_t>(hkv / heads), static_cast<cuuint64_t>(page_size),
                        static_cast<cuuint64_t>(total_pages) * 2};
  cuuint64_t strides[3] = {row, static_cast<cuuint64_t>(hkv) * d, static_cast<cuuint64_t>(page_size) * hkv * d};
  cuuint32_t box[4] = {static_cast<cuuint32_t>(row), 1, kBlock, 2};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(layer), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? NQT_OK : NQT_ERR_CUDA;
}

template <int D, int HPC, int STAGES, bool E4M3>
int launch8(const void* layer, Decode8Args a, cudaStream_t s) {
  using Cfg = Cfg8<D, HPC, STAGES>;
  CUtensorMap map;
  if (encode_tiles(&map, layer, a.total_pages, a.page_size, a.hkv, D, Cfg::kBoxHeads) != NQT_OK) {
    set_last_message("decode_attention8: cuTensorMapEncodeTiled failed");
    return NQT_ERR_CUDA;
  }
  static int few_occ = 1;
  static DeviceOnce once;
  auto occupancy = [](int smem) {
    int occ = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, decode8_kernel<D, HPC, STAGES, E4M3>, Cfg::kThreads, smem) !=
            cudaSuccess ||
        occ < 1)
      occ = 1;
    return occ;
  };
  once([&] {
    cudaFuncSetAttribute(decode8_kernel<D, HPC, STAGES, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         Cfg::smem(kMaxRows8));
    few_occ = occupancy(Cfg::smem(kFewRows8));
  });
  const int smem = Cfg::smem(a.batch <= kFewRows8 ? kFewRows8 : a.batch);
  const int occ = a.batch <= kFewRows8 ? few_occ : occupancy(smem);
  const int groups = a.hkv / HPC;
  int n = num_sms() * occ / groups;
  static_assert(HPC <= kMaxHpc, "the tickets' place");
  n = n > kMaxCtas / groups ? kMaxCtas / groups : n;  // hkv <= 256: at least 4
  n = n < 1 ? 1 : n;
  a.n_ctas = n;
  a.by_row = 2 * a.batch <= n && a.batch <= kFewRows8;
  const cudaError_t err = launch_pdl(decode8_kernel<D, HPC, STAGES, E4M3>, dim3(n, groups), dim3(Cfg::kThreads), smem,
                                     s, map, a);
  if (err != cudaSuccess) {
    set_last_error("decode_attention8", err);
    return NQT_ERR_CUDA;
  }
  return NQT_OK;
}

template <int D, bool E4M3>
int dispatch8(const void* layer, const Decode8Args& a, cudaStream_t s) {
  constexpr int kDeep = 128 / D;  // stages of D = 64 hold half the bytes
  if (a.hkv % 4 == 0) return launch8<D, 4, 4 * kDeep, E4M3>(layer, a, s);
  if (a.hkv % 2 == 0) return launch8<D, 2, 8 * kDeep, E4M3>(layer, a, s);
  return launch8<D, 1, 16 * kDeep, E4M3>(layer, a, s);
}

}  // namespace
}  // namespace nqt

using namespace nqt;

extern "C" size_t nqt_decode8_workspace_bytes(int batch_capacity, int num_qo_heads, int head_dim) {
  if (batch_capacity < 1 || num_qo_heads < 1 || head_dim < 1) return 0;
  return ws8_layout(num_qo_heads, head_dim).total;
}

extern "C" int nqt_decode_attention8(const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                                     const void* layer_cache, const float* layer_scales, int total_pages,
                                     int page_size, const int32_t* kv_indptr, const int32_t* kv_indices,
                                     const int32_t* last_page_len, int batch, int batch_capacity, int num_qo_heads,
                                     int num_kv_heads, int head_dim, float sm_scale, int code, void* out,
                                     int64_t out_stride_tok, int64_t out_stride_head, void* workspace,
                                     size_t workspace_bytes, int flags, int32_t* status, void* stream) {
  int rc = c8::check_layer(layer_cache, layer_scales, total_pages, page_size, num_kv_heads, head_dim, code);
  if (rc != NQT_OK) return rc;
  if (!q || !kv_indptr || !kv_indices || !last_page_len || !out || !workspace) return NQT_ERR_ARG;
  if (batch < 0 || batch > batch_capacity || num_qo_heads < 1 || num_qo_heads % num_kv_heads) return NQT_ERR_ARG;
  if (num_qo_heads / num_kv_heads > 8) return NQT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) & 3) || (reinterpret_cast<uintptr_t>(out) & 3)) return NQT_ERR_ARG;
  if ((q_stride_tok & 1) || (q_stride_head & 1) || (out_stride_tok & 1) || (out_stride_head & 1)) return NQT_ERR_ARG;
  if (flags & ~(NQT_DECODE_OVERLAP_KV_WRITE | NQT_DECODE_SHORT_WAIT)) return NQT_ERR_ARG;
  if (batch > kMaxRows8) return NQT_ERR_CAPACITY;
  const Ws8 w = ws8_layout(num_qo_heads, head_dim);
  if (workspace_bytes < w.total) return NQT_ERR_CAPACITY;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return NQT_ERR_ARG;
  if (batch == 0) return NQT_OK;
  uint8_t* base = static_cast<uint8_t*>(workspace);
  Decode8Args a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.o_st = out_stride_tok;
  a.o_sh = out_stride_head;
  a.scales = layer_scales;
  a.indptr = kv_indptr;
  a.indices = kv_indices;
  a.last_len = last_page_len;
  a.tickets = reinterpret_cast<int32_t*>(base);
  a.group_tickets = reinterpret_cast<int32_t*>(base + w.groups);
  a.part_lse = reinterpret_cast<float*>(base + w.lse);
  a.part_o = reinterpret_cast<float*>(base + w.o);
  a.status = status;
  a.batch = batch;
  a.hq = num_qo_heads;
  a.hkv = num_kv_heads;
  a.group = num_qo_heads / num_kv_heads;
  a.page_size = page_size;
  a.total_pages = total_pages;
  a.early = (flags & NQT_DECODE_OVERLAP_KV_WRITE) ? 1 : 0;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.wait_ns = (flags & NQT_DECODE_SHORT_WAIT) ? 0 : kWaitLimitNs;
  cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return code == NQT_E4M3 ? dispatch8<128, true>(layer_cache, a, s) : dispatch8<128, false>(layer_cache, a, s);
  return code == NQT_E4M3 ? dispatch8<64, true>(layer_cache, a, s) : dispatch8<64, false>(layer_cache, a, s);
}
