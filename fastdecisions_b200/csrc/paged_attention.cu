// Causal GQA attention of the newest tokens of packed sequences over a paged KV cache.
//
// Segment s's n = cu[s+1] - cu[s] tokens are the last of its kv_lens[s] cached positions (their own keys
// are already written): token i attends to positions 0 .. kv_lens[s] - n + i.  A token whose mask leaves
// nothing gets zeros.  The query heads of a KV head are packed with the tokens into rows (row = token *
// group + head), so every cached row brought into shared memory feeds them all.
//
// Calls with more than 16 to 32 rows a KV head run the tcgen05 kernel of paged_attention_chunk.cuh.  This file:
// the few-row kernel (mma.sync, split over the keys) and the join of splits.  Its work is bound by
// reading the cache: at one token a sequence each cached byte is used by `group` rows only, far below the
// tensor cores' rate, so warp-level MMAs -- which need no padding to 128 rows and keep S and P in
// registers -- lose nothing to the memory time they hide behind.  What competes with the loads is
// instruction issue, so the products are transposed: S^T = K Q^T and O^T = V^T P^T put 16 keys (columns
// of V) on the MMA's 16-row side and the query rows on its 8-column side.  Four rows then waste half an
// MMA instead of three quarters, and each K / V fragment is converted from e4m3 once for all rows.
//
//   CTA: BM = 8 NR WM rows of one (segment, KV head), keys [kb, ke) in tiles of 64; 4 warps = WM row
//   groups x WK = 4 / WM key groups.  Tiles stream through a ring of cp.async stages.  Each warp keeps
//   its own running maximum (raised only when a score exceeds it by more than 2^8, so most tiles
//   need no reduction across lanes), sum and O (fp32) over its keys; key groups are joined through
//   shared memory at the end.  Up to eight splits are a cluster and join through each other's shared memory,
//   more through a float32 workspace and a second kernel.
//   8-bit cache: e4m3 -> fp16 is exact, one instruction a pair; K's row scale multiplies S, V's enters P
//   before its rounding to fp16.  So P V is in units of the row's largest weight times scale so far, a second
//   running maximum beside the one that the sum is relative to: what a row loses depends on the keys it sees
//   only (one unit for all rows of a warp, from every key of a tile, lost the weights of early tokens behind a
//   later token's large V row; the second exponential a weight costs 64 sequences x 8 tokens, e4m3, 127 us for 122,
//   one token each nothing).  q is brought to fp16 with a power of two a row.
//
// Measured (back to back in a graph): one token behind 1535 positions, 16 / 4 heads of 128, bf16, 7.8 us; 64 x 8192,
// e4m3, 97 us, 5.6 TB/s, bf16 170 us in the parts that the rule below takes, 6.3 TB/s: near the copy rate.  64 ragged
// sequences of 500 to 8192, e4m3, 48.7 us, 4.0 TB/s, and bf16 69.5 us, 5.5 TB/s: what the shorter call loses is its
// start, its uneven end and the join.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "paged.cuh"
#include "sm100.cuh"

namespace fdk {
namespace pattn {
using paged::scale_value;
using sm100::ex2;

__device__ int g_error = 0;

// sigmoid by the fast exponential and quotient: a relative error below 2^-16 for x > -87.3, where the rounding of
// the result to bf16 has 2^-8; below that 0 (the quotient's divisor passes 2^126), where the sigmoid is less than
// 2^-125.  With the exact ones 1532 tokens of 8 heads of 256 behind a shared prefix of 1490 took 58 us, 42 without a
// gate; with these 46.
__device__ __forceinline__ float gate_of(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

struct Params {
  const bf16* q;
  int64_t ld_q;
  const uint8_t* k_cache;  // bytes
  const uint8_t* v_cache;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  int64_t kpage, vpage;  // bytes between pages
  int64_t kscale_page, vscale_page;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* cu;
  const int32_t* kv_lens;
  int64_t tokens, num_pages;
  int nseg, max_pages, page_shift, hq, hkv, group, nsplit, row_blocks;
  int max_seqlen;  // the caller's bound on a segment's tokens
  int split_keys;  // keys a split (a multiple of every tile's), the last one takes what is left
  int block_rows;  // rows of a row block (a CTA's)
  int clustered;   // few rows: the splits of a row block are one cluster
  int picked;      // many rows: x counts the call's units of work, longest first
  int units;       // ... and this many of them, a KV head
  int part_cost;   // ... one part's float32 rows, written and read, in keys of a CTA's work
  float sl2;  // softmax scale * log2(e)
  const bf16* gate;
  int64_t ld_gate;
  int gate_hstride;
  bf16* out;
  float* part_o;   // [nsplit][tokens * hq][D], each divided by its sum: no larger than the largest V row
  int* part_keys;  // many rows, picked: the part size
  float2* part_ml; // [nsplit][tokens * hq]: (running max in the exp2 domain, sum); the sum weighs the row in the join
};

// One segment's metadata, checked.  n: new tokens, past: cached positions before them (may be negative:
// then the first -past tokens see nothing).  Invalid metadata reads as "no keys" and is reported.
struct Seg {
  int begin, n;
  int64_t past;
};
__device__ __forceinline__ Seg segment(const Params& p, int s, bool report) {
  Seg r;
  int end;
  if (!paged::segment_range(p.cu, s, p.tokens, r.begin, end)) {
    if (report) atomicOr(&g_error, 1);
    r.begin = end = 0;
  }
  r.n = end - r.begin;
  int64_t len = p.kv_lens[s];
  if (len < 0 || len > ((int64_t)p.max_pages << p.page_shift)) {
    if (report) atomicOr(&g_error, 1);
    len = 0;
  }
  r.past = len - r.n;
  return r;
}

// Keys [kb, ke) of a split of a row block that sees keys [0, kend).  The split size is fixed, so short
// sequences use few of the grid's splits.
__device__ __forceinline__ void split_range(const Params& p, int part_keys, int split, int kend, int& kb, int& ke) {
  kb = (int)min((int64_t)kend, (int64_t)split * part_keys);
  ke = split == p.nsplit - 1 ? kend : (int)min((int64_t)kend, (int64_t)kb + part_keys);
}
// Whether a row block that sees keys [0, kend) is computed in parts.  One that fits a split is not: its CTA
// writes the result and the join passes over its rows.
__device__ __forceinline__ bool in_parts(const Params& p, int part_keys, int64_t kend) {
  return p.nsplit > 1 && kend > part_keys;
}
// Parts of a row that sees `visible` keys: the splits that hold one of them (at least one is written).
__device__ __forceinline__ int parts_of(const Params& p, int part_keys, int64_t visible) {
  return visible <= part_keys ? 1 : (int)min((int64_t)p.nsplit, (visible + part_keys - 1) / part_keys);
}

// Many rows, at most 32 * PICK segments: the call's row tiles, the segments spread over a warp's lanes.
// Tile rb of a segment sees past + min((rb + 1) tokens, n) keys.
constexpr int PICK = 2;
struct Tiles {
  int past[PICK], n[PICK], tiles[PICK];
  int tokens, least, most;  // tokens a tile, keys of the shortest and of the longest tile
  uint32_t inv;
  // ceil(x / tokens) for x < 2^24 (the host's rule).  floor(y / tokens) as a multiplication is exact for any y where
  // tokens is a power of two, else for y < 2^32 / tokens, and then tokens <= 84; the reciprocal of one token does not
  // fit 32 bits.
  __device__ __forceinline__ int div_up(int x) const {
    return tokens == 1 ? x : (int)__umulhi((uint32_t)(x + tokens - 1), inv);
  }
  __device__ __forceinline__ void load(const Params& p, int tokens_a_tile, int lane) {
    tokens = tokens_a_tile;
    inv = 0xffffffffu / (uint32_t)tokens + 1u;
    int m = 0, l = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PICK; ++i) {
      const int s = lane * PICK + i;
      n[i] = past[i] = tiles[i] = 0;
      if (s < p.nseg) {
        const Seg g = segment(p, s, false);
        // a segment past the call's bound has the bound's tiles: more would take other segments' places in the grid
        n[i] = (int)min((int64_t)g.n, (int64_t)p.row_blocks * tokens);
        past[i] = (int)g.past;
        tiles[i] = div_up(n[i]);
        if (n[i] > 0) {
          m = max(m, past[i] + n[i]);
          l = min(l, max(past[i] + min(n[i], tokens), 0));
        }
      }
    }
    most = (int)__reduce_max_sync(0xffffffffu, (unsigned)m);
    least = min((int)__reduce_min_sync(0xffffffffu, (unsigned)l), most);
  }
};

// Keys a part of such a call, from its lengths: lane j - 1 prices j parts of the longest range.  In units of
// one key of a CTA's work: while every CTA has an SM the longest part is the time, else the whole work
// shared out, with half a part more for its uneven end; a CTA's start is START, the join JOIN and the
// float32 rows of each part written and read.  Measured against a rule on the longest range alone, which has
// to favour even or ragged contexts: 8 segments of 100 to 700 tokens behind 600 to 8000 positions, e4m3, page
// 64, 107 us (170 unsplit); 74 of 32 behind 4608, 2 KV heads of 256, 113 us (152 in two parts).  Every CTA gets
// the same answer (integers only); one leaves it for the join, whose many warps would take 20 us to work it out
// again.
constexpr int SMS = 148;
constexpr int START_KEYS = 448, JOIN_KEYS = 256;
__device__ __forceinline__ int best_part_keys(const Params& p, const Tiles& t, int lane) {
  const int j = lane + 1;
  const int most = max(t.most, 1);
  const int keys = ((most + j - 1) / j + 127) / 128 * 128;
  int64_t work = 0, ctas = 0;  // of one KV head
#pragma unroll
  for (int i = 0; i < PICK; ++i) {
    // the launched units cover `ctas`, which counts every tile of a segment as its last one
    for (int src = 0; src * PICK + i < p.nseg; ++src) {
      const int past = __shfl_sync(0xffffffffu, t.past[i], src), n = __shfl_sync(0xffffffffu, t.n[i], src);
      const int tiles = __shfl_sync(0xffffffffu, t.tiles[i], src);
      ctas += (int64_t)tiles * max(((unsigned)(past + n) + keys - 1u) / keys, 1u);
      work += (int64_t)tiles * max(past + n / 2, 0);
    }
  }
  int64_t cost = keys;
  if (ctas * p.hkv > SMS) cost = max(cost, (work + START_KEYS * ctas) * p.hkv / SMS + keys / 2);
  if (j > 1) cost += JOIN_KEYS + j * (int64_t)p.part_cost;
  if (j > 1 && (j > p.nsplit || ctas > p.units)) cost = 0x7fffffff;
  const unsigned mine = (unsigned)min(cost, (int64_t)0x7fffffff);
  const unsigned best = __reduce_min_sync(0xffffffffu, mine);
  return __shfl_sync(0xffffffffu, keys, __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1);
}

// 1 / a softmax sum; 0 for a row that saw no key, NaN for one that met a NaN.  FAST: to two units in the last place
// (few rows: the exact quotient costs one token behind 1535 positions 0.1 us; in the join it costs nothing, and
// without it the compiler no longer keeps four parts' loads in flight: 64 segments of 500 to 8192, e4m3, 49.5 us, 50.7)
template <bool FAST = false>
__device__ __forceinline__ float reciprocal_sum(float l) {
  return l > 0.f ? (FAST ? __fdividef(1.f, l) : 1.f / l) : (l == 0.f ? 0.f : l);
}
// What a part's row, of maximum m and sum l, counts beside a common maximum.  A sum of 0 is a part without a visible
// key; a row of NaN scores has a NaN for its sum and no maximum.
__device__ __forceinline__ float part_weight(float m, float l, float common) { return l == 0.f ? 0.f : l * ex2(m - common); }

// Page ids of the 16-key groups from `key0` on (page sizes are multiples of 16).  The index is clamped to
// the range's last key, so the loads need no branch and are all in flight at once; they are issued a
// tile ahead of their use.  An id outside the cache gives -1 (rows of zeros) and is reported.
template <int N>
__device__ __forceinline__ void load_page_ids(const Params& p, const int32_t* table, int key0, int last, int (&id)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) id[i] = __ldg(table + (min(key0 + 16 * i, last) >> p.page_shift));
}
template <int N>
__device__ __forceinline__ void check_page_ids(const Params& p, int (&id)[N]) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if ((uint32_t)id[i] >= (uint32_t)p.num_pages) {
      id[i] = -1;
      bad = true;
    }
  if (bad) atomicOr(&g_error, 1);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr int BN = 64;        // keys a tile
constexpr int THREADS = 128;

template <int D, bool QUANT>
struct Geo {
  static constexpr int ROW = QUANT ? D : 2 * D;   // bytes of a cached row
  static constexpr int CH = ROW / 16;             // 16-byte chunks of it
  static constexpr int TILE = BN * ROW;
  static constexpr int STAGE = 2 * TILE + (QUANT ? 2 * BN : 0);
  static constexpr int STAGES = 3;                // 50 KB (e4m3, head_dim 128) to 192 KB (bf16, 256) a CTA
  static constexpr int RING = STAGES * STAGE;
};

// 16-byte chunk c of row r of a tile: the chunk index is XORed with the row so that the eight rows of an
// 8x8 matrix fall into different banks
template <int CH>
__device__ __forceinline__ uint32_t tile_at(int r, int c) { return (uint32_t)((r * CH + (c ^ (r & 7))) * 16); }

// 2^(b - 127), with 0 for b <= 0
__device__ __forceinline__ float pow2_byte(int b) { return __int_as_float(max(b, 0) << 23); }

// transpose of an 8x8 matrix of 16-bit elements held two a lane
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}

// Cluster: barrier, and loads from the shared memory of CTA `rank` at this CTA's address `a`.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t a, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t a, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(map_rank(a, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t a, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(map_rank(a, rank)) : "memory");
  return v;
}

constexpr float GROW = 8.f;     // the running maximum lags by at most 2^GROW
// fp16 P: times 2^V_SHIFT, at most 2^(GROW + V_SHIFT); contributions down to 2^-30 of the row's largest stay
constexpr float V_SHIFT = 6.f;

template <int D, bool QUANT, int WM, int NR>
__global__ void __launch_bounds__(THREADS) few_rows_kernel(const Params p) {
  using G = Geo<D, QUANT>;
  constexpr int WK = 4 / WM;        // key groups
  constexpr int KPW = BN / WK;      // keys a warp and tile
  constexpr int BM = 8 * NR * WM;
  constexpr int KK = D / 16;        // 16-column steps of D
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp % WM, wk = warp / WM;
  const int g = lane >> 2, t4 = lane & 3;

  // grid: x = (segment, kv head, row block) with the kv head fastest, y = split
  const int hk = (int)(blockIdx.x % (unsigned)p.hkv);
  const int srb = (int)(blockIdx.x / (unsigned)p.hkv);
  const int s = srb / p.row_blocks, rb = srb % p.row_blocks;
  const int split = blockIdx.y;
  const bool first = tid == 0 && hk == 0 && rb == 0 && split == 0;
  const Seg seg = segment(p, s, first);
  const int rows = seg.n * p.group;
  const int row0 = rb * BM;
  if (first && seg.n > p.max_seqlen) atomicOr(&g_error, 1);
  if (row0 >= rows) return;
  const int last_tok = (min(row0 + BM, rows) - 1) / p.group;
  const int64_t kend64 = seg.past + last_tok + 1;
  const int kend = kend64 > 0 ? (int)kend64 : 0;       // keys the row block can see
  int kb, ke;
  split_range(p, p.split_keys, split, kend, kb, ke);
  if (kb >= ke && split > 0) return;  // no join reads this part
  const int ntiles = (ke - kb + BN - 1) / BN;

  // tile loads: chunk lc of rows lr + i * RPP; the rows of a pass lie in one group of 16 keys
  constexpr int RPP = THREADS / G::CH, GROUPS = BN / 16;
  const int lc = tid % G::CH, lr = tid / G::CH;
  const int32_t* table = p.table + (int64_t)s * p.ld_table;
  const int page_mask = (1 << p.page_shift) - 1;
  const int64_t head_at = (int64_t)(hk << p.page_shift) * G::ROW + lr * G::ROW + lc * 16;
  int ids[GROUPS];  // of the next tile to load
  if (ntiles > 0) load_page_ids(p, table, kb, ke - 1, ids);
  auto load_tile = [&](int j) {
    const int key0 = kb + j * BN;
    const uint32_t dst = sbase + (uint32_t)(j % G::STAGES) * G::STAGE;
    check_page_ids(p, ids);
    bool whole = key0 + BN <= ke;
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) whole = whole && ids[u] >= 0;
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
      const int64_t pg = ids[u] >= 0 ? ids[u] : 0;
      const int64_t at = head_at + ((key0 + 16 * u) & page_mask) * G::ROW;
      const uint8_t* ks = p.k_cache + (pg * p.kpage + at);
      const uint8_t* vs = p.v_cache + (pg * p.vpage + at);
#pragma unroll
      for (int i = 0; i < 16 / RPP; ++i) {
        const int r = 16 * u + i * RPP;
        const uint32_t to = dst + tile_at<G::CH>(lr + r, lc);
        if (whole) {
          cp_async16(to, ks + i * RPP * G::ROW);
          cp_async16(to + G::TILE, vs + i * RPP * G::ROW);
        } else {  // rows past the range or on a bad page are zero-filled
          const uint32_t bytes = ids[u] >= 0 && key0 + lr + r < ke ? 16u : 0u;
          cp_async16(to, ks + i * RPP * G::ROW, bytes);
          cp_async16(to + G::TILE, vs + i * RPP * G::ROW, bytes);
        }
      }
    }
    if (QUANT && tid < 8) {  // scale bytes: 16 keys at a time
      const int u = tid & 3, r = u * 16;
      const int id = u == 0 ? ids[0] : u == 1 ? ids[1] : u == 2 ? ids[2] : ids[3];
      const bool ok = id >= 0 && key0 + r < ke;
      const int64_t pg = ok ? id : 0;
      const int at = (hk << p.page_shift) + ((key0 + r) & page_mask);
      cp_async16(dst + 2 * G::TILE + (tid < 4 ? 0 : BN) + r,
                 tid < 4 ? p.k_scale + (pg * p.kscale_page + at) : p.v_scale + (pg * p.vscale_page + at), ok ? 16u : 0u);
    }
    load_page_ids(p, table, key0 + BN, ke - 1, ids);
  };
#pragma unroll
  for (int j = 0; j < G::STAGES - 1; ++j) {
    if (j < ntiles) load_tile(j);
    cp_commit();
  }

  // B fragments of q: row 8 nr + g of this warp's rows.  bf16: columns 2t, 2t+1 (+8) of each 16; 8-bit
  // cache: columns 4t .. 4t+3, in the order the byte-wise K fragments come in, as fp16 times a power of
  // two a row.
  uint32_t qf[NR][KK][2];
  float qs[NR][2];   // of this lane's columns of S^T: rows 2t, 2t+1
  int lim[NR][2];    // their last visible key
  int wlim = 0x7fffffff;  // the smallest of the warp's live rows
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) {
    const int base_row = row0 + (wm * NR + nr) * 8;
    const int r = base_row + g;
    const bool live = r < rows;
    const int tok = live ? r / p.group : 0;
    const bf16* src = p.q + (int64_t)(seg.begin + tok) * p.ld_q + (int64_t)(hk * p.group + (live ? r - tok * p.group : 0)) * D;
    float unit = 1.f;
    if (!QUANT) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        qf[nr][kk][0] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 2 * t4) : 0u;
        qf[nr][kk][1] = live ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8 + 2 * t4) : 0u;
      }
    } else {
      float a = 0.f;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const uint2 raw = live ? *reinterpret_cast<const uint2*>(src + kk * 16 + 4 * t4) : make_uint2(0u, 0u);
        qf[nr][kk][0] = raw.x;
        qf[nr][kk][1] = raw.y;
        const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
        const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
        a = fmaxf(fmaxf(a, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
      }
      a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
      a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
      // the row's largest magnitude goes to [1, 2): fp16 keeps bf16's 8 bits down to 2^-14 of it
      const int e = min(max((int)(__float_as_uint(a) >> 23), 1), 253);
      const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
      unit = __uint_as_float((uint32_t)e << 23);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[nr][kk][u]));
          qf[nr][kk][u] = pack_f16x2(x.x * inv, x.y * inv);
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      qs[nr][u] = p.sl2 * (QUANT ? __shfl_sync(0xffffffffu, unit, (2 * t4 + u) * 4) : 1.f);
      const int rr = base_row + 2 * t4 + u;
      lim[nr][u] = rr < rows ? (int)(seg.past + rr / p.group) : -1;
      wlim = min(wlim, rr < rows ? lim[nr][u] : 0x7fffffff);
    }
  }
  wlim = min(__reduce_min_sync(0xffffffffu, wlim), ke - 1);  // every key up to here needs no mask

  float o[KK][NR][4];  // O^T: columns (of D) down, rows across
#pragma unroll
  for (int i = 0; i < KK; ++i)
#pragma unroll
    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][nr][c] = 0.f;
  float m[NR][2], l[NR][2];
#pragma unroll
  for (int nr = 0; nr < NR; ++nr)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      m[nr][u] = -FLT_MAX;  // finite: a hidden key's score of -inf is -inf beside it
      l[nr][u] = 0.f;
    }
  // 8-bit cache: O of a row is in units of 2^(un - m - 127), un the running maximum of score + scale byte - V_SHIFT
  float un[NR][2];
#pragma unroll
  for (int nr = 0; nr < NR; ++nr) un[nr][0] = un[nr][1] = -FLT_MAX;

  for (int j = 0; j < ntiles; ++j) {
    cp_wait<G::STAGES - 2>();
    __syncthreads();  // tile j is in, and every warp is done with the stage that tile j + STAGES - 1 takes
    if (j + G::STAGES - 1 < ntiles) load_tile(j + G::STAGES - 1);
    cp_commit();
    const uint32_t kt = sbase + (uint32_t)(j % G::STAGES) * G::STAGE, vt = kt + G::TILE;
    const uint8_t* scales = smem + (kt - sbase) + 2 * G::TILE;
#pragma unroll
    for (int kg = 0; kg < KPW / 16; ++kg) {
      const int krow = wk * KPW + kg * 16;  // first of 16 keys in the tile
      const int key0 = kb + j * BN + krow;
      // S^T = K Q^T: element c of row tile nr is key g + 8 (c / 2), row 2 t + (c & 1)
      float sc[NR][4];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[nr][c] = 0.f;
      const int kr = krow + (lane & 15), vr = krow + (lane & 7) + ((lane >> 4) << 3);
      if (!QUANT) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          uint32_t a[4];
          ldsm4(a, kt + tile_at<G::CH>(kr, 2 * kk + (lane >> 4)));
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) mma<false>(sc[nr], a, qf[nr][kk][0], qf[nr][kk][1]);
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < KK; kk += 2) {
          uint32_t b[4];
          ldsm4(b, kt + tile_at<G::CH>(kr, kk + (lane >> 4)));
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t a[4] = {paged::e4m3x2_to_f16x2((uint16_t)b[2 * u]), paged::e4m3x2_to_f16x2((uint16_t)b[2 * u + 1]),
                                   paged::e4m3x2_to_f16x2((uint16_t)(b[2 * u] >> 16)),
                                   paged::e4m3x2_to_f16x2((uint16_t)(b[2 * u + 1] >> 16))};
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mma<true>(sc[nr], a, qf[nr][kk + u][0], qf[nr][kk + u][1]);
          }
        }
      }
      float vb[2] = {0.f, 0.f};  // V's scale bytes; any byte where the key is hidden: its score is -inf
      if (QUANT) {
        const float k0 = pow2_byte(scales[krow + g]), k1 = pow2_byte(scales[krow + g + 8]);
        vb[0] = scales[BN + krow + g];
        vb[1] = scales[BN + krow + g + 8];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
          sc[nr][0] *= k0 * qs[nr][0];
          sc[nr][1] *= k0 * qs[nr][1];
          sc[nr][2] *= k1 * qs[nr][0];
          sc[nr][3] *= k1 * qs[nr][1];
        }
      } else {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int c = 0; c < 4; ++c) sc[nr][c] *= p.sl2;
      }
      if (key0 + 15 > wlim) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (key0 + g + 8 * (c >> 1) > min(lim[nr][c & 1], ke - 1)) sc[nr][c] = -INFINITY;
      }
      // the keys' exponents beside the running maxima: d of their weights, e of what they add to O (with the scale: one
      // more float32 rounding of the score)
      float d[NR][4], e[NR][4];
      bool up = false;
      auto exponents = [&] {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            d[nr][c] = sc[nr][c] - m[nr][c & 1];
            if (QUANT) e[nr][c] = (sc[nr][c] + vb[c >> 1]) - un[nr][c & 1];
          }
          up |= fmaxf(fmaxf(d[nr][0], d[nr][1]), fmaxf(d[nr][2], d[nr][3])) > GROW;
          if (QUANT) up |= fmaxf(fmaxf(e[nr][0], e[nr][1]), fmaxf(e[nr][2], e[nr][3])) > GROW + V_SHIFT;
        }
      };
      exponents();
      // raise the maxima (and the units of O) only where needed
      if (__any_sync(0xffffffffu, up)) {
#pragma unroll
        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float mx = fmaxf(sc[nr][u], sc[nr][2 + u]), cx = fmaxf(sc[nr][u] + vb[0], sc[nr][2 + u] + vb[1]) - V_SHIFT;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
              if (QUANT) cx = fmaxf(cx, __shfl_xor_sync(0xffffffffu, cx, off));
            }
            float corr = 1.f;
            if (mx > m[nr][u]) {
              corr = ex2(m[nr][u] - mx);  // 0 when nothing was visible before
              m[nr][u] = mx;
            }
            l[nr][u] *= corr;
            if (QUANT) {
              corr = 1.f;
              if (cx > un[nr][u]) {
                corr = ex2(un[nr][u] - cx);
                un[nr][u] = cx;
              }
            }
#pragma unroll
            for (int i = 0; i < KK; ++i) {
              o[i][nr][u] *= corr;
              o[i][nr][2 + u] *= corr;
            }
          }
        exponents();
      }
      // P^T, this lane's part of the row sums (of the unrounded weights), and O^T += V^T P^T
      uint32_t pb[NR][2];
#pragma unroll
      for (int nr = 0; nr < NR; ++nr) {
        const float p0 = ex2(d[nr][0]), p1 = ex2(d[nr][1]), p2 = ex2(d[nr][2]), p3 = ex2(d[nr][3]);
        l[nr][0] += p0 + p2;
        l[nr][1] += p1 + p3;
        pb[nr][0] = transpose8(QUANT ? pack_f16x2(ex2(e[nr][0]), ex2(e[nr][1])) : pack_bf16x2(p0, p1));
        pb[nr][1] = transpose8(QUANT ? pack_f16x2(ex2(e[nr][2]), ex2(e[nr][3])) : pack_bf16x2(p2, p3));
      }
      if (!QUANT) {
#pragma unroll
        for (int i = 0; i < KK; ++i) {
          uint32_t a[4];
          ldsm4t(a, vt + tile_at<G::CH>(vr, 2 * i + ((lane >> 3) & 1)));
#pragma unroll
          for (int nr = 0; nr < NR; ++nr) mma<false>(o[i][nr], a, pb[nr][0], pb[nr][1]);
        }
      } else {
        // b16 pairs are two neighbouring columns of a key: after the transpose a register holds columns
        // (2g, 2g+1) x keys (2t, 2t+1); its bytes reordered give rows g (even columns) and g + 8 (odd)
#pragma unroll
        for (int i = 0; i < KK; i += 2) {
          uint32_t b[4];
          ldsm4t(b, vt + tile_at<G::CH>(vr, i + ((lane >> 3) & 1)));
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t x = __byte_perm(b[u], 0, 0x3120), y = __byte_perm(b[2 + u], 0, 0x3120);
            const uint32_t a[4] = {paged::e4m3x2_to_f16x2((uint16_t)x), paged::e4m3x2_to_f16x2((uint16_t)(x >> 16)),
                                   paged::e4m3x2_to_f16x2((uint16_t)y), paged::e4m3x2_to_f16x2((uint16_t)(y >> 16))};
#pragma unroll
            for (int nr = 0; nr < NR; ++nr) mma<true>(o[i + u][nr], a, pb[nr][0], pb[nr][1]);
          }
        }
      }
    }
  }
  cp_wait<0>();
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  __syncthreads();  // the ring is free: it holds the join now

  // join of the key groups: [wk][row][D + 4] floats (the padding spreads the four row pairs of a store
  // over the banks) and [wk][row] (m, l)
  constexpr int LDO = D + 4;
  float* so = reinterpret_cast<float*>(smem);
  float2* sml = reinterpret_cast<float2*>(smem + WK * BM * LDO * 4);
#pragma unroll
  for (int nr = 0; nr < NR; ++nr)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[nr][u] += __shfl_xor_sync(0xffffffffu, l[nr][u], off);
      if (g == 0) sml[wk * BM + (wm * NR + nr) * 8 + 2 * t4 + u] = make_float2(m[nr][u], l[nr][u]);
    }
  __syncthreads();
#pragma unroll
  for (int nr = 0; nr < NR; ++nr)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = (wm * NR + nr) * 8 + 2 * t4 + u;
      // 8-bit cache: the unit's root twice, as the unit itself may leave float32's range where the result does not
      const float root = !QUANT ? 1.f : l[nr][u] == 0.f ? 0.f : ex2(0.5f * (un[nr][u] - m[nr][u] - 127.f));
      const float f = reciprocal_sum<true>(l[nr][u]) * root;
      float* dst = so + (wk * BM + row) * LDO;
#pragma unroll
      for (int i = 0; i < KK; ++i) {
        dst[i * 16 + (QUANT ? 2 * g : g)] = o[i][nr][u] * f * root;
        dst[i * 16 + (QUANT ? 2 * g + 1 : g + 8)] = o[i][nr][2 + u] * f * root;
      }
    }
  __syncthreads();
  // 8 columns a thread: sum of the key groups, then the result or this split's part
  const bool part = in_parts(p, p.split_keys, kend);
  auto finish = [&](float (&y)[8], int gr, int c) {
    const int64_t tok = seg.begin + gr / p.group;
    const int head = hk * p.group + gr % p.group;
    if (p.gate) {
      float gv[8];
      unpack8(*reinterpret_cast<const uint4*>(p.gate + tok * p.ld_gate + (int64_t)head * p.gate_hstride + c), gv);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= gate_of(gv[i]);
    }
    *reinterpret_cast<uint4*>(p.out + (tok * p.hq + head) * D + c) = pack8(y);
  };
  for (int e = tid; e < BM * (D / 8); e += THREADS) {
    const int row = e / (D / 8), c = (e % (D / 8)) * 8;
    const int gr = row0 + row;
    if (gr >= rows) break;
    float mm = -INFINITY, ll = 0.f, f[WK];
#pragma unroll
    for (int w = 0; w < WK; ++w) mm = fmaxf(mm, sml[w * BM + row].x);
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float2 x = sml[w * BM + row];
      ll += f[w] = part_weight(x.x, x.y, mm);
    }
    const float inv = reciprocal_sum<true>(ll);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      f[w] *= inv;
      const float4 a = *reinterpret_cast<const float4*>(so + (w * BM + row) * LDO + c);
      const float4 b = *reinterpret_cast<const float4*>(so + (w * BM + row) * LDO + c + 4);
      y[0] = fmaf(f[w], a.x, y[0]); y[1] = fmaf(f[w], a.y, y[1]); y[2] = fmaf(f[w], a.z, y[2]); y[3] = fmaf(f[w], a.w, y[3]);
      y[4] = fmaf(f[w], b.x, y[4]); y[5] = fmaf(f[w], b.y, y[5]); y[6] = fmaf(f[w], b.z, y[6]); y[7] = fmaf(f[w], b.w, y[7]);
    }
    if (!part) {
      finish(y, gr, c);
    } else if (p.clustered) {  // in the place of the first key group, read by the cluster
      float* dst = so + row * LDO + c;
      *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(y[4], y[5], y[6], y[7]);
      if (c == 0) sml[WK * BM + row] = make_float2(mm, ll);
    } else {
      const int64_t idx = (int64_t)(seg.begin + gr / p.group) * p.hq + hk * p.group + gr % p.group;
      float* dst = p.part_o + ((int64_t)split * p.tokens * p.hq + idx) * D + c;
      *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(y[4], y[5], y[6], y[7]);
      if (c == 0) p.part_ml[(int64_t)split * p.tokens * p.hq + idx] = make_float2(mm, ll);
    }
  }
  if (!part || !p.clustered) return;
  // join in the cluster: CTA `split` of the `parts` that have keys takes every parts-th piece.  The ones
  // without keys have left already, which the cluster barrier counts as arrived.
  __syncthreads();
  cluster_sync();
  const int parts = parts_of(p, p.split_keys, kend);
  for (int e = tid * parts + split; e < BM * (D / 8); e += THREADS * parts) {
    const int row = e / (D / 8), c = (e % (D / 8)) * 8;
    const int gr = row0 + row;
    if (gr >= rows) break;
    const uint32_t ml_at = smem_u32(sml + WK * BM + row), o_at = smem_u32(so + row * LDO + c);
    float2 ml[8];
    float mm = -INFINITY, ll = 0.f, y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ml[i] = i < parts ? cluster_load2(ml_at, i) : make_float2(-INFINITY, 0.f);
      mm = fmaxf(mm, ml[i].x);
      y[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ll += ml[i].y = part_weight(ml[i].x, ml[i].y, mm);
    const float inv = reciprocal_sum<true>(ll);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < parts) {
        const float f = ml[i].y * inv;
        const float4 a = cluster_load4(o_at, i), b = cluster_load4(o_at + 16, i);
        y[0] = fmaf(f, a.x, y[0]); y[1] = fmaf(f, a.y, y[1]); y[2] = fmaf(f, a.z, y[2]); y[3] = fmaf(f, a.w, y[3]);
        y[4] = fmaf(f, b.x, y[4]); y[5] = fmaf(f, b.y, y[5]); y[6] = fmaf(f, b.z, y[6]); y[7] = fmaf(f, b.w, y[7]);
      }
    }
    finish(y, gr, c);
  }
  __syncthreads();
  cluster_sync();  // no CTA leaves while another reads its shared memory
}

// Join of the splits: one warp a (token, head) row, 8 columns a lane (two rows a warp at D = 128), four parts
// at a time so that their loads are in flight together.  It is launched while the kernel before it drains;
// what that kernel does not write is read before the wait for the parts.
template <int D>
__global__ void __launch_bounds__(128) join_kernel(const Params p) {
  auto wait = [] { asm volatile("griddepcontrol.wait;\n" ::: "memory"); };  // every thread, also one that leaves
  constexpr int LPR = D / 8, RPW = 32 / LPR;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t per_tok = (p.hq + RPW - 1) / RPW;   // warps a token
  const int64_t tok = w / per_tok;
  if (tok >= p.tokens) return wait();
  const int s = paged::find_segment_warp(p.cu, p.nseg, (int)tok, lane);
  if (s < 0 || s >= p.nseg) return wait();          // behind the last segment
  const int end = p.cu[s + 1];
  if (end <= tok || end > p.tokens || p.cu[s] < 0) return wait();
  const int head = (int)(w % per_tok) * RPW + lane / LPR, c = (lane % LPR) * 8;
  if (head >= p.hq) return wait();
  const int64_t idx = tok * p.hq + head, plane = p.tokens * p.hq;
  int64_t len = p.kv_lens[s];
  if (len < 0 || len > ((int64_t)p.max_pages << p.page_shift)) len = 0;
  // the last token of the row's block decides whether there are parts
  const int n = end - p.cu[s], row = (int)(tok - p.cu[s]) * p.group + head % p.group;
  if (row / p.block_rows >= p.row_blocks) return wait();  // past the call's bound: not computed
  const int last = min((row / p.block_rows + 1) * p.block_rows, n * p.group) - 1;
  uint4 gate = {};
  if (p.gate) gate = *reinterpret_cast<const uint4*>(p.gate + tok * p.ld_gate + (int64_t)head * p.gate_hstride + c);
  wait();
  const int part_keys = p.picked ? *p.part_keys : p.split_keys;
  if (!in_parts(p, part_keys, len - n + last / p.group + 1)) return;
  const int parts = parts_of(p, part_keys, len - (end - tok) + 1);
  float mm = -INFINITY, ll = 0.f, y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 4) {
    float2 ml[4];
    float4 o[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      o[i][0] = o[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i0 + i < parts) {
        const float* src = p.part_o + ((i0 + i) * plane + idx) * D + c;
        ml[i] = p.part_ml[(i0 + i) * plane + idx];
        o[i][0] = *reinterpret_cast<const float4*>(src);
        o[i][1] = *reinterpret_cast<const float4*>(src + 4);
      }
    }
    float m = mm;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, ml[i].x);
    // y is the mean over the parts so far, of weight ll beside the maximum mm
    const float keep = part_weight(mm, ll, m);
    ll = keep;
#pragma unroll
    for (int i = 0; i < 4; ++i) ll += ml[i].y = part_weight(ml[i].x, ml[i].y, m);
    mm = m;
    const float inv = reciprocal_sum(ll);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] *= keep * inv;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = ml[i].y * inv;
      const float4 a = o[i][0], b = o[i][1];
      y[0] = fmaf(f, a.x, y[0]); y[1] = fmaf(f, a.y, y[1]); y[2] = fmaf(f, a.z, y[2]); y[3] = fmaf(f, a.w, y[3]);
      y[4] = fmaf(f, b.x, y[4]); y[5] = fmaf(f, b.y, y[5]); y[6] = fmaf(f, b.z, y[6]); y[7] = fmaf(f, b.w, y[7]);
    }
  }
  if (p.gate) {
    float gv[8];
    unpack8(gate, gv);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= gate_of(gv[i]);
  }
  *reinterpret_cast<uint4*>(p.out + idx * D + c) = pack8(y);
}

template <int D, bool QUANT, int WM, int NR>
static int launch_few(const Params& p, cudaStream_t s) {
  using G = Geo<D, QUANT>;
  constexpr int BM = 8 * NR * WM, WK = 4 / WM;
  constexpr int join = WK * BM * (D + 4) * 4 + (WK + 1) * BM * 8;
  constexpr int bytes = G::RING > join ? G::RING : join;
  const void* fn = (const void*)few_rows_kernel<D, QUANT, WM, NR>;
  if (int st = ensure_smem_attr(fn, bytes, "paged_gqa")) return st;
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = 1;
  cluster.val.clusterDim.y = (unsigned)p.nsplit;
  cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)p.nseg * p.row_blocks * p.hkv), (unsigned)p.nsplit);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = &cluster;
  cfg.numAttrs = p.clustered ? 1 : 0;
  cudaLaunchKernelEx(&cfg, few_rows_kernel<D, QUANT, WM, NR>, p);
  return check_launch("paged_gqa");
}

// `rows` (8, 16 or 32) a CTA.  O of 32 rows at head_dim 128, 16 at 256, takes 128 registers a lane; the
// other 16 go to other warps.
template <int D, bool QUANT>
static int launch_rows(const Params& p, int rows, cudaStream_t s) {
  constexpr int most = D == 128 ? 4 : 2;
  switch (rows) {
    case 8: return launch_few<D, QUANT, 1, 1>(p, s);
    case 16: return launch_few<D, QUANT, 1, 2>(p, s);
    default: return launch_few<D, QUANT, 4 / most, most>(p, s);
  }
}

// Positions of a sequence.  The kernels step through them in 32 bits and look ahead: the scan of the scale bytes by up
// to 21504 keys, the others by less than 512.
constexpr int64_t MOST_POSITIONS = 0x7fff0000;

// Tiling of a call: the kernel, its rows a CTA and the split of the keys.  All follow from host-side
// sizes only, so a captured call replays with any lengths.
struct Plan {
  bool many;           // the tcgen05 kernel
  int rows;            // few-row kernel: rows a CTA
  int64_t row_blocks;  // row blocks (tiles) of the longest segment, a KV head
  int64_t tiles;       // many rows: row tiles that can exist, a KV head
  int64_t units;       // ... and CTAs in the grid's first dimension
  int64_t part_cost;   // ... a part's float32 rows in keys of a CTA's work
  bool picked, clustered;
  int nsplit, split_keys;
};
constexpr int MAX_SPLIT = 64, MAX_CLUSTER = 8;
// The few-row kernel's time grows with the rows, the tcgen05 kernel's does not below a tile.  Measured, 64
// segments x 8192 positions, 16 / 4 heads of 128 and 8 / 2 of 256, few against many rows in us, bf16: 16
// rows 173 / 302 and 204 / 214, 32 rows 253 / 296 and 284 / 209, 64 rows 365 / 299 and 520 / 208; e4m3:
// 32 rows 229 / 363 and 202 / 279, 64 rows 364 / 363 and 323 / 286.
constexpr int few_rows_most(int64_t d, bool quant) { return d == 256 && !quant ? 16 : 32; }
// Few rows, CTAs an SM to aim at.  A part costs its rows in float32 and a CTA's start, so below one CTA an SM
// the parts fill the SMs once, with what a ring's shared memory leaves room for: one CTA of head_dim 256 in bf16,
// two of 128, three of an 8-bit cache (8 segments x 8192 positions, 4 KV heads, bf16: 26 us with 8 parts, 34 with
// 13).  Above, ragged contexts want many parts (64 segments of 500 to 8192, e4m3: 99 us unsplit, 59 in 4, 45 in 6),
// even ones lose a little by them (64 x 8192, bf16: 153 us unsplit, 169 in 6), and more rows a part cost more.
// Short parts pay while SMs are idle (20 segments of 190 to 725, 6 heads on one: 10.5 us in parts of 256 keys,
// 8.7 of 128; 64 segments of 500 on 4 heads: 11.4 us unsplit, 15.7 in parts of 256).
constexpr int few_ctas(int64_t ctas, int rows, int64_t d, bool quant) {
  return ctas < SMS ? (quant ? 3 : d == 128 ? 2 : 1) : rows <= 16 ? 12 : 4;
}
// Splits as clusters while all of them run at once, up to eight, and eight where more would be short: one token
// behind 1535 positions 12.4 -> 10.3 us, 8 x 2048 12.6 -> 9.6 us (bf16, head_dim 128).  With more CTAs the short
// parts would wait for the long ones: 64 segments of 500 to 8192, e4m3, 54 us with the second kernel, 70 in
// clusters.  At head_dim 256 in bf16 a CTA fills an SM, and more than eight clusters no longer find their eight
// SMs in one GPC: 13 us against 20 at 8 x 2048.
static Plan make_plan(int64_t num_segments, int64_t max_seqlen, int64_t max_kv, int64_t tokens, int64_t hkv,
                      int64_t group, int64_t d, bool quant) {
  Plan r = {};
  if (max_seqlen > tokens) max_seqlen = tokens;
  if (max_seqlen < 1) max_seqlen = 1;  // a bound of no tokens is still checked against the segments
  const int64_t rows = max_seqlen * group;
  int64_t split, least;
  r.many = rows > few_rows_most(d, quant) && group <= 128;
  if (r.many) {
    const int64_t per = (d == 128 ? 2 : 1) * (128 / group);  // tokens a CTA
    r.row_blocks = (max_seqlen + per - 1) / per;
    // CTAs that have work: from the tokens, half a tile more a segment and one at least, not from the longest one
    int64_t ctas = hkv * std::max((2 * tokens + per * (num_segments + 2) - 1) / (2 * per), std::min(num_segments, tokens));
    const int64_t most = num_segments * hkv * r.row_blocks;
    const bool even = 10 * ctas > 7 * most;  // even lengths, `most` is exact; else `ctas` is rather too many
    if (even) ctas = most;
    ctas = std::max<int64_t>(ctas, 1);
    // More than half of the SMs busy: few segments are cut and sorted on the device, which knows their lengths.
    r.picked = 2 * ctas > SMS && num_segments <= 64 && tokens < 1 << 24;
    // upper bound of the parts where the device picks (see best_part_keys), else the parts
    split = r.picked ? (2 * SMS + ctas / 2) / ctas : (SMS + (even ? 0 : ctas / 16)) / ctas;
    if (split > 32) split = 32;
    r.part_cost = tokens * group * hkv * d / 8192;  // 8 bytes a value; a key's work lasts as long as 64 KB of them
    if (r.part_cost > 1 << 24) r.part_cost = 1 << 24;
    // no more than can pay
    while (split > 1 && max_kv * (split - 1) <= split * (JOIN_KEYS + split * r.part_cost)) --split;
    if (split == 1 && most <= SMS) r.picked = false;  // one wave in any order
    r.tiles = num_segments * r.row_blocks;
    if (r.picked && tokens / per + num_segments < r.tiles) r.tiles = tokens / per + num_segments;
    least = 128;
  } else {
    r.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
    r.row_blocks = (rows + r.rows - 1) / r.rows;
    const int64_t ctas = num_segments * hkv * (r.row_blocks > 0 ? r.row_blocks : 1);
    split = few_ctas(ctas, r.rows, d, quant) * SMS / ctas;
    least = ctas >= SMS ? 512 : max_kv > 4096 ? 256 : 128;
  }
  if (split > MAX_SPLIT) split = MAX_SPLIT;
  if (split < 1) split = 1;
  auto cut = [&](int64_t parts) {
    int64_t keys = (max_kv + parts - 1) / parts;
    if (keys < least) keys = least;
    keys = (keys + 127) / 128 * 128;
    r.split_keys = (int)keys;
    r.nsplit = max_kv > keys ? (int)((max_kv + keys - 1) / keys) : 1;
  };
  cut(split);
  r.units = r.tiles;
  if (r.picked && r.nsplit > 1) {
    r.units += 2 * SMS / hkv;
    if (r.units > r.tiles * r.nsplit) r.units = r.tiles * r.nsplit;
  }
  // a cluster's join costs no launch and no workspace: a little over eight splits become eight
  const int64_t in_cluster = r.nsplit < MAX_CLUSTER ? r.nsplit : MAX_CLUSTER;
  r.clustered = !r.many && r.nsplit > 1 && (r.nsplit <= MAX_CLUSTER || max_kv <= 256 * MAX_CLUSTER) &&
                num_segments * hkv * r.row_blocks * in_cluster <= (d == 256 && !quant ? 64 : 2 * SMS);
  if (r.clustered) cut(in_cluster);
  return r;
}

}  // namespace pattn
}  // namespace fdk

#include "paged_attention_chunk.cuh"

namespace fdk {

int paged_attn_take_device_error() {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, pattn::g_error, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (h) {
    const int zero = 0;
    cudaMemcpyToSymbol(pattn::g_error, &zero, sizeof(int));
  }
  return h;
}

}  // namespace fdk

using namespace fdk;

static bool sizes_ok(int64_t num_segments, int64_t max_seqlen, int64_t max_kv_len, int64_t tokens, int64_t hq,
                     int64_t hkv, int64_t head_dim) {
  return num_segments >= 1 && num_segments <= 0x7ffffffe && max_seqlen >= 0 && max_seqlen <= 0x7fffffff &&
         max_kv_len >= 0 && max_kv_len <= 0x7fffff00 && tokens >= 0 && tokens <= 0x7fffffff && hkv >= 1 && hq >= 1 && hq <= 4096 &&
         hq % hkv == 0 && (head_dim == 128 || head_dim == 256);
}

extern "C" size_t fdk_paged_gqa_workspace_size(int64_t num_segments, int64_t max_seqlen, int64_t max_kv_len,
                                               int64_t tokens, int64_t hq, int64_t hkv, int64_t head_dim,
                                               int cache_is_e4m3) {
  if (!sizes_ok(num_segments, max_seqlen, max_kv_len, tokens, hq, hkv, head_dim)) return 0;
  const pattn::Plan pl = pattn::make_plan(num_segments, max_seqlen, max_kv_len, tokens, hkv, hq / hkv, head_dim, cache_is_e4m3 != 0);
  if (pl.nsplit == 1 || pl.clustered) return 0;
  return (size_t)pl.nsplit * tokens * hq * (head_dim * 4 + 8) + (pl.picked ? 16 : 0);  // + the part size
}

extern "C" int fdk_paged_gqa_fwd(const void* q, int64_t ld_q, const void* k_cache, int64_t ld_kpage,
                                 const void* v_cache, int64_t ld_vpage, int cache_is_e4m3, const void* k_scale,
                                 int64_t ld_kscale_page, const void* v_scale, int64_t ld_vscale_page,
                                 int64_t num_pages, int64_t page_size, const int32_t* page_table, int64_t ld_table,
                                 int64_t max_pages, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                 int64_t num_segments, int64_t max_seqlen, int64_t max_kv_len, int64_t tokens,
                                 int64_t hq, int64_t hkv, int64_t head_dim, float scale, const void* gate,
                                 int64_t ld_gate, int gate_interleaved, void* out, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  using namespace fdk::pattn;
  if (int st = check_device()) return st;
  const char* what = "paged_gqa";
  if (head_dim != 128 && head_dim != 256)
    return set_error(FDK_ERR_UNSUPPORTED, "%s: head_dim=%lld (128 and 256 supported)", what, (long long)head_dim);
  if (hkv < 1 || hq < 1 || hq % hkv) return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: hq must be a multiple of hkv", what);
  if (!sizes_ok(num_segments, max_seqlen, max_kv_len, tokens, hq, hkv, head_dim))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: bad segment count or sizes", what);
  if (!(scale > 0.f) || !(scale < 1e30f))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: scale must be positive and finite", what);
  int shift = 0;
  for (int i = 4; i <= 8; ++i)
    if (page_size == (int64_t)1 << i) shift = i;
  if (!shift) return set_error(FDK_ERR_UNSUPPORTED, "%s: page_size=%lld (16, 32, 64, 128 or 256)", what, (long long)page_size);
  if (tokens == 0) return FDK_OK;
  if (!q || !k_cache || !v_cache || !page_table || !cu_seqlens || !kv_lens || !out)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  const bool quant = cache_is_e4m3 != 0;
  if (quant && (!k_scale || !v_scale))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: an e4m3 cache needs k_scale and v_scale", what);
  if (num_pages < 1 || num_pages > 0x7fffffff || max_pages < 1 || max_pages > 0x7fffffff || ld_table < max_pages ||
      max_pages * page_size > MOST_POSITIONS)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: bad page counts (at most 2^31 - 2^16 positions a sequence)", what);
  const int64_t page_elems = page_size * hkv * head_dim;
  if (ld_kpage < page_elems || ld_vpage < page_elems ||
      (quant && (ld_kscale_page < page_size * hkv || ld_vscale_page < page_size * hkv)))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: page stride too small", what);
  if (ld_q < hq * head_dim || (gate && ld_gate < (gate_interleaved ? 2 * hq - 1 : hq) * head_dim))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: row stride too small", what);
  const int esz = quant ? 1 : 2;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) || ld_q % 8 ||
      ld_kpage * esz % 16 || ld_vpage * esz % 16 || (gate && (!aligned16(gate) || ld_gate % 8)) ||
      (quant && (!aligned16(k_scale) || !aligned16(v_scale) || ld_kscale_page % 16 || ld_vscale_page % 16)))
    return set_error(FDK_ERR_ALIGNMENT, "%s: pointers and strides must be 16-byte aligned", what);
  Plan pl = make_plan(num_segments, max_seqlen, max_kv_len, tokens, hkv, hq / hkv, head_dim, quant);
  if (std::min(max_seqlen, tokens) * (hq / hkv) > 0x7fffffff || hkv * (pl.many ? pl.units : num_segments * pl.row_blocks) > 0x7fffffff)
    return set_error(FDK_ERR_UNSUPPORTED, "%s: too many segments or query rows", what);
  Params p = {};
  p.q = static_cast<const bf16*>(q); p.ld_q = ld_q;
  p.k_cache = static_cast<const uint8_t*>(k_cache); p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.k_scale = static_cast<const uint8_t*>(k_scale); p.v_scale = static_cast<const uint8_t*>(v_scale);
  p.kpage = ld_kpage * esz; p.vpage = ld_vpage * esz;
  p.kscale_page = ld_kscale_page; p.vscale_page = ld_vscale_page;
  p.table = page_table; p.ld_table = ld_table; p.cu = cu_seqlens; p.kv_lens = kv_lens;
  p.tokens = tokens; p.num_pages = num_pages; p.nseg = (int)num_segments; p.max_pages = (int)max_pages;
  p.page_shift = shift; p.hq = (int)hq; p.hkv = (int)hkv; p.group = (int)(hq / hkv);
  p.nsplit = pl.nsplit; p.row_blocks = (int)pl.row_blocks; p.split_keys = pl.split_keys;
  p.max_seqlen = (int)max_seqlen;
  p.picked = pl.picked; p.clustered = pl.clustered; p.units = (int)pl.units;
  p.part_cost = (int)pl.part_cost;
  p.block_rows = pl.many ? (head_dim == 128 ? 2 : 1) * (128 / p.group) * p.group : pl.rows;
  p.sl2 = scale * 1.4426950408889634f;
  p.gate = static_cast<const bf16*>(gate); p.ld_gate = ld_gate;
  p.gate_hstride = (int)(gate_interleaved ? 2 * head_dim : head_dim);
  p.out = static_cast<bf16*>(out);
  if (pl.nsplit > 1 && !pl.clustered) {
    const size_t need = fdk_paged_gqa_workspace_size(num_segments, max_seqlen, max_kv_len, tokens, hq, hkv, head_dim, quant);
    if (!workspace || workspace_bytes < need)
      return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes needed", what, need);
    if (!aligned16(workspace)) return set_error(FDK_ERR_ALIGNMENT, "%s: workspace must be 16-byte aligned", what);
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)pl.nsplit * tokens * hq * head_dim);
    p.part_keys = reinterpret_cast<int*>(p.part_ml + (int64_t)pl.nsplit * tokens * hq);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int st;
  if (pl.many) {
    if (head_dim == 128)
      st = quant ? chunk::launch<128, true>(p, s) : chunk::launch<128, false>(p, s);
    else
      st = quant ? chunk::launch<256, true>(p, s) : chunk::launch<256, false>(p, s);
  } else if (head_dim == 128) st = quant ? launch_rows<128, true>(p, pl.rows, s) : launch_rows<128, false>(p, pl.rows, s);
  else st = quant ? launch_rows<256, true>(p, pl.rows, s) : launch_rows<256, false>(p, pl.rows, s);
  if (st || pl.nsplit == 1 || pl.clustered) return st;
  const int64_t rpw = head_dim == 128 ? 2 : 1;
  const int64_t warps = tokens * ((hq + rpw - 1) / rpw);
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((warps + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  if (head_dim == 128) cudaLaunchKernelEx(&cfg, join_kernel<128>, p);
  else cudaLaunchKernelEx(&cfg, join_kernel<256>, p);
  return check_launch("paged_gqa (join of splits)");
}
