// The many-row kernel of paged_attention.cu (included there): tcgen05 tensor cores, TMEM accumulators.
//
// Tensor-core bound: 128 or more rows share every cached row.  Rows are (token, head of the KV head's
// group) pairs, token-major, so one 128-row tile holds 128 / group tokens with all their heads -- no
// padding of short chunks to 128 tokens a head, and K/V are read once a group, not once a head.
//
//   head_dim 128: a CTA owns two 128-row tiles A, B, KV blocks of 128 keys.  Issue order per block j:
//     PV_A(j), S_A(j+1), PV_B(j), S_B(j+1): the softmax of one tile overlaps the MMAs of the other, and
//     PV starts on the block's first 64 keys while the softmax computes the weights of the other 64.
//     TMEM: S_A [0,128) S_B [128,256) O_A [256,384) O_B [384,512).
//   head_dim 256: one tile (two would not fit TMEM), KV blocks of 64 keys, S ping-pong one block ahead.
//     TMEM: S0 [0,64) S1 [64,128) Q [128,256) O [256,512).  Q is the S MMA's A operand from TMEM: read
//     from shared memory it would be 64 of the 192 KB a block moves there, and its 64 KB make room for
//     more KV slots.
//   P overwrites S in TMEM (A operand of the PV MMA).  Softmax: thread = row = TMEM lane, online in the
//   exp2 domain, O rescaled only when the running maximum grows by more than 2^8.
//
//   bf16 cache: one warp issues TMA loads, a box a page (or 128 / 64 keys of it) and 64 columns; a page id
//   outside the cache is an out-of-range coordinate, which TMA fills with zeros.  V rows at or behind
//   kv_lens[s] may hold anything (0 * NaN would reach the sums): the block that has them is zeroed there
//   after its load and before the MMA warp sees it.
//   8-bit cache: TMA brings the raw e4m3 rows; six converter warps turn them into fp16 operands (e4m3 ->
//   fp16 is exact) multiplied by the row's scale relative to the largest one of the CTA's key range and by
//   2^7, which takes e4m3's 448 to 57344, just inside fp16.  So scales within 2^22 of the largest are exact, down to
//   2^-31 of it elements are rounded to multiples of 2^-31 of it, and below the factor itself is 0.  The largest K
//   scale then folds into the softmax scale, V's into the final normalisation, so the softmax costs what it
//   does for bf16.  q goes to fp16 with a power of two a row.
//
//   K and V blocks share one ring of operand slots, in the order K_0 V_0 K_1 V_1 ..: four slots for bf16,
//   three for the 8-bit cache (PV of block j and S of block j + 1 hold two, the converters fill the
//   third), which leaves room for a ring of four raw tiles.
//
// Measured (B200, back to back in a graph): 2 x 2048 tokens behind 6144 and 14000 positions, 16 / 4 heads of 128, bf16: 241
// us, 1.10 PF/s; a block of 128 keys takes 3500 cycles where its MMAs take 2050, as long as the softmax's exponentials
// and the operands' shared-memory traffic each: no unit is full, a tile's chain of S, softmax, P and PV is what is
// left.  8 ragged chunks (2544 tokens behind 600 to 8000), e4m3, page 16: 109 us; 3700 cycles a block, 20000 before
// the first, and uneven CTAs (tensor pipe 27%, issue slots 30%).  48 questions of 9 to 70 tokens behind 1490 shared
// positions, 8 / 2 heads of 256, bf16: 42 us; a block of 64 keys brings 64 KB to an SM in its 2050 cycles, L2 as a whole
// 16% busy (which of the copies' latency and the SM's share of L2 sets this was not separated); the start and the
// epilogue of the one wave are a third of the call.  74 x 32 tokens behind 4096 shared positions, 8 / 2 heads of 256,
// e4m3: 93 us.  Whole prompts, no history, 16 / 4 heads of 128, bf16: 8192 tokens 252 us, 32 x 1024 299 us.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

namespace fdk {
namespace pattn {
namespace chunk {
using namespace sm100;

template <int D>
struct Geo {
  static constexpr int NT = D == 128 ? 2 : 1;          // 128-row tiles a CTA
  static constexpr int BN = D == 128 ? 128 : 64;       // keys a block
  static constexpr int NBX = D / 64;                   // 64-column (128-byte) boxes of a row
  static constexpr uint32_t QBOX = 128 * 128, KBOX = (uint32_t)BN * 128;
  static constexpr uint32_t QT = NBX * QBOX, KT = NBX * KBOX;
  static constexpr bool Q_TMEM = D == 256;
  static constexpr uint32_t TM_Q = 128;
  static constexpr uint32_t TM_S(int i) { return (uint32_t)(BN * i); }         // tile i, or ping-pong buffer i
  static constexpr uint32_t TM_O(int i) { return 256u + 128u * (uint32_t)i; }  // tile i
};
// Shared memory: Q tiles, operand ring, raw ring (8-bit cache), barriers and small state.
// barriers: F / E operand slot full / empty, RF / RE raw slot full / empty, S and P per tile or buffer (P2: P's
// second 64 keys, two tiles);
// VT: V of the block that ends past kv_lens, before its tail is zeroed
enum { B_Q = 0, B_F, B_E = B_F + 6, B_RF = B_E + 6, B_RE = B_RF + 4, B_S = B_RE + 4, B_P = B_S + 2, B_P2 = B_P + 2,
       B_VT = B_P2 + 2,
       B_PV, B_O, NBAR };
constexpr int RAW_SLOTS = 4;
template <int D, bool QUANT>
struct Smem {
  using G = Geo<D>;
  static constexpr int SLOTS = G::Q_TMEM ? (QUANT ? 4 : 6) : QUANT ? 3 : 4;
  static constexpr uint32_t RAWT = QUANT ? (uint32_t)(G::BN * D) : 0;  // bytes of a raw tile
  static constexpr uint32_t OFF_Q = 0, OFF_KV = G::Q_TMEM ? 0 : G::NT * G::QT, OFF_RAW = OFF_KV + SLOTS * G::KT,
                            OFF_BAR = OFF_RAW + RAW_SLOTS * RAWT, OFF_MISC = OFF_BAR + 8 * NBAR,
                            OFF_QS = OFF_MISC + 64,                       // row scale exponents of q: 256 bytes (head_dim 128)
                            OFF_FT = OFF_QS + (QUANT ? 256 : 0),          // row factors of two tiles: half2
                            OFF_STAGE = OFF_FT + (QUANT ? 1024 : 0),      // q on its way to TMEM: 4 KB a softmax warp
                            BYTES = OFF_STAGE + (G::Q_TMEM ? 16384 : 0) + 1024;  // + slack for 1024-byte alignment
  static_assert(OFF_MISC % 16 == 0, "alignment of the small state");
  static_assert(BYTES <= 232448, "shared memory of a CTA");
};
constexpr uint32_t TM_COLS = 512;
constexpr float P_SHIFT = 6.f;  // fp16 P is scaled by 2^6: weights down to 2^-30 of the row's largest stay
constexpr int ROW_SHIFT = 7;    // fp16 K and V of the 8-bit cache are scaled by 2^7
constexpr float ROW_UNIT = 1.f / (1 << ROW_SHIFT);
constexpr long long DRAIN_BUDGET = 2000000000LL;

// warps: NT * 4 softmax, one producer, one MMA issuer and TMEM allocator; with the 8-bit cache six
// converter warps, which fill the warpgroups (with four of them 8 ragged chunks took 128 us, not 115)
template <int D, bool QUANT>
struct Roles {
  static constexpr int PRODUCER = Geo<D>::NT * 4, MMA = PRODUCER + 1, CONV = MMA + 1;
  static constexpr int CT = QUANT ? 192 : 0;  // converter threads
  static constexpr int THREADS = CONV * 32 + CT;
  static constexpr bool SPLIT_REGS = QUANT && D == 128;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(dst),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ bool drain(uint32_t bar, uint32_t parity) {
  volatile int never = 0;
  return mbar_wait(bar, parity, &never, DRAIN_BUDGET);
}
// idesc_bf16 with fp16 operands (format field 0)
__host__ __device__ constexpr uint32_t idesc(int M, int N, bool b_mn_major, bool f16) {
  return idesc_bf16(M, N, false, b_mn_major) & (f16 ? ~((1u << 7) | (1u << 10)) : ~0u);
}
__device__ __forceinline__ uint32_t half2_bits(float x) {
  const __half2 h = __float2half2_rn(x);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x for two x <= 64 on the float32 pipe, for the share of the weights that would leave the softmax waiting for
// the special-function unit (16 results a clock and SM, half of what its two tiles take): x = n + f with
// |f| <= 1/2, 2^f by a cubic fitted to the least relative error (2^-13.7, below the fp16 and bf16
// roundings of P), 2^n from the bits of n + 127.  x below -126.5 gives 0; NaN stays NaN.
// Every 3rd pair of columns (2 x 2048 tokens behind 6144 and 14000, bf16, when it was chosen: none 275 us, every 2nd
// 268, 3rd 259, 4th 261, 6th 261).  Not with an 8-bit cache, whose converters need the issue slots (37 x 64 tokens
// behind 4096 shared positions: 98 us without, 110 with every 3rd, 103 with every 6th).
constexpr int EXP_POLY = 3;
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n" : "+f"(x.x));  // -127: the factor 2^n below is then 0
  asm("max.NaN.f32 %0, %0, 0fC2FE0000;\n" : "+f"(x.y));
  const float magic = 12582912.f + 127.f;  // 1.5 * 2^23: its sum with x holds round(x) + 127 in the low bits
  const float2 t = __fadd2_rn(x, make_float2(magic, magic));
  const float2 n = __fadd2_rn(t, make_float2(-magic, -magic));
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
  float2 y = make_float2(0.0551716685f, 0.0551716685f);
  y = __ffma2_rn(y, f, make_float2(0.2426111251f, 0.2426111251f));
  y = __ffma2_rn(y, f, make_float2(0.6932609677f, 0.6932609677f));
  y = __ffma2_rn(y, f, make_float2(0.9999280572f, 0.9999280572f));
  return __fmul2_rn(y, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

// 16-byte chunk c (8 columns) of row r in a [boxes of 64 columns][rows][128 B] operand tile, 128-byte swizzle
template <uint32_t BOX>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)(c >> 3) * BOX + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) * 16);
}

// The `rank`-th unit of work of the call (a warp's work), for calls whose segments fit one warp's lanes: the
// whole parts of all row tiles first, then each tile's last part (or the tile that is not split), both in
// descending order of the keys that the tile sees.  So the grid starts with the longest CTAs and launches
// what exists.  The number of tiles with at least L keys has a closed form a segment, so a tile is found
// by bisection over L with the segments spread over the lanes.  False when there are no more than `rank`
// units.
struct Unit {
  int s, rb, split;
};
__device__ __forceinline__ bool pick_unit(const Params& p, const Tiles& t, int part_keys, int rank, int lane, Unit& u) {
  auto count1 = [&](int i, int L) {  // tiles of the lane's segment i that see at least L keys
    if (L <= 0) return t.tiles[i];
    if (t.tiles[i] == 0 || t.past[i] + t.n[i] < L) return 0;
    const int need = max(min(L - t.past[i], t.n[i]), 1);  // the first tile with (rb + 1) tokens >= need
    return t.tiles[i] - t.div_up(need) + 1;
  };
  auto count = [&](int L) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < PICK; ++i) c += count1(i, L);
    return (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
  };
  u.split = -1;
  for (int i = 0; i + 1 < p.nsplit; ++i) {  // tiles whose part i is a whole one and not their last
    const int64_t more = (int64_t)(i + 1) * part_keys + 1;
    const int c = more > t.most ? 0 : count((int)more);
    if (c == 0) break;
    if (rank < c) {
      u.split = i;
      break;
    }
    rank -= c;
  }
  if (count(0) <= rank) return false;
  int lo = t.least, hi = t.most + 1;  // count(lo) > rank >= count(hi)
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (count(mid) > rank) lo = mid;
    else hi = mid;
  }
  // of the tiles with exactly lo keys, in segment order
  int skip = rank - count(lo + 1), mine = 0, eq[PICK];
#pragma unroll
  for (int i = 0; i < PICK; ++i) mine += eq[i] = count1(i, lo) - count1(i, lo + 1);
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += x;
  }
  skip -= before - mine;
  int found = -1, rb = 0;
#pragma unroll
  for (int i = 0; i < PICK; ++i) {
    if (found < 0 && skip >= 0 && skip < eq[i]) {
      found = lane * PICK + i;
      rb = t.tiles[i] - count1(i, lo) + skip;
    }
    skip -= eq[i];
  }
  const unsigned who = __ballot_sync(0xffffffffu, found >= 0);
  const int src = __ffs(who) - 1;
  u.s = __shfl_sync(0xffffffffu, found, src);
  u.rb = __shfl_sync(0xffffffffu, rb, src);
  // lo: the tile's keys.  Without parts part_keys is the host's, from its hint, and bounds nothing.
  if (u.split < 0) u.split = p.nsplit > 1 ? min((lo - 1) / part_keys, p.nsplit - 1) : 0;
  return true;
}

template <int D, bool QUANT>
__global__ void __launch_bounds__(Roles<D, QUANT>::THREADS, 1)
many_rows_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                 const __grid_constant__ CUtensorMap tv, const Params p) {
  using G = Geo<D>;
  using M = Smem<D, QUANT>;
  using R = Roles<D, QUANT>;
  constexpr int NT = G::NT, BN = G::BN, NBX = G::NBX;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + M::OFF_BAR;
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + M::OFF_MISC);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + M::OFF_MISC + 4);
  volatile int* scale_max = reinterpret_cast<volatile int*>(gbase + M::OFF_MISC + 8);  // largest K, V scale byte
  int* warp_max = reinterpret_cast<int*>(gbase + M::OFF_MISC + 16);                    // [6][2]; over `pick`, read by then
  uint8_t* q_exp = gbase + M::OFF_QS;
  uint32_t* factor = reinterpret_cast<uint32_t*>(gbase + M::OFF_FT);                   // [2][BN] half2

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int tpt = 128 / p.group;                 // tokens a tile
  const int rpt = tpt * p.group;                 // rows of it in use
  // grid: with few segments x = (units of work, KV head), the head fastest, longest first (short calls end
  // on their longest CTA, and only the device knows the lengths).  With many, x counts each segment's row
  // tiles up to the longest one's number, from the last tile down, and y the splits of the keys from the
  // last one (only long ranges have it: short tiles come at the end).
  const int hk = (int)(blockIdx.x % (unsigned)p.hkv), item = (int)(blockIdx.x / (unsigned)p.hkv);
  int s, rb, split, part_keys = p.split_keys;
  if (p.picked) {
    int* pick = reinterpret_cast<int*>(gbase + M::OFF_MISC + 48);
    if (warp == 0) {
      Tiles t;
      t.load(p, NT * tpt, lane);
      if (p.nsplit > 1) part_keys = best_part_keys(p, t, lane);
      Unit u = {-1, 0, 0};
      const bool some = pick_unit(p, t, part_keys, item, lane, u);
      if (lane == 0) {
        pick[0] = some ? u.s : -1;
        pick[1] = u.rb;
        pick[2] = u.split;
        pick[3] = part_keys;
        if (p.nsplit > 1 && item == 0 && hk == 0) *p.part_keys = part_keys;
      }
    }
    __syncthreads();
    s = pick[0];
    rb = pick[1];
    split = pick[2];
    part_keys = pick[3];
  } else {
    s = item % p.nseg;
    rb = p.row_blocks - 1 - item / p.nseg;
    split = p.nsplit - 1 - (int)blockIdx.y;
  }
  if (item == 0 && hk == 0 && blockIdx.y == 0) {  // one CTA reports what is wrong with the segments
    for (int i = tid; i < p.nseg; i += R::THREADS)
      if (segment(p, i, true).n > p.max_seqlen) atomicOr(&g_error, 1);
  }
  if (s < 0) return;
  const Seg seg = segment(p, s, false);
  const int rows = seg.n * p.group;
  const int tok0 = rb * NT * tpt;                // first token of the CTA
  if (tok0 >= seg.n) return;
  const int last_tok = min(tok0 + NT * tpt, seg.n) - 1;
  const int64_t kend64 = seg.past + last_tok + 1;
  const int kend = kend64 > 0 ? (int)kend64 : 0;
  const int kv_len = (int)(seg.past + seg.n);
  int kb, ke;
  split_range(p, part_keys, split, kend, kb, ke);
  if (kb >= ke && split > 0) return;  // the join does not read this part
  const int n_kv = (ke - kb + BN - 1) / BN;
  const bool part = in_parts(p, part_keys, kend);
  if (n_kv == 0) {  // no keys at all: zeros
    for (int e = tid; e < NT * rpt; e += R::THREADS) {
      const int64_t gr = (int64_t)tok0 * p.group + e;
      if (gr >= rows) break;
      const int64_t idx = (seg.begin + gr / p.group) * p.hq + hk * p.group + gr % p.group;
      for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(p.out + idx * D + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  // the second tile may have no rows: its MMAs are skipped
  const bool two = NT == 2 && tok0 + tpt < seg.n;

  if (tid == 0) {
    for (int i = 0; i < NBAR; ++i) {
      uint32_t count = 1;
      if (i >= B_P && i < B_P2 + 2) count = 128;
      if ((QUANT || G::Q_TMEM) && i == B_Q) count = two ? 256 : 128;
      if (QUANT && ((i >= B_F && i < B_F + 6) || (i >= B_RE && i < B_RE + 4))) count = R::CT;
      mbar_init(bar(i), count);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == R::MMA) {
    tmem_alloc(smem_u32(tmem_slot), TM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int32_t* table = p.table + (int64_t)s * p.ld_table;
  const int page_mask = (1 << p.page_shift) - 1;

  // ------------------------------------------------------------------ TMA producer (one whole warp)
  // items 2 j and 2 j + 1 are K and V of block j; ring of operand slots (bf16) or raw slots (8-bit cache)
  auto producer = [&]() {
    constexpr int RING = QUANT ? RAW_SLOTS : M::SLOTS;
    constexpr int FULL = QUANT ? B_RF : B_F, EMPTY = QUANT ? B_RE : B_E;
    constexpr uint32_t BYTES = QUANT ? M::RAWT : G::KT;
    // a block's boxes: keys in pages of 2^page_shift, at most BN a box
    const int box_keys = min(BN, 1 << p.page_shift);
    constexpr int COLS = QUANT ? 1 : NBX;  // boxes across a row: the raw row, or 64 bf16 columns each
    const int boxes = (BN / box_keys) * COLS;
    if (lane == 0) {
      prefetch_tmap(&tk);
      prefetch_tmap(&tv);
      if (!QUANT && !G::Q_TMEM) {
        const int tiles = two ? 2 : 1;
        mbar_expect_tx(bar(B_Q), (uint32_t)(tiles * NBX) * 128u * (uint32_t)rpt);
        for (int i = 0; i < tiles; ++i)
          for (int b = 0; b < NBX; ++b)
            tma_load_3d(base + M::OFF_Q + i * G::QT + b * G::QBOX, &tq, bar(B_Q), b * 64, hk * p.group,
                        seg.begin + tok0 + i * tpt);
      }
    }
    // at most 16 boxes: lane b issues box b.  Its page id is loaded a block ahead.
    const int sub = lane / COLS, col = lane % COLS;
    auto page_of = [&](int j) { return __ldg(table + (min(kb + j * BN + sub * box_keys, ke - 1) >> p.page_shift)); };
    int id = 0, id_next = page_of(0);
    int issued = 0;
    for (int i = 0; i < 2 * n_kv; ++i) {
      if ((i & 1) == 0) {
        id = id_next;
        id_next = page_of((i >> 1) + 1);
      }
      const int slot = i % RING;
      if (i >= RING &&
          !__all_sync(0xffffffffu, mbar_wait(bar(EMPTY + slot), (uint32_t)(i / RING - 1) & 1u, abort_flag) ? 1 : 0))
        break;
      const bool is_v = i & 1;
      const int key0 = kb + (i >> 1) * BN;
      const int live = kv_len - key0;                      // rows of the block that are cached positions
      const bool tail = !QUANT && is_v && live < BN;       // at most the last block
      const uint32_t fb = bar(tail ? B_VT : FULL + slot);
      const uint32_t dst = base + (QUANT ? M::OFF_RAW + slot * M::RAWT : M::OFF_KV + slot * G::KT);
      if (lane == 0) mbar_expect_tx(fb, BYTES);
      __syncwarp();
      if (lane < boxes) {
        const int key = key0 + sub * box_keys;
        int page = (int)p.num_pages;  // out of range: zeros
        if (key < ke) {
          if (id >= 0 && id < p.num_pages) page = id;
          else atomicOr(&g_error, 1);
        }
        const uint32_t at = QUANT ? (uint32_t)(sub * box_keys * D) : (uint32_t)col * G::KBOX + (uint32_t)(sub * box_keys) * 128u;
        tma_load_4d(dst + at, is_v ? &tv : &tk, fb, col * 64, key & page_mask, hk, page);
      }
      issued = i + 1;
      if (tail) {
        drain(bar(B_VT), 0);
        __syncwarp();
        uint8_t* v = gbase + M::OFF_KV + slot * G::KT;
        for (int e = lane; e < (BN - live) * NBX * 8; e += 32) {
          const int r = live + e / (NBX * 8), c = e % (NBX * 8);
          *reinterpret_cast<uint4*>(v + chunk_at<G::KBOX>(r, c)) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(FULL + slot));
      }
    }
    // drain: every issued load must have landed before shared memory is released
    if (lane == 0) {
      if (!QUANT && !G::Q_TMEM) drain(bar(B_Q), 0);
      for (int i = (issued > RING ? issued - RING : 0); i < issued; ++i) drain(bar(FULL + i % RING), (uint32_t)(i / RING) & 1u);
    }
  };

  if (warp >= R::PRODUCER) {
    // With the 8-bit cache at head_dim 128, 512 threads are launched with 128 registers each; the softmax
    // needs more (a row of S and of P), the other two warpgroups less: 256 * 192 + 256 * 64 = 65536.
    if constexpr (R::SPLIT_REGS) reg_dec<64>();
    if (warp == R::PRODUCER) {
      producer();
    } else if (warp == R::MMA) {
      // ------------------------------------------------------------------ MMA issuer
      if (lane == 0) {
        constexpr uint32_t ID_QK = idesc(128, BN, false, QUANT);
        constexpr uint32_t ID_PV = idesc(128, D, true, QUANT);  // V is MN-major (columns contiguous)
        auto issue_s = [&](int j, int tile, uint32_t tm) {
          const uint64_t dq = G::Q_TMEM ? 0 : sdesc_sw128(base + M::OFF_Q + tile * G::QT, 16, 1024);
          const uint64_t dk = sdesc_sw128(base + M::OFF_KV + (2 * j % M::SLOTS) * G::KT, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t qo = ((kk >> 2) * G::QBOX + (kk & 3) * 32) >> 4, ko = ((kk >> 2) * G::KBOX + (kk & 3) * 32) >> 4;
            if (G::Q_TMEM) umma_ts(tmem + tm, tmem + G::TM_Q + 8 * kk, dk + ko, ID_QK, kk > 0);
            else umma_ss(tmem + tm, dq + qo, dk + ko, ID_QK, kk > 0);
          }
        };
        auto issue_pv = [&](int j, uint32_t tm_p, uint32_t tm_o, int k0) {
          const uint64_t dv = sdesc_sw128(base + M::OFF_KV + ((2 * j + 1) % M::SLOTS) * G::KT, G::KBOX, 1024);
#pragma unroll
          for (int kk = k0; kk < k0 + 4; ++kk)  // 64 keys
            umma_ts(tmem + tm_o, tmem + tm_p + 8 * kk, dv + (uint32_t)(kk * 2048 >> 4), ID_PV, (j > 0 || kk > 0) ? 1u : 0u);
        };
        auto wait = [&](int i, int parity) { return mbar_wait(bar(i), (uint32_t)parity & 1u, abort_flag); };
        auto full = [&](int item) { return wait(B_F + item % M::SLOTS, item / M::SLOTS); };
        auto release = [&](int item) { umma_commit(bar(B_E + item % M::SLOTS)); };
        bool ok = wait(B_Q, 0) && full(0);
        if (NT == 2) {
          if (ok) {
            tc_fence_after();
            issue_s(0, 0, G::TM_S(0));
            umma_commit(bar(B_S));
            if (two) {
              issue_s(0, 1, G::TM_S(1));
              umma_commit(bar(B_S + 1));
            }
            release(0);
          }
          for (int j = 0; ok && j < n_kv; ++j) {
            const bool more = j + 1 < n_kv;
            if (!full(2 * j + 1) || !wait(B_P, j)) break;
            tc_fence_after();
            issue_pv(j, G::TM_S(0), G::TM_O(0), 0);
            if (!wait(B_P2, j)) break;
            tc_fence_after();
            issue_pv(j, G::TM_S(0), G::TM_O(0), 4);
            if (more) {
              if (!full(2 * j + 2)) break;
              tc_fence_after();
              issue_s(j + 1, 0, G::TM_S(0));
              umma_commit(bar(B_S));
            }
            if (two) {
              if (!wait(B_P + 1, j)) break;
              tc_fence_after();
              issue_pv(j, G::TM_S(1), G::TM_O(1), 0);
              if (!wait(B_P2 + 1, j)) break;
              tc_fence_after();
              issue_pv(j, G::TM_S(1), G::TM_O(1), 4);
            }
            release(2 * j + 1);
            if (more) {
              if (two) {
                issue_s(j + 1, 1, G::TM_S(1));
                umma_commit(bar(B_S + 1));
              }
              release(2 * j + 2);
            }
          }
        } else {
          auto s_block = [&](int j) {
            issue_s(j, 0, G::TM_S(j & 1));
            umma_commit(bar(B_S + (j & 1)));
            release(2 * j);
          };
          if (ok) {
            tc_fence_after();
            s_block(0);
            if (n_kv > 1 && (ok = full(2))) {
              tc_fence_after();
              s_block(1);
            }
          }
          for (int j = 0; ok && j < n_kv; ++j) {
            if (!full(2 * j + 1) || !wait(B_P + (j & 1), j >> 1)) break;
            tc_fence_after();
            issue_pv(j, G::TM_S(j & 1), G::TM_O(0), 0);
            umma_commit(bar(B_PV));
            release(2 * j + 1);
            if (j + 2 < n_kv) {
              if (!full(2 * j + 4)) break;
              tc_fence_after();
              s_block(j + 2);
            }
          }
        }
        umma_commit(bar(B_O));  // arrives when every MMA above has completed
        drain(bar(B_O), 0);
      }
    } else if constexpr (QUANT) {
      // ------------------------------------------------------------------ converters
      const int ct = tid - R::CONV * 32, cw = ct >> 5;
      auto slot_of = [&](int key) { return (hk << p.page_shift) + (key & page_mask); };
      const int my = ct < BN ? ct : 0;
      auto page_at = [&](int key) { return __ldg(table + (min(key, ke - 1) >> p.page_shift)); };
      auto scale_at = [&](const uint8_t* scales, int64_t page_ld, int key, int id) -> int {
        const bool live = (uint32_t)id < (uint32_t)p.num_pages && key < ke;  // a bad id is reported by the producer
        const int b = __ldg(scales + ((live ? id : 0) * page_ld + slot_of(key)));
        return live ? b : 0;
      };
      int id = page_at(kb + my);
      int kbyte = scale_at(p.k_scale, p.kscale_page, kb + my, id), vbyte = scale_at(p.v_scale, p.vscale_page, kb + my, id);
      id = page_at(kb + BN + my);
      // largest scale bytes of the range, 16 keys a load
      uint32_t mk = 0, mv = 0;
      constexpr int AHEAD = 4;  // page ids, then scales, of that many steps in flight
      for (int key0 = kb + ct * 16; key0 < ke; key0 += AHEAD * R::CT * 16) {
        int64_t ids[AHEAD];
        uint4 a[AHEAD], b[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) ids[u] = __ldg(table + (min(key0 + u * R::CT * 16, ke - 1) >> p.page_shift));
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int key = key0 + u * R::CT * 16;
          a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);
          if (key < ke && ids[u] >= 0 && ids[u] < p.num_pages) {  // a bad id is reported by the loads below
            a[u] = __ldg(reinterpret_cast<const uint4*>(p.k_scale + ids[u] * p.kscale_page + slot_of(key)));
            b[u] = __ldg(reinterpret_cast<const uint4*>(p.v_scale + ids[u] * p.vscale_page + slot_of(key)));
          }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int key = key0 + u * R::CT * 16;
          const uint32_t aw[4] = {a[u].x, a[u].y, a[u].z, a[u].w}, bw[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int left = ke - (key + 4 * i);  // bytes of this word inside the range
            const uint32_t mask = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
            mk = __vmaxu4(mk, aw[i] & mask);
            mv = __vmaxu4(mv, bw[i] & mask);
          }
        }
      }
      auto byte_max = [](uint32_t w) { return max(max(w & 255u, (w >> 8) & 255u), max((w >> 16) & 255u, w >> 24)); };
      mk = __reduce_max_sync(0xffffffffu, byte_max(mk));
      mv = __reduce_max_sync(0xffffffffu, byte_max(mv));
      if (lane == 0) {
        warp_max[2 * cw] = (int)mk;
        warp_max[2 * cw + 1] = (int)mv;
      }
      asm volatile("bar.sync 1, 192;\n" ::: "memory");
      int ek = 0, ev = 0;
#pragma unroll
      for (int i = 0; i < R::CT / 32; ++i) {
        ek = max(ek, warp_max[2 * i]);
        ev = max(ev, warp_max[2 * i + 1]);
      }
      if (ct == 0) {  // the softmax reads them behind the first S, the epilogue later still
        scale_max[0] = ek;
        scale_max[1] = ev;
      }
      constexpr int TPR = D / 8, RPP = R::CT / TPR;  // threads a row, rows a pass
      const int lc = ct % TPR, lr = ct / TPR;
      // Items: thread ct is row ct's keeper (its scale byte, loaded a block ahead) and, for the conversion,
      // piece lc (8 columns) of rows lr, lr + RPP, ..: 8 raw bytes become one 16-byte operand chunk.  Eight
      // neighbouring threads read 64 consecutive bytes and store all eight chunk positions: no conflicts.
      constexpr int PASSES = (BN + RPP - 1) / RPP;  // the last one is short
      // Rows loaded before the first store (the compiler keeps their order, so a load behind a store waits for it): at
      // head_dim 256 the converters set the pace (74 x 32 tokens behind 4096 shared positions: 92 us with 4, 93
      // with 6, 97 with 8; 130 with 1 and four warps); at 128 issue slots do, which the softmax needs as well (37 x
      // 64: 95 us with 1, 96.5 with 2, 96 with 4; a test of `live` in full blocks too cost 15%).
      constexpr int BURST = D == 128 ? 1 : 4;
      // once a wait has run out, a thread only keeps step at the named barrier (the others may be behind it)
      bool ok = true;
      for (int j = 0; j < n_kv; ++j) {
        const int key0 = kb + j * BN;
        const uint32_t fk = half2_bits(scale_value(max(kbyte - ek + 127 + ROW_SHIFT, 0)));
        const uint32_t fv = half2_bits(scale_value(max(vbyte - ev + 127 + ROW_SHIFT, 0)));
        // rows behind the range may hold anything, NaN included: their operands are zeros, not 0 * NaN
        const int live = ke - key0;
        kbyte = scale_at(p.k_scale, p.kscale_page, key0 + BN + my, id);
        vbyte = scale_at(p.v_scale, p.vscale_page, key0 + BN + my, id);
        id = page_at(key0 + 2 * BN + my);
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          const int item = 2 * j + which, raw_slot = item % RAW_SLOTS, slot = item % M::SLOTS;
          if (ct < BN) factor[which * BN + ct] = which ? fv : fk;
          asm volatile("bar.sync 1, 192;\n" ::: "memory");  // factors written; also: nobody still reads the other table
          ok = ok && mbar_wait(bar(B_RF + raw_slot), (uint32_t)(item / RAW_SLOTS) & 1u, abort_flag) &&
               (item < M::SLOTS || mbar_wait(bar(B_E + slot), (uint32_t)(item / M::SLOTS - 1) & 1u, abort_flag));
          if (!ok) continue;
          const uint8_t* src = gbase + M::OFF_RAW + raw_slot * M::RAWT + lr * D + lc * 8;
          uint8_t* dst = gbase + M::OFF_KV + slot * G::KT;
          const uint32_t* fac = factor + which * BN + lr;
          auto convert = [&](bool partial) {
#pragma unroll
            for (int i0 = 0; i0 < PASSES; i0 += BURST) {
              uint2 w[BURST];
              uint32_t f[BURST];
#pragma unroll
              for (int i = 0; i < BURST; ++i) {
                if (i0 + i >= PASSES || ((i0 + i + 1) * RPP > BN && lr + (i0 + i) * RPP >= BN)) continue;
                w[i] = *reinterpret_cast<const uint2*>(src + (i0 + i) * RPP * D);
                if (partial && lr + (i0 + i) * RPP >= live) w[i] = make_uint2(0u, 0u);
                f[i] = fac[(i0 + i) * RPP];
              }
#pragma unroll
              for (int i = 0; i < BURST; ++i) {
                if (i0 + i >= PASSES || ((i0 + i + 1) * RPP > BN && lr + (i0 + i) * RPP >= BN)) continue;
                uint4 h;
                h.x = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)w[i].x), f[i]);
                h.y = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)(w[i].x >> 16)), f[i]);
                h.z = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)w[i].y), f[i]);
                h.w = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)(w[i].y >> 16)), f[i]);
                *reinterpret_cast<uint4*>(dst + chunk_at<G::KBOX>(lr + (i0 + i) * RPP, lc)) = h;
              }
            }
          };
          if (live >= BN) convert(false);
          else convert(true);
          fence_proxy_async_smem();
          mbar_arrive(bar(B_F + slot));
          mbar_arrive(bar(B_RE + raw_slot));
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax
    if constexpr (R::SPLIT_REGS) reg_inc<192>();
    const int tile = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_base + G::TM_O(tile);
    const int tok = tok0 + tile * tpt + row / p.group;
    const bool valid = row < rpt && tok < seg.n;
    const int64_t lim64 = valid ? seg.past + tok : -1;  // last visible key
    const int lim = (int)(lim64 > kend ? kend : lim64 < -1 ? -1 : lim64);
    float r_run = -INFINITY, l_run = 0.f;  // running maximum (unscaled) and sum
    bool ok = tile == 0 || two;
    float sl2 = p.sl2;
    if (G::Q_TMEM) {
      // q's row of this thread to its TMEM lane, two elements a column; 8-bit cache: as fp16 with the row's
      // largest magnitude in [1, 2).  Read with eight lanes to 128 bytes of a row, turned in shared memory.
      const int64_t q_at = (int64_t)(seg.begin + (valid ? tok : 0)) * p.ld_q + (int64_t)(hk * p.group + (valid ? row % p.group : 0)) * D;
      const int r8 = lane >> 3, c8 = lane & 7;  // a pass: rows 4 i + r8, columns 8 c8 .. + 7
      // Straight code runs at the speed of instruction fetches: the loops stay rolled.
      uint4 w[8];
      auto load = [&](int c) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = __ldg(reinterpret_cast<const uint4*>(p.q + __shfl_sync(0xffffffffu, q_at, 4 * i + r8) + c * 64 + c8 * 8));
      };
      float inv = 1.f, unit = 1.f;
      if (QUANT) {
        float m[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = 0.f;
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          load(c);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            __nv_bfloat162 x = __habs2(*reinterpret_cast<__nv_bfloat162*>(&w[i].x));
            x = __hmax2(x, __habs2(*reinterpret_cast<__nv_bfloat162*>(&w[i].y)));
            x = __hmax2(x, __habs2(*reinterpret_cast<__nv_bfloat162*>(&w[i].z)));
            x = __hmax2(x, __habs2(*reinterpret_cast<__nv_bfloat162*>(&w[i].w)));
            m[i] = fmaxf(m[i], fmaxf(__low2float(x), __high2float(x)));
          }
        }
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
          const float x = __shfl_sync(0xffffffffu, m[i], (lane & 3) * 8);  // row 4 i + (lane & 3)
          if (lane >> 2 == i) a = x;
        }
        const int e = a == 0.f ? 127 : min(max((int)(__float_as_uint(a) >> 23), 1), 253);
        inv = __uint_as_float((uint32_t)(254 - e) << 23);
        unit = __uint_as_float((uint32_t)e << 23);
      }
      load(0);
      const uint32_t stage = base + M::OFF_STAGE + (uint32_t)warp * 4096u;
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + r8;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(stage + (uint32_t)(r * 128 + ((c8 ^ (r & 7)) * 16))),
                       "r"(w[i].x), "r"(w[i].y), "r"(w[i].z), "r"(w[i].w)
                       : "memory");
        }
        __syncwarp();
        if (c + 1 < D / 64) load(c + 1);
        uint32_t col[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t ww[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                       : "=r"(ww[0]), "=r"(ww[1]), "=r"(ww[2]), "=r"(ww[3])
                       : "r"(stage + (uint32_t)(lane * 128 + ((i ^ (lane & 7)) * 16)))
                       : "memory");
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ww[u]));
            col[4 * i + u] = QUANT ? pack_f16x2(x.x * inv, x.y * inv) : ww[u];
          }
        }
        __syncwarp();
        tmem_st32(tmem + lane_base + G::TM_Q + c * 32, col);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(bar(B_Q));
      if (QUANT) {
        // S of the first block follows the scale maxima
        ok = __all_sync(0xffffffffu, mbar_wait(bar(B_S), 0, abort_flag) ? 1 : 0);
        // never 0: a masked score is -inf * sl2
        if (ok) sl2 = fmaxf(sl2 * ROW_UNIT * unit * scale_value(scale_max[0]), 1e-37f);
      }
    } else if (QUANT && ok) {
      // this tile's q: D / 8 threads a row, fp16 with the row's largest magnitude in [1, 2)
      constexpr int TPR = D / 8, RPP = 128 / TPR;
      const int ct = tid & 127, lc = ct % TPR, lr = ct / TPR;
      const int inv_group = 65536 / p.group + 1;  // x / group == x * inv_group >> 16 for x < 128
#pragma unroll 1
      for (int r0 = lr; r0 < 128; r0 += 8 * RPP) {
        uint4 w[8];  // eight rows' loads in flight, from a valid row where there is none
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int r = r0 + u * RPP, dt = r * inv_group >> 16, t = tok0 + tile * tpt + dt;
          const bool live = r < rpt && t < seg.n;
          w[u] = __ldg(reinterpret_cast<const uint4*>(p.q + (int64_t)(seg.begin + (live ? t : 0)) * p.ld_q +
                                                      (int64_t)(hk * p.group + (live ? r - dt * p.group : 0)) * D + lc * 8));
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int r = r0 + u * RPP;
          float f[8], a = 0.f;
          unpack8(w[u], f);
#pragma unroll
          for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(f[i]));
#pragma unroll
          for (int o = TPR / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
          const int e = a == 0.f ? 127 : min(max((int)(__float_as_uint(a) >> 23), 1), 253);
          const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
          if (lc == 0) q_exp[tile * 128 + r] = (uint8_t)e;  // q's row is fp16 * 2^(e - 127)
          *reinterpret_cast<uint4*>(gbase + M::OFF_Q + tile * G::QT + chunk_at<G::QBOX>(r, lc)) =
              make_uint4(pack_f16x2(f[0] * inv, f[1] * inv), pack_f16x2(f[2] * inv, f[3] * inv),
                         pack_f16x2(f[4] * inv, f[5] * inv), pack_f16x2(f[6] * inv, f[7] * inv));
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(bar(B_Q));
      // S of the first block follows every thread's q and the scale maxima
      ok = __all_sync(0xffffffffu, mbar_wait(bar(B_S + (NT == 2 ? tile : 0)), 0, abort_flag) ? 1 : 0);
      // never 0: a masked score is -inf * sl2
      if (ok) sl2 = fmaxf(sl2 * ROW_UNIT * scale_value(q_exp[tile * 128 + row]) * scale_value(scale_max[0]), 1e-37f);
    }
    const int n_blocks = ok ? n_kv : 0;
    for (int j = 0; j < n_blocks; ++j) {
      const int buf = NT == 2 ? tile : (j & 1);
      const uint32_t tS = tmem + lane_base + G::TM_S(buf);
      // warp-uniform: the tcgen05.ld below is warp-collective
      if (!__all_sync(0xffffffffu, mbar_wait(bar(B_S + buf), (NT == 2 ? j : j >> 1) & 1, abort_flag) ? 1 : 0)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sr[BN / 32][32];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) tmem_ld32(tS + c * 32, sr[c]);
      tmem_ld_wait();
      const int vis = lim - (kb + j * BN);  // columns 0 .. vis are visible
      if (__any_sync(0xffffffffu, vis < BN - 1)) {
#pragma unroll
        for (int c = 0; c < BN / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i > vis) sr[c][i] = __float_as_uint(-INFINITY);
      }
      float mx8[8];
#pragma unroll
      for (int a = 0; a < 8; ++a) mx8[a] = __uint_as_float(sr[0][a]);
#pragma unroll
      for (int i = 8; i < BN; i += 2)  // three-operand maximum, eight chains
        mx8[(i >> 1) & 7] = max3(mx8[(i >> 1) & 7], __uint_as_float(sr[i >> 5][i & 31]), __uint_as_float(sr[(i + 1) >> 5][(i + 1) & 31]));
      const float mx = fmaxf(max3(mx8[0], mx8[1], mx8[2]), max3(max3(mx8[3], mx8[4], mx8[5]), mx8[6], mx8[7]));
      float alpha = 1.f;
      bool rescale = false;
      if (j == 0) {
        r_run = mx;
      } else if ((mx - r_run) * sl2 > 8.0f) {  // also from nothing visible so far (-inf): alpha = 0
        alpha = ex2((r_run - mx) * sl2);
        r_run = mx;
        rescale = true;
      }
      // a row that has seen nothing yet: every exponent below is -inf
      const float r0 = r_run == -INFINITY ? 0.f : r_run;
      const float shift = r0 * sl2 - (QUANT ? P_SHIFT : 0.f);
      if (__any_sync(0xffffffffu, rescale)) {  // O row *= alpha
        // NT == 2: S_j's commit covers PV(j-1) of this tile; NT == 1: it covers PV(j-2), so wait for PV(j-1)
        if (NT == 1 && !__all_sync(0xffffffffu, mbar_wait(bar(B_PV), (j - 1) & 1, abort_flag) ? 1 : 0)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(tO + c * 32, o);
        }
      }
      float2 sum4[4];  // packed float32: two columns an operation
#pragma unroll
      for (int a = 0; a < 4; ++a) sum4[a] = make_float2(0.f, 0.f);
      const float2 sl2v = make_float2(sl2, sl2);
      // s * sl2 - shift in one operation, unless scores are so large that shift's own rounding (float32
      // spacing 0.25 and more) would show in the exponent
      const bool large = __any_sync(0xffffffffu, fabsf(shift) > 2097152.f);
#pragma unroll
      for (int half = 0; half < BN / 64; ++half) {
        uint32_t pk[32];
        auto weights = [&](auto expo) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int i = half * 64 + 2 * c;
            const float2 x = expo(make_float2(__uint_as_float(sr[i >> 5][i & 31]), __uint_as_float(sr[(i + 1) >> 5][(i + 1) & 31])));
            const float2 e = NT == 2 && !QUANT && c % EXP_POLY == EXP_POLY - 1 ? exp2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
            sum4[c & 3] = __fadd2_rn(sum4[c & 3], e);
            pk[c] = QUANT ? pack_f16x2(e.x, e.y) : pack_bf16x2(e.x, e.y);
          }
        };
        if (!large)
          weights([&](float2 x) { return __ffma2_rn(x, sl2v, make_float2(-shift, -shift)); });
        else
          weights([&](float2 x) {
            const float up = QUANT ? P_SHIFT : 0.f;
            return __ffma2_rn(make_float2(x.x - r0, x.y - r0), sl2v, make_float2(up, up));
          });
        tmem_st32(tS + half * 32, pk);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar(half == 0 ? B_P + buf : B_P2 + buf));
      }
      const float2 sum2 = __fadd2_rn(__fadd2_rn(sum4[0], sum4[1]), __fadd2_rn(sum4[2], sum4[3]));
      l_run = l_run * alpha + (sum2.x + sum2.y);
    }
    // ------------------------------------------------------------------ epilogue
    // A thread's row of O is 2 D bytes from its neighbour's: stored (and its gate loaded) row by row, every
    // access of a warp would touch 32 lines.  So 32 rows x 64 columns at a time go through the warp's part of
    // the operands' shared memory, free by now, and eight lanes hold 128 bytes of one row.  The gate's rows follow it
    // there, all of them at once.  16-byte chunks are XORed with the row: no bank conflicts either way.
    // This code runs once a CTA, at the speed of instruction fetches: the loops stay rolled.
    const int64_t tk_ = (int64_t)seg.begin + tok;
    const int head = hk * p.group + row % p.group;
    const int64_t idx = tk_ * p.hq + head;
    const bool gated = p.gate != nullptr && !part;
    const unsigned live = __ballot_sync(0xffffffffu, valid);
    const int64_t gate_at = tk_ * p.ld_gate + (int64_t)head * p.gate_hstride;
    const int r8 = lane >> 3, c8 = lane & 7;  // a pass: rows 4 i + r8, columns 8 c8 .. + 7
    if (ok && __all_sync(0xffffffffu, mbar_wait(bar(B_O), 0, abort_flag) ? 1 : 0)) {
      tc_fence_after();
      // l and O both carry 2^P_SHIFT with the 8-bit cache; O is in units of V's largest scale over 2^ROW_SHIFT, which
      // is multiplied in last: the smallest scale's unit divided by l would be subnormal
      const float unit = QUANT ? scale_value(scale_max[1]) : 1.f;
      const float inv = (QUANT ? ROW_UNIT : 1.f) * reciprocal_sum(l_run);
      if (part && valid) p.part_ml[(int64_t)split * p.tokens * p.hq + idx] = make_float2(r_run * sl2, l_run);
      constexpr uint32_t GATE = 64u * D;  // 32 rows of the gate
      static_assert(G::NT * 4 * (8192 + GATE) <= M::OFF_RAW, "shared memory of the epilogue");
      const uint32_t stage = base + (uint32_t)warp * (8192u + GATE), gates = stage + 8192u;
      if (gated) {
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {  // D / 8 lanes a row
          const int e = i * 32 + lane, r = e / (D / 8), ch = e % (D / 8);
          const int64_t at = __shfl_sync(0xffffffffu, gate_at, r);
          const uint32_t to = gates + (uint32_t)(r * 2 * D + ((ch ^ (r & 7)) * 16));
          if (live >> r & 1) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(p.gate + at + ch * 8) : "memory");
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
      }
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
          tmem_ld32(tO + c * 64 + h * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint32_t at = stage + (uint32_t)lane * 256u + (uint32_t)(((8 * h + q) ^ (lane & 7)) * 16);
            auto value = [&](int i) { return QUANT ? __uint_as_float(o[i]) * inv * unit : __uint_as_float(o[i]) * inv; };
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "f"(value(4 * q)), "f"(value(4 * q + 1)),
                         "f"(value(4 * q + 2)), "f"(value(4 * q + 3))
                         : "memory");
          }
        }
        asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        __syncwarp();
        auto staged = [&](int r, int chunk) {
          float4 x;
          const uint32_t at = stage + (uint32_t)r * 256u + (uint32_t)((chunk ^ (r & 7)) * 16);
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
          return x;
        };
        if (part) {
#pragma unroll 4
          for (int i = 0; i < 16; ++i) {
            const int r = 2 * i + (lane >> 4);
            const int64_t at = __shfl_sync(0xffffffffu, idx, r);
            const float4 x = staged(r, lane & 15);
            if (live >> r & 1)
              *reinterpret_cast<float4*>(p.part_o + ((int64_t)split * p.tokens * p.hq + at) * D + c * 64 + (lane & 15) * 4) = x;
          }
        } else {
#pragma unroll 1
          for (int i0 = 0; i0 < 8; i0 += 4) {  // four rows a lane: their chains of exponential and quotient overlap
            float4 first[4], second[4];
            uint4 gw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 4 * (i0 + i) + r8;
              // the second half of the lanes reads its chunks in the other order: all eight differ in their bank
              first[i] = staged(r, 2 * c8 + (c8 >> 2));
              second[i] = staged(r, 2 * c8 + 1 - (c8 >> 2));
              if (gated)
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                             : "=r"(gw[i].x), "=r"(gw[i].y), "=r"(gw[i].z), "=r"(gw[i].w)
                             : "r"(gates + (uint32_t)(r * 2 * D + (((c * 8 + c8) ^ (r & 7)) * 16)))
                             : "memory");
            }
            uint4 res[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 lo = c8 < 4 ? first[i] : second[i], hi = c8 < 4 ? second[i] : first[i];
              float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
              if (gated) {
                float gv[8];
                unpack8(gw[i], gv);
#pragma unroll
                for (int u = 0; u < 8; ++u) y[u] *= gate_of(gv[u]);
              }
              res[i] = pack8(y);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 4 * (i0 + i) + r8;
              const int64_t at = __shfl_sync(0xffffffffu, idx, r);
              if (live >> r & 1) *reinterpret_cast<uint4*>(p.out + at * D + c * 64 + c8 * 8) = res[i];
            }
          }
        }
        __syncwarp();
      }
    }
  }
  // ------------------------------------------------------------------ teardown
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == R::MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, TM_COLS);
  }
  if (tid == 0 && *abort_flag) atomicOr(&g_error, 2);
}

using EncodeFn = PFN_cuTensorMapEncodeTiled_v12000;
static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    if (!ok) cudaGetLastError();
    return ok ? reinterpret_cast<EncodeFn>(ptr) : nullptr;
  }();
  return fn;
}

// bf16 with the 128-byte swizzle, or plain bytes
static int encode(CUtensorMap* m, const void* ptr, bool bytes, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box) {
  EncodeFn enc = encode_fn();
  if (!enc) return set_error(FDK_ERR_DEVICE, "paged_gqa: cuTensorMapEncodeTiled unavailable");
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank,
                         const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         bytes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(FDK_ERR_INVALID_ARGUMENT, "paged_gqa: tensor map encode failed (%d)", (int)r);
  return FDK_OK;
}

template <int D, bool QUANT>
static int launch(const Params& p, cudaStream_t s) {
  using G = Geo<D>;
  CUtensorMap mq = {}, mk = {}, mv = {};
  const cuuint64_t esz = QUANT ? 1 : 2, ps = (cuuint64_t)1 << p.page_shift;
  const cuuint64_t kd[4] = {(cuuint64_t)D, ps, (cuuint64_t)p.hkv, (cuuint64_t)p.num_pages};
  const cuuint32_t kb[4] = {QUANT ? (cuuint32_t)D : 64u, (cuuint32_t)(ps < (cuuint64_t)G::BN ? ps : (cuuint64_t)G::BN), 1, 1};
  const cuuint64_t ks[3] = {(cuuint64_t)D * esz, ps * D * esz, (cuuint64_t)p.kpage};
  const cuuint64_t vs[3] = {(cuuint64_t)D * esz, ps * D * esz, (cuuint64_t)p.vpage};
  if (int st = encode(&mk, p.k_cache, QUANT, 4, kd, ks, kb)) return st;
  if (int st = encode(&mv, p.v_cache, QUANT, 4, kd, vs, kb)) return st;
  if (!QUANT && !G::Q_TMEM) {
    const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)p.hq, (cuuint64_t)p.tokens};
    const cuuint64_t qs[2] = {(cuuint64_t)D * 2, (cuuint64_t)p.ld_q * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t)p.group, (cuuint32_t)(128 / p.group)};
    if (int st = encode(&mq, p.q, false, 3, qd, qs, qb)) return st;
  }
  constexpr uint32_t bytes = Smem<D, QUANT>::BYTES;
  const void* fn = (const void*)many_rows_kernel<D, QUANT>;
  if (int st = ensure_smem_attr(fn, (int)bytes, "paged_gqa")) return st;
  const dim3 grid((unsigned)((int64_t)p.units * p.hkv), p.picked ? 1u : (unsigned)p.nsplit);
  many_rows_kernel<D, QUANT><<<grid, Roles<D, QUANT>::THREADS, bytes, s>>>(mq, mk, mv, p);
  return check_launch("paged_gqa (many rows)");
}

}  // namespace chunk
}  // namespace pattn
}  // namespace fdk
