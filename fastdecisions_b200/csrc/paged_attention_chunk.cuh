// The many-row kernel of paged_attention.cu (included there): tcgen05 tensor cores, TMEM accumulators.
//
// Tensor-core bound: 128 or more rows share every cached row.  Rows are (token, head of the KV head's
// group) pairs, token-major, so one 128-row tile holds 128 / group tokens with all their heads -- no
// padding of short chunks to 128 tokens a head, and K/V are read once a group, not once a head.
//
//   head_dim 128: a CTA owns two 128-row tiles A, B, KV blocks of 128 keys.  Issue order per block j:
//     PV_A(j), S_A(j+1), PV_B(j), S_B(j+1): the softmax of one tile overlaps the MMAs of the other.
//     TMEM: S_A [0,128) S_B [128,256) O_A [256,384) O_B [384,512).
//   head_dim 256: one tile (two would not fit TMEM), KV blocks of 64 keys, S ping-pong one block ahead.
//     TMEM: S0 [0,64) S1 [64,128) O [256,512).
//   P overwrites S in TMEM (A operand of the PV MMA).  Softmax: thread = row = TMEM lane, online in the
//   exp2 domain, O rescaled only when the running maximum grows by more than 2^8.
//
//   bf16 cache: one warp issues TMA loads, a box a page (or 128 / 64 keys of it) and 64 columns; a page id
//   outside the cache is an out-of-range coordinate, which TMA fills with zeros.  V rows at or behind
//   kv_lens[s] may hold anything (0 * NaN would reach the sums): the block that has them is zeroed there
//   after its load and before the MMA warp sees it.
//   8-bit cache: TMA brings the raw e4m3 rows; four converter warps turn them into fp16 operands (e4m3 ->
//   fp16 is exact) multiplied by the row's scale relative to the largest one of the CTA's key range
//   (exact for scales within 2^15 of it; smaller ones lose bits below 2^-33 of the range's largest
//   element).  The largest K scale then folds into the softmax scale, V's into the final normalisation,
//   so the softmax costs what it does for bf16.  q goes to fp16 with a power of two a row.
//
//   K and V blocks share one ring of operand slots, in the order K_0 V_0 K_1 V_1 ..: four slots for bf16,
//   three for the 8-bit cache (PV of block j and S of block j + 1 hold two, the converters fill the
//   third), which leaves room for a ring of four raw tiles.
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
  static constexpr uint32_t TM_S(int i) { return (uint32_t)(BN * i); }         // tile i, or ping-pong buffer i
  static constexpr uint32_t TM_O(int i) { return 256u + 128u * (uint32_t)i; }  // tile i
};
// Shared memory: Q tiles, operand ring, raw ring (8-bit cache), barriers and small state.
// barriers: F / E operand slot full / empty, RF / RE raw slot full / empty, S and P per tile or buffer;
// VT: V of the block that ends past kv_lens, before its tail is zeroed
enum { B_Q = 0, B_F, B_E = B_F + 4, B_RF = B_E + 4, B_RE = B_RF + 4, B_S = B_RE + 4, B_P = B_S + 2, B_VT = B_P + 2,
       B_PV, B_O, NBAR };
constexpr int RAW_SLOTS = 4;
template <int D, bool QUANT>
struct Smem {
  using G = Geo<D>;
  static constexpr int SLOTS = QUANT ? 3 : 4;
  static constexpr uint32_t RAWT = QUANT ? (uint32_t)(G::BN * D) : 0;  // bytes of a raw tile
  static constexpr uint32_t OFF_Q = 0, OFF_KV = G::NT * G::QT, OFF_RAW = OFF_KV + SLOTS * G::KT,
                            OFF_BAR = OFF_RAW + RAW_SLOTS * RAWT, OFF_MISC = OFF_BAR + 8 * NBAR,
                            OFF_QS = OFF_MISC + 64,                       // row scale exponents of q: 256 bytes
                            OFF_FT = OFF_QS + (QUANT ? 256 : 0),          // row factors of two tiles: half2
                            BYTES = OFF_FT + (QUANT ? 1024 : 0) + 1024;   // + slack for 1024-byte alignment
  static_assert(OFF_MISC % 16 == 0, "alignment of the small state");
  static_assert(BYTES <= 232448, "shared memory of a CTA");
};
constexpr uint32_t TM_COLS = 512;
constexpr float P_SHIFT = 6.f;  // fp16 P is scaled by 2^6: weights down to 2^-30 of the row's largest stay
constexpr long long DRAIN_BUDGET = 2000000000LL;

// warps: NT * 4 softmax, one producer, one MMA issuer and TMEM allocator; with the 8-bit cache four
// converter warps on a warpgroup boundary
template <int D, bool QUANT>
struct Roles {
  static constexpr int PRODUCER = Geo<D>::NT * 4, MMA = PRODUCER + 1, CONV = PRODUCER + 4;
  static constexpr int THREADS = QUANT ? (CONV + 4) * 32 : (MMA + 1) * 32;
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
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

// 16-byte chunk c (8 columns) of row r in a [boxes of 64 columns][rows][128 B] operand tile, 128-byte swizzle
template <uint32_t BOX>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)(c >> 3) * BOX + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) * 16);
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
  int* warp_max = reinterpret_cast<int*>(gbase + M::OFF_MISC + 16);                    // [4][2]
  uint8_t* q_exp = gbase + M::OFF_QS;
  uint32_t* factor = reinterpret_cast<uint32_t*>(gbase + M::OFF_FT);                   // [2][BN] half2

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // grid: x = (segment, KV head) with the head fastest, y = row tile from the last one down (the longest
  // key ranges first), z = split of the keys
  const int s = (int)(blockIdx.x / (unsigned)p.hkv), hk = (int)(blockIdx.x % (unsigned)p.hkv);
  const int rb = (int)gridDim.y - 1 - (int)blockIdx.y;
  const int split = (int)blockIdx.z;
  const bool first = hk == 0 && rb == 0 && split == 0;
  const Seg seg = segment(p, s, tid == 0 && first);
  const int tpt = 128 / p.group;                 // tokens a tile
  const int rpt = tpt * p.group;                 // rows of it in use
  const int rows = seg.n * p.group;
  const int tok0 = rb * NT * tpt;                // first token of the CTA
  if (tid == 0 && first && seg.n > (int)gridDim.y * NT * tpt) atomicOr(&g_error, 1);
  if (tok0 >= seg.n) return;
  const int last_tok = min(tok0 + NT * tpt, seg.n) - 1;
  const int64_t kend64 = seg.past + last_tok + 1;
  const int kend = kend64 > 0 ? (int)kend64 : 0;
  const int kv_len = (int)(seg.past + seg.n);
  const int per = ((kend + p.nsplit * BN - 1) / (p.nsplit * BN)) * BN;
  const int kb = min(kend, split * per), ke = min(kend, kb + per);
  const int n_kv = (ke - kb + BN - 1) / BN;
  if (n_kv == 0) {  // nothing to see: zeros, or an empty part
    for (int e = tid; e < NT * rpt; e += R::THREADS) {
      const int64_t gr = (int64_t)tok0 * p.group + e;
      if (gr >= rows) break;
      const int64_t idx = (seg.begin + gr / p.group) * p.hq + hk * p.group + gr % p.group;
      if (p.nsplit > 1) {
        p.part_ml[(int64_t)split * p.tokens * p.hq + idx] = make_float2(-INFINITY, 0.f);
      } else {
        for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(p.out + idx * D + c) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    return;
  }
  // the second tile may have no rows: its MMAs are skipped
  const bool two = NT == 2 && tok0 + tpt < seg.n;

  if (tid == 0) {
    for (int i = 0; i < NBAR; ++i) {
      uint32_t count = 1;
      if (i == B_P || i == B_P + 1) count = 128;
      if (QUANT && (i == B_Q || (i >= B_F && i < B_F + 4) || (i >= B_RE && i < B_RE + 4))) count = 128;
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
    // a block's boxes: keys in pages of 2^page_shift, at most BN a box; lane i issues box i, i + 32, ..
    const int box_keys = min(BN, 1 << p.page_shift);
    constexpr int COLS = QUANT ? 1 : NBX;  // boxes across a row: the raw row, or 64 bf16 columns each
    const int boxes = (BN / box_keys) * COLS;
    if (lane == 0) {
      prefetch_tmap(&tk);
      prefetch_tmap(&tv);
      if (!QUANT) {
        const int tiles = two ? 2 : 1;
        mbar_expect_tx(bar(B_Q), (uint32_t)(tiles * NBX) * 128u * (uint32_t)rpt);
        for (int i = 0; i < tiles; ++i)
          for (int b = 0; b < NBX; ++b)
            tma_load_3d(base + M::OFF_Q + i * G::QT + b * G::QBOX, &tq, bar(B_Q), b * 64, hk * p.group,
                        seg.begin + tok0 + i * tpt);
      }
    }
    int issued = 0;
    for (int i = 0; i < 2 * n_kv; ++i) {
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
      for (int b = lane; b < boxes; b += 32) {
        const int sub = b / COLS, col = b % COLS;
        const int key = key0 + sub * box_keys;
        int page = (int)p.num_pages;  // out of range: zeros
        if (key < ke) {
          const int id = __ldg(table + (key >> p.page_shift));
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
      if (!QUANT) drain(bar(B_Q), 0);
      for (int i = (issued > RING ? issued - RING : 0); i < issued; ++i) drain(bar(FULL + i % RING), (uint32_t)(i / RING) & 1u);
    }
  };

  if (warp == R::PRODUCER && !R::SPLIT_REGS) {
    producer();
  } else if (QUANT ? warp >= R::PRODUCER && warp < R::CONV : warp == R::MMA) {
    // With the 8-bit cache at head_dim 128, 512 threads are launched with 128 registers each; the softmax
    // needs more (a row of S and of P), the other warpgroups less: 256 * 192 + 128 * (40 + 88) = 65536.
    if constexpr (R::SPLIT_REGS) {
      reg_dec<40>();
      if (warp == R::PRODUCER) producer();
    }
    // ------------------------------------------------------------------ MMA issuer
    if (warp == R::MMA && lane == 0) {
      constexpr uint32_t ID_QK = idesc(128, BN, false, QUANT);
      constexpr uint32_t ID_PV = idesc(128, D, true, QUANT);  // V is MN-major (columns contiguous)
      auto issue_s = [&](int j, int tile, uint32_t tm) {
        const uint64_t dq = sdesc_sw128(base + M::OFF_Q + tile * G::QT, 16, 1024);
        const uint64_t dk = sdesc_sw128(base + M::OFF_KV + (2 * j % M::SLOTS) * G::KT, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t qo = ((kk >> 2) * G::QBOX + (kk & 3) * 32) >> 4, ko = ((kk >> 2) * G::KBOX + (kk & 3) * 32) >> 4;
          umma_ss(tmem + tm, dq + qo, dk + ko, ID_QK, kk > 0);
        }
      };
      auto issue_pv = [&](int j, uint32_t tm_p, uint32_t tm_o) {
        const uint64_t dv = sdesc_sw128(base + M::OFF_KV + ((2 * j + 1) % M::SLOTS) * G::KT, G::KBOX, 1024);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
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
          issue_pv(j, G::TM_S(0), G::TM_O(0));
          if (more) {
            if (!full(2 * j + 2)) break;
            tc_fence_after();
            issue_s(j + 1, 0, G::TM_S(0));
            umma_commit(bar(B_S));
          }
          if (two) {
            if (!wait(B_P + 1, j)) break;
            tc_fence_after();
            issue_pv(j, G::TM_S(1), G::TM_O(1));
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
          issue_pv(j, G::TM_S(j & 1), G::TM_O(0));
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
  } else if (QUANT && warp >= R::CONV) {
    // ------------------------------------------------------------------ converters (128 threads)
    if constexpr (R::SPLIT_REGS) reg_dec<88>();
    const int ct = tid - R::CONV * 32, cw = ct >> 5;
    auto slot_of = [&](int key) { return (hk << p.page_shift) + (key & page_mask); };
    // largest scale bytes of the range, 16 keys a load
    uint32_t mk = 0, mv = 0;
    for (int key = kb + ct * 16; key < ke; key += 128 * 16) {
      const int64_t id = __ldg(table + (key >> p.page_shift));
      if (id < 0 || id >= p.num_pages) continue;  // reported by the loads below
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(p.k_scale + id * p.kscale_page + slot_of(key)));
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(p.v_scale + id * p.vscale_page + slot_of(key)));
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int left = ke - (key + 4 * i);  // bytes of this word inside the range
        const uint32_t mask = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        mk = __vmaxu4(mk, aw[i] & mask);
        mv = __vmaxu4(mv, bw[i] & mask);
      }
    }
    auto byte_max = [](uint32_t w) { return max(max(w & 255u, (w >> 8) & 255u), max((w >> 16) & 255u, w >> 24)); };
    mk = __reduce_max_sync(0xffffffffu, byte_max(mk));
    mv = __reduce_max_sync(0xffffffffu, byte_max(mv));
    if (lane == 0) {
      warp_max[2 * cw] = (int)mk;
      warp_max[2 * cw + 1] = (int)mv;
    }
    asm volatile("bar.sync 1, 128;\n" ::: "memory");
    int ek = 0, ev = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ek = max(ek, warp_max[2 * i]);
      ev = max(ev, warp_max[2 * i + 1]);
    }
    if (ct == 0) {
      scale_max[0] = ek;
      scale_max[1] = ev;
    }
    // q: a row a thread, fp16 with its largest magnitude in [1, 2)
    for (int i = 0; i < (two ? 2 : 1); ++i) {
      const int tok = tok0 + i * tpt + ct / p.group;
      const bool live = ct < rpt && tok < seg.n;
      const bf16* src = p.q + (int64_t)(seg.begin + (live ? tok : 0)) * p.ld_q + (int64_t)(hk * p.group + (live ? ct % p.group : 0)) * D;
      float a = 0.f;
      for (int c = 0; c < D / 8; ++c) {
        float f[8];
        unpack8(live ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u), f);
#pragma unroll
        for (int u = 0; u < 8; ++u) a = fmaxf(a, fabsf(f[u]));
      }
      const int e = a == 0.f ? 127 : min(max((int)(__float_as_uint(a) >> 23), 1), 253);
      const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
      q_exp[i * 128 + ct] = (uint8_t)e;  // q's row is fp16 * 2^(e - 127)
      for (int c = 0; c < D / 8; ++c) {
        float f[8];
        unpack8(live ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u), f);
        const uint4 h = make_uint4(pack_f16x2(f[0] * inv, f[1] * inv), pack_f16x2(f[2] * inv, f[3] * inv),
                                   pack_f16x2(f[4] * inv, f[5] * inv), pack_f16x2(f[6] * inv, f[7] * inv));
        *reinterpret_cast<uint4*>(gbase + M::OFF_Q + i * G::QT + chunk_at<G::QBOX>(ct, c)) = h;
      }
    }
    fence_proxy_async_smem();
    mbar_arrive(bar(B_Q));
    // Items: thread ct is row ct's keeper (its scale byte, loaded a block ahead) and, for the conversion,
    // piece lc (8 columns) of rows lr, lr + RPP, ..: 8 raw bytes become one 16-byte operand chunk.  Eight
    // neighbouring threads read 64 consecutive bytes and store all eight chunk positions: no conflicts.
    constexpr int TPR = D / 8, RPP = 128 / TPR, PASSES = BN / RPP;
    const int lc = ct % TPR, lr = ct / TPR;
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
    // once a wait has run out, a thread only keeps step at the named barrier (the others may be behind it)
    bool ok = true;
    for (int j = 0; j < n_kv; ++j) {
      const int key0 = kb + j * BN;
      const uint32_t fk = half2_bits(scale_value(max(kbyte - ek + 127, 0))), fv = half2_bits(scale_value(max(vbyte - ev + 127, 0)));
      // rows behind the range may hold anything, NaN included: their operands are zeros, not 0 * NaN
      const int live = ke - key0;
      kbyte = scale_at(p.k_scale, p.kscale_page, key0 + BN + my, id);
      vbyte = scale_at(p.v_scale, p.vscale_page, key0 + BN + my, id);
      id = page_at(key0 + 2 * BN + my);
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {
        const int item = 2 * j + which, raw_slot = item % RAW_SLOTS, slot = item % M::SLOTS;
        if (ct < BN) factor[which * BN + ct] = which ? fv : fk;
        asm volatile("bar.sync 1, 128;\n" ::: "memory");  // factors written; also: nobody still reads the other table
        ok = ok && mbar_wait(bar(B_RF + raw_slot), (uint32_t)(item / RAW_SLOTS) & 1u, abort_flag) &&
             (item < M::SLOTS || mbar_wait(bar(B_E + slot), (uint32_t)(item / M::SLOTS - 1) & 1u, abort_flag));
        if (!ok) continue;
        const uint8_t* src = gbase + M::OFF_RAW + raw_slot * M::RAWT + lr * D + lc * 8;
        uint8_t* dst = gbase + M::OFF_KV + slot * G::KT;
        const uint32_t* fac = factor + which * BN + lr;
        auto convert = [&](bool partial) {
#pragma unroll
          for (int i = 0; i < PASSES; ++i) {
            uint2 w = *reinterpret_cast<const uint2*>(src + i * RPP * D);
            if (partial && lr + i * RPP >= live) w = make_uint2(0u, 0u);
            const uint32_t f = fac[i * RPP];
            uint4 h;
            h.x = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)w.x), f);
            h.y = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)(w.x >> 16)), f);
            h.z = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)w.y), f);
            h.w = hmul2_bits(paged::e4m3x2_to_f16x2((uint16_t)(w.y >> 16)), f);
            *reinterpret_cast<uint4*>(dst + chunk_at<G::KBOX>(lr + i * RPP, lc)) = h;
          }
        };
        if (live >= BN) convert(false);
        else convert(true);
        fence_proxy_async_smem();
        mbar_arrive(bar(B_F + slot));
        mbar_arrive(bar(B_RE + raw_slot));
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
    if (QUANT && ok) {
      ok = __all_sync(0xffffffffu, mbar_wait(bar(B_Q), 0, abort_flag) ? 1 : 0);
      // never 0: a masked score is -inf * sl2
      if (ok) sl2 = fmaxf(sl2 * scale_value(q_exp[tile * 128 + row]) * scale_value(scale_max[0]), 1e-37f);
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
      for (int a = 0; a < 8; ++a) mx8[a] = -INFINITY;
#pragma unroll
      for (int c = 0; c < BN / 32; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) mx8[i & 7] = fmaxf(mx8[i & 7], __uint_as_float(sr[c][i]));
      const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                             fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
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
      float sum8[8];
#pragma unroll
      for (int a = 0; a < 8; ++a) sum8[a] = 0.f;
      uint32_t pk[BN / 64][32];
      auto weights = [&](auto expo) {
#pragma unroll
        for (int c = 0; c < BN / 2; ++c) {
          const float e0 = ex2(expo(__uint_as_float(sr[(2 * c) >> 5][(2 * c) & 31])));
          const float e1 = ex2(expo(__uint_as_float(sr[(2 * c + 1) >> 5][(2 * c + 1) & 31])));
          sum8[(2 * c) & 7] += e0;
          sum8[(2 * c + 1) & 7] += e1;
          pk[c >> 5][c & 31] = QUANT ? pack_f16x2(e0, e1) : pack_bf16x2(e0, e1);
        }
      };
      // s * sl2 - shift in one operation, unless scores are so large that shift's own rounding (float32
      // spacing 0.25 and more) would show in the exponent
      if (!__any_sync(0xffffffffu, fabsf(shift) > 2097152.f))
        weights([&](float x) { return fmaf(x, sl2, -shift); });
      else
        weights([&](float x) { return fmaf(x - r0, sl2, QUANT ? P_SHIFT : 0.f); });
#pragma unroll
      for (int c = 0; c < BN / 64; ++c) tmem_st32(tS + c * 32, pk[c]);
      const float sum = ((sum8[0] + sum8[1]) + (sum8[2] + sum8[3])) + ((sum8[4] + sum8[5]) + (sum8[6] + sum8[7]));
      l_run = l_run * alpha + sum;
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
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(bar(B_P + buf));
    }
    // ------------------------------------------------------------------ epilogue
    if (ok && __all_sync(0xffffffffu, mbar_wait(bar(B_O), 0, abort_flag) ? 1 : 0)) {
      tc_fence_after();
      const int64_t tk_ = (int64_t)seg.begin + tok;
      const int head = hk * p.group + row % p.group;
      const int64_t idx = tk_ * p.hq + head;
      // l and O both carry 2^P_SHIFT with the 8-bit cache; O is in units of V's largest scale
      const float unit = QUANT ? scale_value(scale_max[1]) : 1.f;
      const float inv = p.nsplit > 1 ? unit : (l_run > 0.f ? unit / l_run : (l_run == 0.f ? 0.f : l_run));
      const bool part = p.nsplit > 1;
      float* prow = part ? p.part_o + ((int64_t)split * p.tokens * p.hq + idx) * D : nullptr;
      if (part && valid) p.part_ml[(int64_t)split * p.tokens * p.hq + idx] = make_float2(r_run * sl2, l_run);
      bf16* orow = p.out + idx * D;
      const bf16* grow = p.gate ? p.gate + tk_ * p.ld_gate + (int64_t)head * p.gate_hstride : nullptr;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_ld_wait();
        if (valid && part) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            *reinterpret_cast<float4*>(prow + c * 32 + i) =
                make_float4(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv, __uint_as_float(o[i + 2]) * inv,
                            __uint_as_float(o[i + 3]) * inv);
        } else if (valid) {
#pragma unroll
          for (int v8 = 0; v8 < 4; ++v8) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(o[v8 * 8 + i]) * inv;
            if (grow) {
              float gv[8];
              unpack8(*reinterpret_cast<const uint4*>(grow + c * 32 + v8 * 8), gv);
#pragma unroll
              for (int i = 0; i < 8; ++i) y[i] *= sigmoidf_(gv[i]);
            }
            *reinterpret_cast<uint4*>(orow + c * 32 + v8 * 8) = pack8(y);
          }
        }
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
static int launch(const Params& p, int64_t row_tiles, cudaStream_t s) {
  using G = Geo<D>;
  CUtensorMap mq = {}, mk = {}, mv = {};
  const cuuint64_t esz = QUANT ? 1 : 2, ps = (cuuint64_t)1 << p.page_shift;
  const cuuint64_t kd[4] = {(cuuint64_t)D, ps, (cuuint64_t)p.hkv, (cuuint64_t)p.num_pages};
  const cuuint32_t kb[4] = {QUANT ? (cuuint32_t)D : 64u, (cuuint32_t)(ps < (cuuint64_t)G::BN ? ps : (cuuint64_t)G::BN), 1, 1};
  const cuuint64_t ks[3] = {(cuuint64_t)D * esz, ps * D * esz, (cuuint64_t)p.kpage};
  const cuuint64_t vs[3] = {(cuuint64_t)D * esz, ps * D * esz, (cuuint64_t)p.vpage};
  if (int st = encode(&mk, p.k_cache, QUANT, 4, kd, ks, kb)) return st;
  if (int st = encode(&mv, p.v_cache, QUANT, 4, kd, vs, kb)) return st;
  if (!QUANT) {
    const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)p.hq, (cuuint64_t)p.tokens};
    const cuuint64_t qs[2] = {(cuuint64_t)D * 2, (cuuint64_t)p.ld_q * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t)p.group, (cuuint32_t)(128 / p.group)};
    if (int st = encode(&mq, p.q, false, 3, qd, qs, qb)) return st;
  }
  constexpr uint32_t bytes = Smem<D, QUANT>::BYTES;
  const void* fn = (const void*)many_rows_kernel<D, QUANT>;
  if (int st = ensure_smem_attr(fn, (int)bytes, "paged_gqa")) return st;
  const dim3 grid((unsigned)((int64_t)p.nseg * p.hkv), (unsigned)row_tiles, (unsigned)p.nsplit);
  many_rows_kernel<D, QUANT><<<grid, Roles<D, QUANT>::THREADS, bytes, s>>>(mq, mk, mv, p);
  return check_launch("paged_gqa (many rows)");
}

}  // namespace chunk
}  // namespace pattn
}  // namespace fdk
