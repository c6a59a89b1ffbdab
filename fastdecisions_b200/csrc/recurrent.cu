// The Gated-DeltaNet mixer continued from cached state, for few tokens a sequence: the recurrent gated
// delta rule over a pool of states, and the packed causal conv + SiLU over a pool of input histories.
//
// Pools: segment s starts from slot state_indices[s] (negative: from zero) and leaves its new state in
// slot final_indices[s] (negative: nowhere).  The two may be the same slot (a sequence that advances) or
// differ (a fork: many segments may start from one slot).  A slot that one segment writes must not be
// read or written by another segment of the same call.
#include <math.h>

#include "paged.cuh"

namespace fdk {
namespace recur {

__device__ int g_state_error = 0;

__device__ __forceinline__ void flag_error() { atomicOr(&g_state_error, 1); }

// A segment's slot in a pool of `slots`: -1 for none; an id outside the pool is treated as none and
// reported.
__device__ __forceinline__ int64_t slot_of(const int32_t* idx, int s, int64_t slots, bool report) {
  const int64_t i = idx ? idx[s] : s;
  if (i >= slots) {
    if (report) flag_error();
    return -1;
  }
  return i < 0 ? -1 : i;
}

// ------------------------------------------------------------------------------------------------
// Recurrent gated delta rule.  Per token, with the state S [dk][dv] (float32) of one head:
//     S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q
// A CTA is one (segment, head).  Columns of S evolve on their own, so each of its 8 warps owns 16 of the 128
// columns and they never exchange state: lane (r, c) = (lane / 4, lane % 4) holds rows 16 r .. 16 r + 15 of
// columns 4 c .. 4 c + 3 in 64 registers, as pairs of rows (one packed operation works on two).
// Segments of up to eight tokens are walked.  The warps first share the work that every column needs: k and q
// normalised to float32, k . q, e^g, beta and v of all tokens go to shared memory.  The token loop then reads only that.
// S^T k and S^T q of the old state are reduced together, as o = e^g S^T q + (k . q) u with q scaled; the
// reduction over r leaves one of the eight sums in each lane (7 shuffles instead of 24).
// The decay is not applied to the registers: they hold S / G with G the product of the decays so far, and
// the update adds k (u / G), one operation an element instead of two.  When G leaves [1e-18, 1e18] it is
// multiplied in and starts over at 1.
// Bound by HBM where states dominate (64 KiB in, 64 KiB out a head and segment: 96 segments of one token forked from
// one state 36 us, 101 MB written), else by the chain of dependent steps of the two CTAs an SM holds: 96 segments
// of 1 to 24 tokens 65 us, issue slots 32% and tensor cores 10% busy.
constexpr int DK = 128, DV = 128, CPW = 16;   // columns a warp
constexpr int WARPS = DV / CPW;
// Segments of at most this many tokens are walked token by token.  Measured, 16 heads, walked / in batches: 96 segments
// of 4 tokens 51 / 70 us, of 8 64 / 71, of 9 71 / 71, of 16 100 / 72; one segment of 4 7.2 / 9.3, of 16 13.7 / 9.3.
constexpr int WALK_MAX = 8;
constexpr int BATCH = 16;                     // tokens of a batch

struct DeltaParams {
  const bf16* q;
  const bf16* k;
  const bf16* v;
  const float* g;
  const bf16* beta;
  int64_t ld_q, ld_k, ld_v;
  const int32_t* cu;
  int64_t period;       // tokens a segment when cu is null
  int64_t tokens;
  int nseg, heads, group;  // group: value heads a key head
  float scale;
  int l2norm;
  const float* state_in;
  const int32_t* in_idx;
  int64_t in_slots;
  float* state_out;
  const int32_t* out_idx;
  int64_t out_slots;
  bf16* out;
};

// k and q of a token are kept in the order the lanes read them: rows 16 r + 4 i .. + 3 at float4 8 i + r, so
// the eight r of a warp read 128 consecutive bytes.
struct Tokens {
  float4 k[WALK_MAX][DK / 4], q[WALK_MAX][DK / 4];
  float v[WALK_MAX][DV];
  float4 s[WALK_MAX];  // e^g, beta, k . q
};

// ---- More than a few tokens: up to 16 at a time on the tensor cores, at float32 accuracy.  With the state S
// before the batch, decays D_ij = e_{j+1} .. e_i (D_i0 from the batch's start) and normalised k, q:
//     u_i = beta_i (v_i - D_i0 S^T k_i - sum_{j < i} D_ij (k_j . k_i) u_j)
//     o_i = D_i0 S^T q_i + sum_{j <= i} D_ij (k_j . q_i) u_j
//     S  <- D_n0 S + sum_j D_nj k_j u_j^T
// so with L_ij = beta_i D_ij (k_j . k_i) (j < i), N_ij = D_ij (k_j . q_i) (j <= i), T = (I + L)^-1 and
// R = beta (v - D_0 S^T k): U = T R, O = D_0 S^T q + N U.  No quotient of decays appears: any of them may be 0.
// The raw k and q are bf16 and go into the products exactly, their norms are applied to the results; float32
// operands (S, R, T, U, N) go in as three bf16 parts (24 bits), products below 2^-24 of the leading one
// left out.
// Warp w keeps S^T for 16 columns of S (dv) as the MMA's accumulators: row g of its tile is column 16 w + 2 g,
// row g + 8 the next one, so that states are read 8 bytes a lane, and accumulators become A operands as they
// are.  A batch costs the same for 2 to 16 tokens.
constexpr int LDV = DV + 4;  // row stride of v: the four token pairs of a warp's read fall into different banks
struct Batch16 {
  uint4 k[BATCH][DK / 8], q[BATCH][DK / 8];  // bf16 rows, 16-byte chunks XORed with the row
  float v[BATCH * LDV];
  float Lt[BATCH][BATCH], N[BATCH][BATCH], T[BATCH][BATCH];  // L transposed
  alignas(16) float e[BATCH];
  float beta[BATCH], rk[BATCH], rq[BATCH], d0[BATCH], dn[BATCH];
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}
// (x, y) as three packed bf16 pairs whose sum has 24 bits
__device__ __forceinline__ void split3(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {
  h = pack_bf16x2(x, y);
  x -= __uint_as_float(h << 16);
  y -= __uint_as_float(h & 0xffff0000u);
  m = pack_bf16x2(x, y);
  x -= __uint_as_float(m << 16);
  y -= __uint_as_float(m & 0xffff0000u);
  l = pack_bf16x2(x, y);
}
// accumulators of two neighbouring 8-column tiles as the A operand of 16 columns, in three parts
__device__ __forceinline__ void split_a(const float (&c0)[4], const float (&c1)[4], uint32_t (&a)[3][4]) {
  split3(c0[0], c0[1], a[0][0], a[1][0], a[2][0]);
  split3(c0[2], c0[3], a[0][1], a[1][1], a[2][1]);
  split3(c1[0], c1[1], a[0][2], a[1][2], a[2][2]);
  split3(c1[2], c1[3], a[0][3], a[1][3], a[2][3]);
}
// c += A X^T for a float32 16 x 16 matrix X in shared memory (both in parts), 16 columns (tokens) of c.  The six
// products go through two accumulators: half the chain of dependent MMAs.
__device__ __forceinline__ void mma_xt(float (&c)[2][4], const uint32_t (&a)[3][4], const float (*X)[BATCH], int g, int t) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const float2 x0 = *reinterpret_cast<const float2*>(&X[8 * n + g][2 * t]);
    const float2 x1 = *reinterpret_cast<const float2*>(&X[8 * n + g][2 * t + 8]);
    uint32_t b[3][2];
    split3(x0.x, x0.y, b[0][0], b[1][0], b[2][0]);
    split3(x1.x, x1.y, b[0][1], b[1][1], b[2][1]);
    float small[4] = {0.f, 0.f, 0.f, 0.f};
    mma_bf16(small, a[2], b[0][0], b[0][1]);
    mma_bf16(c[n], a[1], b[0][0], b[0][1]);
    mma_bf16(small, a[0], b[2][0], b[2][1]);
    mma_bf16(c[n], a[0], b[1][0], b[1][1]);
    mma_bf16(small, a[1], b[1][0], b[1][1]);
    mma_bf16(c[n], a[0], b[0][0], b[0][1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[n][i] += small[i];
  }
}

// Tokens t0 .. t1 - 1 of one (segment, head) by its CTA.
__device__ __forceinline__ void batched_tokens(const DeltaParams& p, Batch16& sm, int64_t t0, int64_t t1, int h, int hk,
                                               int64_t from, int64_t to) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int col = warp * CPW + 2 * g;  // this lane's two columns of S: rows g and g + 8 of its tile
  // S^T: tile j holds rows (dk) 8 j + 2 t, + 1 of S
  float S[DK / 8][4];
  const int64_t head_at = (int64_t)h * (DK * DV) + (int64_t)(2 * t) * DV + col;
  const int64_t pool_ld = (int64_t)p.heads * (DK * DV);
  if (from >= 0) {
    const float* src = p.state_in + from * pool_ld + head_at;
#pragma unroll
    for (int j = 0; j < DK / 8; ++j) {
      const float2 a = *reinterpret_cast<const float2*>(src + 8 * j * DV), b = *reinterpret_cast<const float2*>(src + (8 * j + 1) * DV);
      S[j][0] = a.x; S[j][1] = b.x; S[j][2] = a.y; S[j][3] = b.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < DK / 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[j][i] = 0.f;
  }
  const uint32_t kbase = (uint32_t)__cvta_generic_to_shared(&sm.k[0][0]), qbase = (uint32_t)__cvta_generic_to_shared(&sm.q[0][0]);
  auto at = [](int row, int chunk) { return (uint32_t)((row * (DK / 8) + (chunk ^ (row & 7))) * 16); };
  // a 16-byte chunk of k, q and v a thread, loaded a batch ahead; rows behind the last token are zeros (beta 0,
  // decay 1)
  const int li = tid >> 4, lcn = tid & 15;
  uint4 kr, qr, vr;
  float ge, be;
  auto load_batch = [&](int64_t tb) {
    const bool live = tb + li < t1;
    const int64_t tok = live ? tb + li : t0;
    kr = __ldg(reinterpret_cast<const uint4*>(p.k + tok * p.ld_k + hk * DK) + lcn);
    qr = __ldg(reinterpret_cast<const uint4*>(p.q + tok * p.ld_q + hk * DK) + lcn);
    vr = __ldg(reinterpret_cast<const uint4*>(p.v + tok * p.ld_v + h * DV) + lcn);
    ge = p.g[tok * p.heads + h];
    be = __bfloat162float(p.beta[tok * p.heads + h]);
  };
  load_batch(t0);
  for (int64_t tb = t0; tb < t1; tb += BATCH) {
    const int nt = (int)(t1 - tb < BATCH ? t1 - tb : BATCH);
    if (tb > t0) __syncthreads();
    {
      if (li >= nt) {
        kr = qr = vr = make_uint4(0u, 0u, 0u, 0u);
        ge = be = 0.f;
      }
      if (lcn == 0) {
        sm.e[li] = expf(ge);
        sm.beta[li] = be;
      }
      sm.k[li][lcn ^ (li & 7)] = kr;
      sm.q[li][lcn ^ (li & 7)] = qr;
      float kf[8], qf[8], vf[8], kk = 0.f, qq = 0.f;
      unpack8(kr, kf);
      unpack8(qr, qf);
      unpack8(vr, vf);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        kk = fmaf(kf[u], kf[u], kk);
        qq = fmaf(qf[u], qf[u], qq);
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) {
        kk += __shfl_xor_sync(0xffffffffu, kk, off);
        qq += __shfl_xor_sync(0xffffffffu, qq, off);
      }
      if (lcn == 0) {
        sm.rk[li] = p.l2norm ? rsqrtf(kk + 1e-6f) : 1.f;
        sm.rq[li] = (p.l2norm ? rsqrtf(qq + 1e-6f) : 1.f) * p.scale;
      }
      float* vd = sm.v + li * LDV + 8 * lcn;
      *reinterpret_cast<float4*>(vd) = make_float4(vf[0], vf[1], vf[2], vf[3]);
      *reinterpret_cast<float4*>(vd + 4) = make_float4(vf[4], vf[5], vf[6], vf[7]);
    }
    __syncthreads();
    if (tb + BATCH < t1) load_batch(tb + BATCH);
    if (warp < 4) {  // L (warps 0, 1: eight columns each) and N (2, 3) from the Gram matrices of k and of q with k
      const uint32_t abase = warp < 2 ? kbase : qbase;
      float acc[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DK / 16; kk += 2) {
        uint32_t a0[4], a1[4], b[4];
        ldsm4(a0, abase + at(lane & 15, 2 * kk + (lane >> 4)));
        ldsm4(a1, abase + at(lane & 15, 2 * kk + 2 + (lane >> 4)));
        ldsm4(b, kbase + at(8 * (warp & 1) + (lane & 7), 2 * kk + (lane >> 3)));
        mma_bf16(acc[0], a0, b[0], b[1]);
        mma_bf16(acc[1], a1, b[2], b[3]);
      }
      float e[BATCH];
#pragma unroll
      for (int m = 0; m < BATCH; m += 4) {
        const float4 x = *reinterpret_cast<const float4*>(&sm.e[m]);
        e[m] = x.x; e[m + 1] = x.y; e[m + 2] = x.z; e[m + 3] = x.w;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int i = g + 8 * (c >> 1), j = 8 * (warp & 1) + 2 * t + (c & 1);
        float d = 1.f;
#pragma unroll
        for (int m = 1; m < BATCH; ++m) d *= m > j && m <= i ? e[m] : 1.f;
        const float x = (acc[0][c] + acc[1][c]) * sm.rk[j] * d;
        if (warp < 2) sm.Lt[j][i] = j < i ? x * sm.rk[i] * sm.beta[i] : 0.f;
        else sm.N[i][j] = j <= i ? x * sm.rq[i] : 0.f;
      }
    } else if (warp == 4 && lane < BATCH) {
      float d0 = 1.f, dn = 1.f;
#pragma unroll
      for (int m = 0; m < BATCH; ++m) {
        const float e = sm.e[m];
        d0 *= m <= lane ? e : 1.f;
        dn *= m > lane ? e : 1.f;
      }
      sm.d0[lane] = d0;
      sm.dn[lane] = dn;
    }
    __syncthreads();
    if (warp == 7 && lane < BATCH) {  // T = (I + L)^-1, a column a lane
      float x[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) x[i] = i == lane ? 1.f : 0.f;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        sm.T[i][lane] = x[i];
#pragma unroll
        for (int m = (i + 1) & ~3; m < BATCH; m += 4) {
          const float4 l = *reinterpret_cast<const float4*>(&sm.Lt[i][m]);  // 0 up to the diagonal
          x[m] = fmaf(-l.x, x[i], x[m]);
          x[m + 1] = fmaf(-l.y, x[i], x[m + 1]);
          x[m + 2] = fmaf(-l.z, x[i], x[m + 2]);
          x[m + 3] = fmaf(-l.w, x[i], x[m + 3]);
        }
      }
    }
    // S^T k and S^T q of all tokens
    float pk[2][4], pq[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) pk[n][i] = pq[n][i] = 0.f;
    const int brow = (lane & 7) + ((lane >> 4) << 3), bchunk = (lane >> 3) & 1;
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk) {
      uint32_t a[3][4], bk[4], bq[4];
      split_a(S[2 * kk], S[2 * kk + 1], a);
      ldsm4(bk, kbase + at(brow, 2 * kk + bchunk));
      ldsm4(bq, qbase + at(brow, 2 * kk + bchunk));
#pragma unroll
      for (int u = 2; u >= 0; --u) {
        mma_bf16(pk[0], a[u], bk[0], bk[1]);
        mma_bf16(pq[0], a[u], bq[0], bq[1]);
        mma_bf16(pk[1], a[u], bk[2], bk[3]);
        mma_bf16(pq[1], a[u], bq[2], bq[3]);
      }
    }
    __syncthreads();  // T
    // R, U = T R, O = D_0 S^T q + N U; tokens i = 8 n + 2 t (+ 1) of columns col, col + 1
    float u[2][4], w[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 8 * n + 2 * t + e;
        const float beta = sm.beta[i], d0 = sm.d0[i], dk = d0 * sm.rk[i], dq = d0 * sm.rq[i];
        const float2 v = *reinterpret_cast<const float2*>(sm.v + i * LDV + col);
        w[n][e] = beta * (v.x - dk * pk[n][e]);
        w[n][2 + e] = beta * (v.y - dk * pk[n][2 + e]);
        pq[n][e] *= dq;
        pq[n][2 + e] *= dq;
        u[n][e] = u[n][2 + e] = 0.f;
      }
    uint32_t a[3][4];
    split_a(w[0], w[1], a);
    mma_xt(u, a, sm.T, g, t);
    split_a(u[0], u[1], a);
    mma_xt(pq, a, sm.N, g, t);
#pragma unroll
    for (int n = 0; n < 2; ++n) {  // token 8 n + g, columns 16 w + 4 t .. + 3 after the transpose
      const uint32_t even = transpose8(pack_bf16x2(pq[n][0], pq[n][1])), odd = transpose8(pack_bf16x2(pq[n][2], pq[n][3]));
      if (8 * n + g < nt)
        *reinterpret_cast<uint2*>(p.out + ((tb + 8 * n + g) * p.heads + h) * DV + warp * CPW + 4 * t) =
            make_uint2(__byte_perm(even, odd, 0x5410), __byte_perm(even, odd, 0x7632));
    }
    // S^T <- D_n0 S^T + sum_j (D_nj |k_j| u_j) k_j^T
    const float dall = sm.d0[BATCH - 1];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 8 * n + 2 * t + e;
        const float f = sm.dn[i] * sm.rk[i];
        u[n][e] *= f;
        u[n][2 + e] *= f;
      }
    split_a(u[0], u[1], a);
#pragma unroll
    for (int j = 0; j < DK / 8; j += 2) {
      uint32_t b[4];
      ldsm4t(b, kbase + at(lane & 15, j + (lane >> 4)));
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) S[j + x][i] *= dall;
#pragma unroll
        for (int y = 2; y >= 0; --y) mma_bf16(S[j + x], a[y], b[2 * x], b[2 * x + 1]);
      }
    }
  }
  if (to >= 0) {
    float* dst = p.state_out + to * pool_ld + head_at;
#pragma unroll
    for (int j = 0; j < DK / 8; ++j) {
      *reinterpret_cast<float2*>(dst + 8 * j * DV) = make_float2(S[j][0], S[j][2]);
      *reinterpret_cast<float2*>(dst + (8 * j + 1) * DV) = make_float2(S[j][1], S[j][3]);
    }
  }
}

__global__ void __launch_bounds__(32 * WARPS, 2) recurrent_delta_kernel(const DeltaParams p) {
  __shared__ union { Tokens walk; Batch16 batch; } shared;
  Tokens& sm = shared.walk;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s = (int)(blockIdx.x / (unsigned)p.heads), h = (int)(blockIdx.x % (unsigned)p.heads);
  const bool report = threadIdx.x == 0 && h == 0;
  int64_t t0, t1;
  if (p.cu) {
    int b, e;
    if (!paged::segment_range(p.cu, s, p.tokens, b, e)) {
      if (report) flag_error();
      b = e = 0;
    }
    t0 = b;
    t1 = e;
  } else {
    t0 = s * p.period;
    t1 = t0 + p.period;
  }
  const int r = lane >> 2, c = lane & 3;
  const int col = warp * CPW + c * 4;
  const int hk = h / p.group;
  const int64_t from = p.state_in ? slot_of(p.in_idx, s, p.in_slots, report) : -1;
  const int64_t to = p.state_out ? slot_of(p.out_idx, s, p.out_slots, report) : -1;
  if (t1 - t0 > WALK_MAX) {
    batched_tokens(p, shared.batch, t0, t1, h, hk, from, to);
    return;
  }
  const int64_t in_slot = (int64_t)r * 16 * DV + col;
  float2 S[4][8];  // [column][pair of rows]
  if (from >= 0) {
    const float* src = p.state_in + (from * p.heads + h) * (DK * DV) + in_slot;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float4 a = *reinterpret_cast<const float4*>(src + (2 * i) * DV);
      const float4 b = *reinterpret_cast<const float4*>(src + (2 * i + 1) * DV);
      S[0][i] = make_float2(a.x, b.x);
      S[1][i] = make_float2(a.y, b.y);
      S[2][i] = make_float2(a.z, b.z);
      S[3][i] = make_float2(a.w, b.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[j][i] = make_float2(0.f, 0.f);
  }
  float G = 1.f;
  auto scale_state = [&](float f) {
    const float2 f2 = make_float2(f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[j][i] = __fmul2_rn(S[j][i], f2);
  };
  const int nt = (int)(t1 - t0);
  static_assert(WALK_MAX <= WARPS, "a warp a token");
  if (warp < nt) {
    const int i = warp;
    const int64_t t = t0 + i;
    const uint2 kr = __ldg(reinterpret_cast<const uint2*>(p.k + t * p.ld_k + hk * DK) + lane);
    const uint2 qr = __ldg(reinterpret_cast<const uint2*>(p.q + t * p.ld_q + hk * DK) + lane);
    const uint2 vr = __ldg(reinterpret_cast<const uint2*>(p.v + t * p.ld_v + h * DV) + lane);
    const float g = p.g[t * p.heads + h], beta = __bfloat162float(p.beta[t * p.heads + h]);
    auto two = [](uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w)); };
    float2 k0 = two(kr.x), k1 = two(kr.y), q0 = two(qr.x), q1 = two(qr.y);
    const float2 v0 = two(vr.x), v1 = two(vr.y);
    float rk = 1.f, rq = p.scale;
    if (p.l2norm) {
      rk = rsqrtf(warp_sum(k0.x * k0.x + k0.y * k0.y + k1.x * k1.x + k1.y * k1.y) + 1e-6f);
      rq *= rsqrtf(warp_sum(q0.x * q0.x + q0.y * q0.y + q1.x * q1.x + q1.y * q1.y) + 1e-6f);
    }
    const float4 kn = make_float4(k0.x * rk, k0.y * rk, k1.x * rk, k1.y * rk);
    const float4 qn = make_float4(q0.x * rq, q0.y * rq, q1.x * rq, q1.y * rq);
    const float kq = warp_sum(kn.x * qn.x + kn.y * qn.y + kn.z * qn.z + kn.w * qn.w);
    const int at = (lane & 3) * 8 + (lane >> 2);
    sm.k[i][at] = kn;
    sm.q[i][at] = qn;
    *reinterpret_cast<float4*>(&sm.v[i][4 * lane]) = make_float4(v0.x, v0.y, v1.x, v1.y);
    if (lane == 0) sm.s[i] = make_float4(expf(g), beta, kq, 0.f);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const float4 sc = sm.s[t];
    G *= sc.x;
    if (!(G >= 1e-18f && G <= 1e18f)) {  // the same for the whole CTA
      scale_state(G);
      G = 1.f;
    }
    float2 k[8], dot[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) dot[j] = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 k4 = sm.k[t][i * 8 + r], q4 = sm.q[t][i * 8 + r];
      k[2 * i] = make_float2(k4.x, k4.y);
      k[2 * i + 1] = make_float2(k4.z, k4.w);
      const float2 q0 = make_float2(q4.x, q4.y), q1 = make_float2(q4.z, q4.w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dot[j] = __ffma2_rn(S[j][2 * i], k[2 * i], dot[j]);
        dot[4 + j] = __ffma2_rn(S[j][2 * i], q0, dot[4 + j]);
        dot[j] = __ffma2_rn(S[j][2 * i + 1], k[2 * i + 1], dot[j]);
        dot[4 + j] = __ffma2_rn(S[j][2 * i + 1], q1, dot[4 + j]);
      }
    }
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = dot[j].x + dot[j].y;
    // sum over r: lane r ends with sum r of S^T k (columns 0 .. 3), S^T q (columns 0 .. 3)
#pragma unroll
    for (int n = 4; n > 0; n >>= 1) {
      const bool upper = (r & n) != 0;
#pragma unroll
      for (int j = 0; j < n; ++j) {
        const float mine = upper ? d[n + j] : d[j], other = upper ? d[j] : d[n + j];
        d[j] = mine + __shfl_xor_sync(0xffffffffu, other, 4 * n);
      }
    }
    // lanes r < 4: u of column r; lanes r >= 4 pick it up for their output
    const float gd = G * d[0];
    const float u = sc.y * (sm.v[t][col + (r & 3)] - gd);
    const float uo = __shfl_xor_sync(0xffffffffu, u, 16);
    if (r >= 4) p.out[((t0 + t) * p.heads + h) * DV + col + (r & 3)] = __float2bfloat16_rn(fmaf(sc.z, uo, gd));
    const float ug = __fdividef(u, G);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float uj = __shfl_sync(0xffffffffu, ug, 4 * j + c);
      const float2 uu = make_float2(uj, uj);
#pragma unroll
      for (int i = 0; i < 8; ++i) S[j][i] = __ffma2_rn(k[i], uu, S[j][i]);
    }
  }
  if (to >= 0) {
    if (t0 < t1) scale_state(G);
    float* dst = p.state_out + (to * p.heads + h) * (DK * DV) + in_slot;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      *reinterpret_cast<float4*>(dst + (2 * i) * DV) = make_float4(S[0][i].x, S[1][i].x, S[2][i].x, S[3][i].x);
      *reinterpret_cast<float4*>(dst + (2 * i + 1) * DV) = make_float4(S[0][i].y, S[1][i].y, S[2][i].y, S[3][i].y);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Packed causal conv (width KW <= 4) + SiLU with history.  The rows before a segment are its slot's
// KW - 1 cached input rows; its last KW - 1 rows (of history and input together) are the new ones.
// Two kinds of work in one grid: jobs below nseg are a segment's head -- its first KW - 1 outputs, the
// only ones that read the history, and the new history, so an in-place update cannot race -- and the
// rest take eight consecutive tokens each and compute those at least KW - 1 tokens into their segment.
// Memory-bound in bytes, in time bound by their latency: 96 segments, 3599 tokens of 6144 channels 27 us (3.4 TB/s,
// 40% of the issue slots); more or fewer tokens a job (4, 16) and a forced occupancy were slower.
constexpr int RPT = 8;

struct ConvParams {
  const bf16* x;
  int64_t ld_x;
  const bf16* w;
  const int32_t* cu;
  int64_t period, tokens;
  int nseg, channels, key_dim, cblocks;
  const bf16* hist_in;
  const int32_t* in_idx;
  int64_t in_slots;
  bf16* hist_out;
  const int32_t* out_idx;
  int64_t out_slots;
  bf16* q;
  bf16* k;
  bf16* v;
};

// silu(x) = h + h tanh(h), h = x / 2, of two channels as bf16
__device__ __forceinline__ uint32_t silu2(float2 x) {
  const float2 h = __fmul2_rn(make_float2(0.5f, 0.5f), x);
  const float2 y = __ffma2_rn(h, make_float2(tanh_approx(h.x), tanh_approx(h.y)), h);
  return pack_bf16x2(y.x, y.y);
}

// One output row of 8 channels from its KW input rows, two channels an operation.
template <int KW>
__device__ __forceinline__ void conv_row(const uint4 (&rows)[KW], const float2 (&w)[KW][4], bf16* dst) {
  uint4 out;
  uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      const uint32_t b = c == 0 ? rows[j].x : c == 1 ? rows[j].y : c == 2 ? rows[j].z : rows[j].w;
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&b));
      acc = j == 0 ? __fmul2_rn(w[0][c], x) : __ffma2_rn(w[j][c], x, acc);
    }
    o[c] = silu2(acc);
  }
  *reinterpret_cast<uint4*>(dst) = out;
}

template <int KW>
__global__ void __launch_bounds__(128) conv_state_kernel(const ConvParams p) {
  constexpr int HR = KW - 1;  // history rows
  const int lane = threadIdx.x & 31;
  const int cblk = (int)(blockIdx.x % (unsigned)p.cblocks);
  const int c0 = (cblk * 32 + lane) * 8;
  const bool active = c0 < p.channels;
  const int64_t job = (int64_t)(blockIdx.x / (unsigned)p.cblocks) * 4 + (threadIdx.x >> 5);
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  bf16* dst;
  int64_t ldd;
  if (c0 < p.key_dim) { dst = p.q + c0; ldd = p.key_dim; }
  else if (c0 < 2 * p.key_dim) { dst = p.k + (c0 - p.key_dim); ldd = p.key_dim; }
  else { dst = p.v + (c0 - 2 * p.key_dim); ldd = p.channels - 2 * p.key_dim; }
  auto load_w = [&](float2 (&w)[KW][4]) {  // 8 channels x KW taps: KW aligned 16-byte loads
    float f[8 * KW];
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      float e[8];
      unpack8(__ldg(reinterpret_cast<const uint4*>(p.w + (int64_t)c0 * KW) + i), e);
#pragma unroll
      for (int u = 0; u < 8; ++u) f[8 * i + u] = e[u];
    }
#pragma unroll
    for (int j = 0; j < KW; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) w[j][c] = make_float2(f[2 * c * KW + j], f[(2 * c + 1) * KW + j]);
  };
  if (job < p.nseg) {
    const int s = (int)job;
    int64_t t0, t1;
    if (p.cu) {
      int b, e;
      if (!paged::segment_range(p.cu, s, p.tokens, b, e)) {
        if (lane == 0 && cblk == 0) flag_error();
        b = e = 0;
      }
      t0 = b;
      t1 = e;
    } else {
      t0 = s * p.period;
      t1 = t0 + p.period;
    }
    if (!active) return;
    const bool report = lane == 0 && cblk == 0;
    const int64_t from = p.hist_in ? slot_of(p.in_idx, s, p.in_slots, report) : -1;
    const int64_t to = p.hist_out ? slot_of(p.out_idx, s, p.out_slots, report) : -1;
    const int64_t n = t1 - t0;
    // rows: history, then the first HR inputs
    uint4 rows[2 * HR];
#pragma unroll
    for (int j = 0; j < HR; ++j) {
      rows[j] = from >= 0 ? *reinterpret_cast<const uint4*>(p.hist_in + (from * HR + j) * p.channels + c0) : zero;
      rows[HR + j] = j < n ? ldg_stream(p.x + (t0 + j) * p.ld_x + c0) : zero;
    }
    uint4 last[HR] = {};  // the new history: rows n .. n + HR - 1 of (history, inputs)
#pragma unroll
    for (int j = 0; j < HR; ++j) {
      const int64_t i = n + j;
      if (i >= 2 * HR) {
        last[j] = ldg_stream(p.x + (t0 + i - HR) * p.ld_x + c0);
      } else {
#pragma unroll
        for (int m = 0; m < 2 * HR; ++m)
          if (m == i) last[j] = rows[m];
      }
    }
    if (to >= 0) {
#pragma unroll
      for (int j = 0; j < HR; ++j)
        *reinterpret_cast<uint4*>(p.hist_out + (to * HR + j) * p.channels + c0) = last[j];
    }
    if (n == 0) return;
    float2 w[KW][4];
    load_w(w);
#pragma unroll
    for (int j = 0; j < HR; ++j) {
      if (j >= n) break;
      uint4 win[KW];
#pragma unroll
      for (int m = 0; m < KW; ++m) win[m] = rows[j + m];
      conv_row<KW>(win, w, dst + (t0 + j) * ldd);
    }
    return;
  }
  const int64_t r0 = (job - p.nseg) * RPT;
  if (r0 >= p.tokens) return;
  const int64_t r1 = r0 + RPT < p.tokens ? r0 + RPT : p.tokens;
  uint4 raw[RPT + HR];  // loaded before the segment is looked up: neither needs the other
#pragma unroll
  for (int j = 0; j < RPT + HR; ++j) {
    const int64_t t = r0 - HR + j;
    raw[j] = active && t >= 0 && t < r1 ? ldg_stream(p.x + t * p.ld_x + c0) : zero;
  }
  int s;
  if (p.cu) {
    s = paged::find_segment_warp(p.cu, p.nseg, (int)r0, lane);
    if (s < 0) s = 0;
  } else {
    s = (int)(r0 / p.period);
  }
  if (!active) return;
  // which of the rows are this job's: at least HR tokens into a segment
  uint32_t mine = 0;
  int64_t begin = -1, end = -1;
  for (int64_t t = r0; t < r1;) {
    while (t >= end && s < p.nseg) {  // the segment that holds t (none: behind the last one)
      begin = p.cu ? p.cu[s] : s * p.period;
      end = p.cu ? p.cu[s + 1] : begin + p.period;
      ++s;
    }
    if (t >= end) break;
    const int64_t stop = end < r1 ? end : r1;
    if (begin >= 0 && end <= p.tokens) {
      const int64_t from = begin + HR > t ? begin + HR : t;
      if (from < stop) mine |= ((1u << (stop - from)) - 1u) << (from - r0);
    }
    t = stop;
  }
  if (mine == 0) return;
  float2 w[KW][4];
  load_w(w);
  // the rows go through a window of KW in float32: each is unpacked once, each output formed and stored if
  // it is this job's
  float2 win[KW][4];
  auto unpack = [](const uint4& u, float2 (&f)[4]) {
    const uint32_t b[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int c = 0; c < 4; ++c) f[c] = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&b[c]));
  };
#pragma unroll
  for (int j = 0; j < HR; ++j) unpack(raw[j], win[j]);
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    unpack(raw[i + HR], win[(i + HR) % KW]);
    uint4 out;
    uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float2 acc = __fmul2_rn(w[0][c], win[i % KW][c]);
#pragma unroll
      for (int j = 1; j < KW; ++j) acc = __ffma2_rn(w[j][c], win[(i + j) % KW][c], acc);
      o[c] = silu2(acc);
    }
    if (mine >> i & 1u) *reinterpret_cast<uint4*>(dst + (r0 + i) * ldd) = out;
  }
}

}  // namespace recur

int state_take_device_error() {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, recur::g_state_error, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (h) {
    const int zero = 0;
    cudaMemcpyToSymbol(recur::g_state_error, &zero, sizeof(int));
  }
  return h;
}

}  // namespace fdk

using namespace fdk;

extern "C" int fdk_recurrent_gated_delta_rule_fwd(
    const void* q, int64_t ld_q, const void* k, int64_t ld_k, const void* v, int64_t ld_v, const float* g,
    const void* beta, const int32_t* cu_seqlens, int64_t num_segments, int64_t tokens, int64_t key_heads,
    int64_t heads, int64_t dk, int64_t dv, float scale, int use_qk_l2norm, const float* initial_state,
    const int32_t* state_indices, int64_t initial_slots, float* final_state, const int32_t* final_indices,
    int64_t final_slots, void* out, void* stream) {
  using namespace fdk::recur;
  if (int st = check_device()) return st;
  const char* what = "recurrent_gated_delta_rule";
  if (dk != DK || dv != DV) return set_error(FDK_ERR_UNSUPPORTED, "%s: head dims must be 128", what);
  if (heads < 1 || key_heads < 1 || heads % key_heads || heads > 65535)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: heads must be a multiple of the key heads", what);
  if (num_segments < 1 || num_segments > 0x7ffffffe || tokens < 0 || tokens > 0x7fffffff)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: bad segment count or tokens", what);
  if (!cu_seqlens && tokens % num_segments)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: without cu_seqlens every segment has tokens / num_segments tokens", what);
  if (tokens && (!q || !k || !v || !g || !beta || !out)) return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if ((initial_state && initial_slots < 1) || (final_state && final_slots < 1) ||
      (initial_state && !state_indices && initial_slots < num_segments) ||
      (final_state && !final_indices && final_slots < num_segments))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: fewer state slots than segments", what);
  if (ld_q < key_heads * DK || ld_k < key_heads * DK || ld_v < heads * DV)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: row stride too small", what);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(initial_state) ||
      !aligned16(final_state) || ld_q % 8 || ld_k % 8 || ld_v % 8)
    return set_error(FDK_ERR_ALIGNMENT, "%s: pointers and strides must be 16-byte aligned", what);
  DeltaParams p = {};
  p.q = static_cast<const bf16*>(q); p.k = static_cast<const bf16*>(k); p.v = static_cast<const bf16*>(v);
  p.g = g; p.beta = static_cast<const bf16*>(beta);
  p.ld_q = ld_q; p.ld_k = ld_k; p.ld_v = ld_v;
  p.cu = cu_seqlens; p.period = tokens / num_segments; p.tokens = tokens;
  p.nseg = (int)num_segments; p.heads = (int)heads; p.group = (int)(heads / key_heads);
  p.scale = scale; p.l2norm = use_qk_l2norm;
  p.state_in = initial_state; p.in_idx = state_indices; p.in_slots = initial_slots;
  p.state_out = final_state; p.out_idx = final_indices; p.out_slots = final_slots;
  p.out = static_cast<bf16*>(out);
  if (num_segments * heads > 0x7fffffff) return set_error(FDK_ERR_UNSUPPORTED, "%s: too many segments", what);
  recurrent_delta_kernel<<<(unsigned)(num_segments * heads), 32 * WARPS, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch(what);
}

extern "C" int fdk_packed_conv_state(const void* x, int64_t ld_x, const void* weight, const int32_t* cu_seqlens,
                                     int64_t num_segments, int64_t tokens, int64_t channels, int kernel_width,
                                     int64_t key_dim, int64_t value_dim, const void* history,
                                     const int32_t* state_indices, int64_t history_slots, void* new_history,
                                     const int32_t* final_indices, int64_t new_history_slots, void* q, void* k,
                                     void* v, void* stream) {
  using namespace fdk::recur;
  if (int st = check_device()) return st;
  const char* what = "packed_conv_state";
  if (channels <= 0 || key_dim <= 0 || value_dim <= 0 || channels != 2 * key_dim + value_dim || channels > 0x7fffff00)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: channels=%lld must equal 2*key_dim + value_dim", what, (long long)channels);
  if (kernel_width < 2 || kernel_width > 4)
    return set_error(FDK_ERR_UNSUPPORTED, "%s: kernel_width=%d (2..4 supported)", what, kernel_width);
  if (key_dim % 8 || value_dim % 8) return set_error(FDK_ERR_UNSUPPORTED, "%s: key/value dims must be multiples of 8", what);
  if (num_segments < 1 || num_segments > 0x7ffffffe || tokens < 0 || tokens > 0x7fffffff)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: bad segment count or tokens", what);
  if (!cu_seqlens && tokens % num_segments)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: without cu_seqlens every segment has tokens / num_segments tokens", what);
  if (!weight || (tokens && (!x || !q || !k || !v))) return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if ((history && history_slots < 1) || (new_history && new_history_slots < 1) ||
      (history && !state_indices && history_slots < num_segments) ||
      (new_history && !final_indices && new_history_slots < num_segments))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: fewer history slots than segments", what);
  if (ld_x < channels) return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: ld_x < channels", what);
  if (!aligned16(x) || ld_x % 8 || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(history) ||
      !aligned16(new_history) || !aligned16(weight))
    return set_error(FDK_ERR_ALIGNMENT, "%s: pointers and row stride must be 16-byte aligned", what);
  ConvParams p = {};
  p.x = static_cast<const bf16*>(x); p.ld_x = ld_x; p.w = static_cast<const bf16*>(weight);
  p.cu = cu_seqlens; p.period = tokens / num_segments; p.tokens = tokens;
  p.nseg = (int)num_segments; p.channels = (int)channels; p.key_dim = (int)key_dim;
  p.hist_in = static_cast<const bf16*>(history); p.in_idx = state_indices; p.in_slots = history_slots;
  p.hist_out = static_cast<bf16*>(new_history); p.out_idx = final_indices; p.out_slots = new_history_slots;
  p.q = static_cast<bf16*>(q); p.k = static_cast<bf16*>(k); p.v = static_cast<bf16*>(v);
  const int64_t jobs = num_segments + (tokens + RPT - 1) / RPT;
  const int64_t rows = (jobs + 3) / 4;
  p.cblocks = (int)((channels / 8 + 31) / 32);
  if (rows * p.cblocks > 0x7fffffff) return set_error(FDK_ERR_UNSUPPORTED, "%s: too many tokens", what);
  const unsigned grid = (unsigned)(rows * p.cblocks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (kernel_width) {
    case 4: conv_state_kernel<4><<<grid, 128, 0, s>>>(p); break;
    case 3: conv_state_kernel<3><<<grid, 128, 0, s>>>(p); break;
    default: conv_state_kernel<2><<<grid, 128, 0, s>>>(p); break;
  }
  return check_launch(what);
}
