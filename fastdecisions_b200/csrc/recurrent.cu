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
// Up to 16 tokens at a time, the warps first share the work that every column needs: k and q normalised to
// float32, k . q, e^g, beta and v go to shared memory.  The token loop then reads only that.
// S^T k and S^T q of the old state are reduced together, as o = e^g S^T q + (k . q) u with q scaled; the
// reduction over r leaves one of the eight sums in each lane (7 shuffles instead of 24).
// The decay is not applied to the registers: they hold S / G with G the product of the decays so far, and
// the update adds k (u / G), one operation an element instead of two.  When G leaves [1e-18, 1e18] it is
// multiplied in and starts over at 1.
// Bound by HBM where states dominate (64 KiB in, 64 KiB out a head and segment), by the float32 pipe at
// several tokens a segment.
constexpr int DK = 128, DV = 128, CPW = 16;   // columns a warp
constexpr int WARPS = DV / CPW;
constexpr int BATCH = 16;                     // tokens in shared memory at a time

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
  float4 k[BATCH][DK / 4], q[BATCH][DK / 4];
  float v[BATCH][DV];
  float4 s[BATCH];  // e^g, beta, k . q
};

__global__ void __launch_bounds__(32 * WARPS, 2) recurrent_delta_kernel(const DeltaParams p) {
  __shared__ Tokens sm;
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
  for (int64_t tb = t0; tb < t1; tb += BATCH) {
    const int nt = (int)(t1 - tb < BATCH ? t1 - tb : BATCH);
    if (tb > t0) __syncthreads();
    for (int i = warp; i < nt; i += WARPS) {
      const int64_t t = tb + i;
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
      if (r >= 4) p.out[((tb + t) * p.heads + h) * DV + col + (r & 3)] = __float2bfloat16_rn(fmaf(sc.z, uo, gd));
      const float ug = __fdividef(u, G);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float uj = __shfl_sync(0xffffffffu, ug, 4 * j + c);
        const float2 uu = make_float2(uj, uj);
#pragma unroll
        for (int i = 0; i < 8; ++i) S[j][i] = __ffma2_rn(k[i], uu, S[j][i]);
      }
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
