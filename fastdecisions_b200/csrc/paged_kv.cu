// Writing the newest keys and values of packed sequences into a paged KV cache (bf16, or quantised to
// e4m3 with a power-of-two scale per row) and reading cached rows back as packed bf16.
//
// Segment s's tokens cu[s] .. cu[s + 1] - 1 are the last of its kv_lens[s] positions: token t sits at
// position kv_lens[s] - (cu[s + 1] - t), in page page_table[s][position / page_size].
// Both directions move every row once and compute next to nothing: HBM-bound (latency-bound for a
// decoding step's few rows).  A warp owns a token and has four rows' loads in flight.  Measured, e4m3: 55899 cached
// positions of 2 heads of 256 read back in 32.5 us (5.3 TB/s); 34198 tokens of 4 heads of 128 written and read back
// in 40.6 us (5.2 TB/s; 55 with one row in flight, 46 with every address worked out in full); 64 tokens written and
// read back 6.2 us with both launches.
#include "paged.cuh"

namespace fdk {
namespace paged {

__device__ int g_kv_error = 0;

struct KvParams {
  const bf16* k;  // rows of the caller (read by write, written by read)
  const bf16* v;
  bf16* k_out;
  bf16* v_out;
  int64_t ld_k, ld_v;
  void* k_cache;
  void* v_cache;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t ld_kpage, ld_vpage;            // elements between pages
  int64_t ld_kscale_page, ld_vscale_page;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* cu;
  const int32_t* kv_lens;
  int64_t tokens, num_pages;
  int nseg, max_pages, page_shift, hkv;
};

// Row of token t: page and offset in it.  Warp-uniform.
//   FOUND  the row is cache row `off` of `page`
//   NONE   the token belongs to a segment but has no cached row: more new tokens than positions, or
//          (error word set) an invalid length or page id.  A write skips it, a read gives zeros.
//   OUTSIDE  behind the last segment (or cu_seqlens is invalid there: error word set): left alone
enum Where { FOUND, NONE, OUTSIDE };
__device__ __forceinline__ Where locate(const KvParams& p, int64_t t, int lane, int64_t& page, int& off) {
  const int s = find_segment_warp(p.cu, p.nseg, (int)t, lane);
  if (s >= p.nseg) return OUTSIDE;
  const int end = s < 0 ? 0 : p.cu[s + 1];
  if (s < 0 || end <= t || end > p.tokens) {
    if (lane == 0) atomicOr(&g_kv_error, 1);
    return OUTSIDE;
  }
  const int64_t len = p.kv_lens[s];
  if (len < 0 || len > ((int64_t)p.max_pages << p.page_shift)) {
    if (lane == 0) atomicOr(&g_kv_error, 1);
    return NONE;
  }
  const int64_t pos = len - (end - t);
  if (pos < 0) return NONE;
  page = p.table[s * p.ld_table + (pos >> p.page_shift)];
  off = (int)(pos & ((1 << p.page_shift) - 1));
  if (page < 0 || page >= p.num_pages) {
    if (lane == 0) atomicOr(&g_kv_error, 1);
    return NONE;
  }
  return FOUND;
}

// One warp a token: D / 8 lanes a row, so two rows (D = 128) or one (D = 256) at a time over the
// 2 * hkv rows (k then v), up to four of those in flight.  READ = false: rows into the cache (loaded
// before the token's place is looked up); READ = true: cached rows out.
template <int D, bool QUANT, bool READ>
__global__ void __launch_bounds__(128) kv_rows_kernel(const KvParams p) {
  constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes a row, rows an iteration
  constexpr int BATCH = 4;
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int sub = lane / LPR, c = (lane % LPR) * 8;
  const int rows = 2 * p.hkv;
  // Issue slots bound the large calls, so every address is a base of the token, chosen once a row, plus the head's
  // 32-bit offset.
  auto pick = [&](bool is_v, auto* k, auto* v) { return is_v ? v : k; };
  uint4 raw[BATCH];
  auto load_new = [&](int r0) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int r = min(r0 + i * RPI + sub, rows - 1);
      const bool is_v = r >= p.hkv;
      raw[i] = ldg_stream(pick(is_v, p.k + t * p.ld_k + c, p.v + t * p.ld_v + c) + (is_v ? r - p.hkv : r) * D);
    }
  };
  if (!READ) load_new(0);
  int64_t page = 0;
  int off = 0;
  const Where where = locate(p, t, lane, page, off);
  if (where == OUTSIDE || (!READ && where == NONE)) return;
  // `page` and `off` are 0 where there is no row: a valid place
  constexpr int ESZ = QUANT ? 1 : 2;
  uint8_t* const k_at = static_cast<uint8_t*>(p.k_cache) + (page * p.ld_kpage + off * D + c) * ESZ;
  uint8_t* const v_at = static_cast<uint8_t*>(p.v_cache) + (page * p.ld_vpage + off * D + c) * ESZ;
  uint8_t* const ks_at = QUANT ? p.k_scale + page * p.ld_kscale_page + off : nullptr;
  uint8_t* const vs_at = QUANT ? p.v_scale + page * p.ld_vscale_page + off : nullptr;
  for (int r0 = 0; r0 < rows; r0 += BATCH * RPI) {
    if (READ) {
      int bytes[BATCH];
      uint2 q8[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = min(r0 + i * RPI + sub, rows - 1);
        const bool is_v = r >= p.hkv;
        const int slot = (is_v ? r - p.hkv : r) << p.page_shift;
        const uint8_t* src = pick(is_v, k_at, v_at) + slot * (D * ESZ);
        if (QUANT) {
          q8[i] = __ldg(reinterpret_cast<const uint2*>(src));
          bytes[i] = __ldg(pick(is_v, ks_at, vs_at) + slot);
        } else {
          raw[i] = ldg_stream(reinterpret_cast<const bf16*>(src));
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = r0 + i * RPI + sub;
        const bool is_v = r >= p.hkv;
        if (QUANT) {
          const float s = scale_value(bytes[i]);
          const uint16_t q[4] = {(uint16_t)q8[i].x, (uint16_t)(q8[i].x >> 16), (uint16_t)q8[i].y, (uint16_t)(q8[i].y >> 16)};
          float f[8];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t h2 = e4m3x2_to_f16x2(q[u]);
            const float2 w = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&h2)), make_float2(s, s));
            f[2 * u] = w.x;
            f[2 * u + 1] = w.y;
          }
          raw[i] = pack8(f);
        }
        if (where == NONE) raw[i] = make_uint4(0u, 0u, 0u, 0u);
        bf16* dst = pick(is_v, p.k_out + t * p.hkv * D + c, p.v_out + t * p.hkv * D + c) + (is_v ? r - p.hkv : r) * D;
        if (r < rows) *reinterpret_cast<uint4*>(dst) = raw[i];
      }
    } else {
      if (r0 > 0) load_new(r0);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = r0 + i * RPI + sub;
        const bool is_v = r >= p.hkv;
        const int slot = (is_v ? r - p.hkv : r) << p.page_shift;
        uint8_t* dst = pick(is_v, k_at, v_at) + slot * (D * ESZ);
        if (!QUANT) {
          if (r < rows) *reinterpret_cast<uint4*>(dst) = raw[i];
        } else {
          const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
          __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
          for (int u = 1; u < 4; ++u) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[u])));
          float a = fmaxf(__low2float(m), __high2float(m));
#pragma unroll
          for (int o = LPR / 2; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
          const int b = scale_byte(a);
          const float inv = scale_inverse(b);
          uint16_t q[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float2 f = __fmul2_rn(make_float2(__uint_as_float(w[u] << 16), __uint_as_float(w[u] & 0xffff0000u)),
                                        make_float2(inv, inv));
            q[u] = f32x2_to_e4m3x2(f.x, f.y);
          }
          if (r < rows) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(q[0] | ((uint32_t)q[1] << 16), q[2] | ((uint32_t)q[3] << 16));
            if (c == 0) pick(is_v, ks_at, vs_at)[slot] = (uint8_t)b;
          }
        }
      }
    }
  }
}

// Page size as a shift; 0 when it is not a power of two from 16 to 256.
static int page_shift_of(int64_t page_size) {
  for (int s = 4; s <= 8; ++s)
    if (page_size == (int64_t)1 << s) return s;
  return 0;
}

static int check_kv(const char* what, const KvParams& p, int64_t page_size, int64_t head_dim, int quant) {
  if (!p.k_cache || !p.v_cache || !p.table || !p.cu || !p.kv_lens)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (quant && (!p.k_scale || !p.v_scale))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: an e4m3 cache needs k_scale and v_scale", what);
  if (head_dim != 128 && head_dim != 256)
    return set_error(FDK_ERR_UNSUPPORTED, "%s: head_dim=%lld (128 and 256 supported)", what, (long long)head_dim);
  if (!page_shift_of(page_size))
    return set_error(FDK_ERR_UNSUPPORTED, "%s: page_size=%lld (16, 32, 64, 128 or 256)", what, (long long)page_size);
  if (p.hkv < 1 || p.hkv > 4096 || p.nseg < 1 || p.tokens < 0 || p.tokens > 0x7fffffff - 4 || p.num_pages < 1 ||
      p.num_pages > 0x7fffffff || p.max_pages < 1 || p.ld_table < p.max_pages)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: bad sizes", what);
  const int64_t page_elems = page_size * p.hkv * head_dim;
  if (p.ld_kpage < page_elems || p.ld_vpage < page_elems ||
      (quant && (p.ld_kscale_page < page_size * p.hkv || p.ld_vscale_page < page_size * p.hkv)))
    return set_error(FDK_ERR_INVALID_ARGUMENT, "%s: page stride too small", what);
  const int64_t per16 = quant ? 16 : 8;
  if (!aligned16(p.k_cache) || !aligned16(p.v_cache) || p.ld_kpage % per16 || p.ld_vpage % per16)
    return set_error(FDK_ERR_ALIGNMENT, "%s: the cache and its pages must be 16-byte aligned", what);
  return FDK_OK;
}

template <bool READ>
static int launch(const KvParams& p, int64_t head_dim, int quant, cudaStream_t s, const char* what) {
  if (p.tokens == 0) return FDK_OK;
  const unsigned grid = (unsigned)((p.tokens + 3) / 4);
  if (head_dim == 128) {
    if (quant) kv_rows_kernel<128, true, READ><<<grid, 128, 0, s>>>(p);
    else kv_rows_kernel<128, false, READ><<<grid, 128, 0, s>>>(p);
  } else {
    if (quant) kv_rows_kernel<256, true, READ><<<grid, 128, 0, s>>>(p);
    else kv_rows_kernel<256, false, READ><<<grid, 128, 0, s>>>(p);
  }
  return check_launch(what);
}

}  // namespace paged

int paged_kv_take_device_error() {
  int h = 0;
  if (cudaMemcpyFromSymbol(&h, paged::g_kv_error, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (h) {
    const int zero = 0;
    cudaMemcpyToSymbol(paged::g_kv_error, &zero, sizeof(int));
  }
  return h;
}

}  // namespace fdk

using namespace fdk;

extern "C" int fdk_paged_kv_write(const void* k, int64_t ld_k, const void* v, int64_t ld_v, void* k_cache,
                                  int64_t ld_kpage, void* v_cache, int64_t ld_vpage, int cache_is_e4m3,
                                  void* k_scale, int64_t ld_kscale_page, void* v_scale, int64_t ld_vscale_page,
                                  int64_t num_pages, int64_t page_size, const int32_t* page_table, int64_t ld_table,
                                  int64_t max_pages, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                  int64_t num_segments, int64_t tokens, int64_t hkv, int64_t head_dim, void* stream) {
  using namespace fdk::paged;
  if (int st = check_device()) return st;
  if (num_segments > 0x7ffffffe || max_pages > 0x7fffffff || hkv > 4096)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "paged_kv_write: bad sizes");
  KvParams p = {};
  p.k = static_cast<const bf16*>(k); p.v = static_cast<const bf16*>(v);
  p.ld_k = ld_k; p.ld_v = ld_v;
  p.k_cache = k_cache; p.v_cache = v_cache; p.ld_kpage = ld_kpage; p.ld_vpage = ld_vpage;
  p.k_scale = static_cast<uint8_t*>(k_scale); p.v_scale = static_cast<uint8_t*>(v_scale);
  p.ld_kscale_page = ld_kscale_page; p.ld_vscale_page = ld_vscale_page;
  p.table = page_table; p.ld_table = ld_table; p.cu = cu_seqlens; p.kv_lens = kv_lens;
  p.tokens = tokens; p.num_pages = num_pages; p.nseg = (int)num_segments; p.max_pages = (int)max_pages;
  p.page_shift = page_shift_of(page_size); p.hkv = (int)hkv;
  if (int st = check_kv("paged_kv_write", p, page_size, head_dim, cache_is_e4m3)) return st;
  if (tokens && (!k || !v)) return set_error(FDK_ERR_INVALID_ARGUMENT, "paged_kv_write: null pointer");
  if (ld_k < hkv * head_dim || ld_v < hkv * head_dim)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "paged_kv_write: row stride too small");
  if (!aligned16(k) || !aligned16(v) || ld_k % 8 || ld_v % 8)
    return set_error(FDK_ERR_ALIGNMENT, "paged_kv_write: pointers and strides must be 16-byte aligned");
  return launch<false>(p, head_dim, cache_is_e4m3, static_cast<cudaStream_t>(stream), "paged_kv_write");
}

extern "C" int fdk_paged_kv_read(const void* k_cache, int64_t ld_kpage, const void* v_cache, int64_t ld_vpage,
                                 int cache_is_e4m3, const void* k_scale, int64_t ld_kscale_page, const void* v_scale,
                                 int64_t ld_vscale_page, int64_t num_pages, int64_t page_size,
                                 const int32_t* page_table, int64_t ld_table, int64_t max_pages,
                                 const int32_t* cu_seqlens, const int32_t* kv_lens, int64_t num_segments,
                                 int64_t tokens, int64_t hkv, int64_t head_dim, void* k_out, void* v_out,
                                 void* stream) {
  using namespace fdk::paged;
  if (int st = check_device()) return st;
  if (num_segments > 0x7ffffffe || max_pages > 0x7fffffff || hkv > 4096)
    return set_error(FDK_ERR_INVALID_ARGUMENT, "paged_kv_read: bad sizes");
  KvParams p = {};
  p.k_out = static_cast<bf16*>(k_out); p.v_out = static_cast<bf16*>(v_out);
  p.k_cache = const_cast<void*>(k_cache); p.v_cache = const_cast<void*>(v_cache);
  p.ld_kpage = ld_kpage; p.ld_vpage = ld_vpage;
  p.k_scale = static_cast<uint8_t*>(const_cast<void*>(k_scale));
  p.v_scale = static_cast<uint8_t*>(const_cast<void*>(v_scale));
  p.ld_kscale_page = ld_kscale_page; p.ld_vscale_page = ld_vscale_page;
  p.table = page_table; p.ld_table = ld_table; p.cu = cu_seqlens; p.kv_lens = kv_lens;
  p.tokens = tokens; p.num_pages = num_pages; p.nseg = (int)num_segments; p.max_pages = (int)max_pages;
  p.page_shift = page_shift_of(page_size); p.hkv = (int)hkv;
  if (int st = check_kv("paged_kv_read", p, page_size, head_dim, cache_is_e4m3)) return st;
  if (tokens && (!k_out || !v_out)) return set_error(FDK_ERR_INVALID_ARGUMENT, "paged_kv_read: null pointer");
  if (!aligned16(k_out) || !aligned16(v_out))
    return set_error(FDK_ERR_ALIGNMENT, "paged_kv_read: outputs must be 16-byte aligned");
  return launch<true>(p, head_dim, cache_is_e4m3, static_cast<cudaStream_t>(stream), "paged_kv_read");
}
