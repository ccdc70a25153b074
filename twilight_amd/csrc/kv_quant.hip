// K / V held in 8 bits: quantised as they are written into pages, and read back.
//
// A row is the 128 channels of one token and kv head. With T the largest value a code stands for
// (127 for int8, 448 for e4m3):
//     scale = max(max|x| / T, 2^-126)      code = round_to_nearest_even(x / scale)
//     value = code * scale
// in fp32 with IEEE division, K and V each with a scale of their own per row. The floor keeps the
// scale a normal number, so that a row of zeros needs no case of its own. A row that holds an
// infinity or a NaN gets scale NaN and codes 0: it reads back as NaN throughout.
//
// Tokens come ragged: rows token_indptr[b] .. token_indptr[b + 1] are the LAST tokens of request b
// as the page table counts them, so a table that has been advanced describes the step completely
// and a call can be repeated. 16 lanes share a row (8 channels a lane: one 16-byte load, one
// 8-byte store) and find its request with a 16-way search, so up to 16 requests cost one load
// round trip and 256 cost two.
//
// Bound by memory: 32768 bf16 tokens of 32 heads, 814 MB either way, are written in 165 us (4.9 TB/s) and read
// in 175 (4.6), where a large copy reaches 5.2 TB/s. A decode step of 8 requests and 8 heads is a chain of
// loads and takes 3.4 us to write, 2.8 to read.
#include "twl_common.h"

namespace twl {

struct KvQuantArgs {
  const void* k_dense;        // [tokens, kv heads, 128] rows: the new ones, or where they are read to
  const void* v_dense;
  uint64_t dense_token, dense_head;             // element strides of the dense rows
  uint8_t* k_cache;
  uint8_t* v_cache;
  uint64_t page_stride, token_stride, head_stride;
  float* k_scale;
  float* v_scale;
  uint64_t scale_page, scale_token, scale_head;
  const int32_t* token_indptr;
  const int32_t* kv_page_indices;
  const int32_t* kv_page_indptr;
  const int32_t* kv_last_page_len;
  uint32_t tokens, batch, num_kv_heads, num_pages;
};

constexpr int kQuantThreads = 256;
constexpr float kQuantMinScale = 1.17549435e-38f;   // 2^-126

// What a token's row has in the cache.
enum RowPlace { kRowBehind, kRowNowhere, kRowPlaced };

// Request, page and slot of token t, by the 16 lanes of a row together. kRowBehind: no request
// names the token. kRowNowhere: its request holds fewer tokens than token_indptr gives it, or the
// page table names a page outside the cache.
__device__ __forceinline__ int find_row(const KvQuantArgs& a, uint32_t t, uint32_t& page, uint32_t& slot) {
  const int lane = lane_id(), sub = lane & 15, shift = lane & 48;
  // b = how many of token_indptr[1 .. batch] are <= t
  uint32_t lo = 0, n = a.batch;
  while (n > 0) {
    const uint32_t step = (n + 15) / 16;
    const uint32_t at = (sub + 1) * step - 1;
    const bool below = at < n && (uint32_t)a.token_indptr[1 + lo + at] <= t;
    const uint32_t c = __builtin_popcount((uint32_t)((__ballot(below) >> shift) & 0xFFFFu));
    lo += c * step;
    n = c * step >= n ? 0 : min(step, n - c * step);
    if (step == 1) break;
    n = min(n, step - 1);          // the probe at the end of this block is known to be above t
  }
  if (lo >= a.batch || t < (uint32_t)a.token_indptr[lo]) return kRowBehind;
  const int end = a.token_indptr[lo + 1];
  const int p0 = a.kv_page_indptr[lo], np = a.kv_page_indptr[lo + 1] - p0;
  const int last = a.kv_last_page_len[lo];
  if (np <= 0 || last < 0 || last > TWL_PAGE) return kRowNowhere;
  const int64_t pos = (int64_t)(np - 1) * TWL_PAGE + last - (end - (int64_t)t);
  if (pos < 0) return kRowNowhere;
  page = (uint32_t)a.kv_page_indices[p0 + (int)(pos / TWL_PAGE)];
  slot = (uint32_t)(pos % TWL_PAGE);
  return page < a.num_pages ? kRowPlaced : kRowNowhere;
}

// largest |x| of a row as its fp32 bit pattern: as integers the patterns of infinities and NaN
// compare above every finite one
__device__ __forceinline__ uint32_t row_amax_bits(const float* x) {
  int m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, as_i32(x[i]) & 0x7FFFFFFF);
  m = max(m, dpp<kDppXor1>(0, m));
  m = max(m, dpp<kDppXor2>(0, m));
  m = max(m, dpp<kDppHalfMirror>(0, m));
  m = max(m, dpp<kDppMirror>(0, m));
  return (uint32_t)m;
}

// codes of a lane's 8 channels, and the row's scale. x / scale as IEEE division rounds it, for the price
// of one division per row: with r the correctly rounded 1 / scale and q0 = x r, one correction
// q0 + r (x - q0 scale) in fused multiply-adds is the correctly rounded quotient (Markstein's
// theorem), as long as the remainder is representable; rows too small for that divide.
template <int FMT>
__device__ __forceinline__ u32x2 quantise8(const float* x, float& scale) {
  const uint32_t amax = row_amax_bits(x);
  u32x2 codes = {0u, 0u};
  if (amax >= 0x7F800000u) {
    scale = __builtin_nanf("");
    return codes;
  }
  scale = fmaxf(as_f32(amax) / (FMT == TWL_I8 ? 127.0f : 448.0f), kQuantMinScale);
  float y[8];
  if (scale >= 8.0779357e-28f) {            // 2^-90: good for quotients from 2^-13 on, smaller ones are code 0
    const float r = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = x[i] * r;
      y[i] = copysignf(fmaf(fmaf(-q, scale, x[i]), r, q), x[i]);   // the correction loses the sign of -0
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] / scale;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w = 0;
    if (FMT == TWL_I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)rintf(y[4 * h + i]) & 0xFFu) << (8 * i);
    } else {
      // the hardware convert rounds to nearest even; |y| <= 448 up to its last bit, which rounds
      // to 448
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], p, true);
      w = (uint32_t)p;
    }
    codes[h] = w;
  }
  return codes;
}

// Heads per row of 16 lanes: a bulk call takes four, so that finding the token's place is paid once and
// eight loads are on their way; a decode step takes one and spreads wider.
template <int HB>
__device__ __forceinline__ bool token_and_head(const KvQuantArgs& a, uint32_t& t, uint32_t& h) {
  const uint32_t sets = (a.num_kv_heads + HB - 1) / HB;
  const uint64_t at = (uint64_t)blockIdx.x * (kQuantThreads / 16) + threadIdx.x / 16;
  t = (uint32_t)(at / sets);
  h = (uint32_t)(at - (uint64_t)t * sets) * HB;
  return t < a.tokens;
}

template <int DT, int FMT, int HB>
__global__ __launch_bounds__(kQuantThreads) void kv_quant_append_kernel(KvQuantArgs a) {
  const int sub = threadIdx.x & 15;
  uint32_t t, h;
  if (!token_and_head<HB>(a, t, h)) return;
  u32x4 kb[HB], vb[HB];
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    const size_t src = t * a.dense_token + min(h + i, a.num_kv_heads - 1) * a.dense_head + 8 * sub;
    kb[i] = __builtin_nontemporal_load((const u32x4*)((const uint16_t*)a.k_dense + src));
    vb[i] = __builtin_nontemporal_load((const u32x4*)((const uint16_t*)a.v_dense + src));
  }
  uint32_t page, slot;
  if (find_row(a, t, page, slot) != kRowPlaced) return;
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    if (h + i >= a.num_kv_heads) break;
    const size_t dst = page * a.page_stride + slot * a.token_stride + (h + i) * a.head_stride + 8 * sub;
    const size_t sdst = page * a.scale_page + slot * a.scale_token + (h + i) * a.scale_head;
    float x[8], scale;
    unpack8<DT>(kb[i], x);
    *(u32x2*)(a.k_cache + dst) = quantise8<FMT>(x, scale);
    if (sub == 0) a.k_scale[sdst] = scale;
    unpack8<DT>(vb[i], x);
    *(u32x2*)(a.v_cache + dst) = quantise8<FMT>(x, scale);
    if (sub == 0) a.v_scale[sdst] = scale;
  }
}

// the values a lane's 8 codes stand for
template <int FMT>
__device__ __forceinline__ void dequantise8(u32x2 codes, float scale, float* x) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = (int)codes[h];
    if (FMT == TWL_I8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = (float)((w << (24 - 8 * i)) >> 24) * scale;
    } else {
      x[4 * h] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * scale;
      x[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale;
      x[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale;
      x[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale;
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* base, size_t at, const float* x) {
  if (DT == TWL_F32) {
    *(f32x4*)((float*)base + at) = f32x4{x[0], x[1], x[2], x[3]};
    *(f32x4*)((float*)base + at + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = f32_to_bits16<DT>(x[2 * i]) | (f32_to_bits16<DT>(x[2 * i + 1]) << 16);
    *(u32x4*)((uint16_t*)base + at) = w;
  }
}

template <int DT, int FMT, int HB>
__global__ __launch_bounds__(kQuantThreads) void kv_quant_read_kernel(KvQuantArgs a) {
  const int sub = threadIdx.x & 15;
  uint32_t t, h;
  if (!token_and_head<HB>(a, t, h)) return;
  uint32_t page, slot;
  const int where = find_row(a, t, page, slot);
  if (where == kRowBehind) return;
  u32x2 kc[HB] = {}, vc[HB] = {};
  float ks[HB] = {}, vs[HB] = {};
  if (where == kRowPlaced) {
#pragma unroll
    for (int i = 0; i < HB; ++i) {
      const uint32_t hh = min(h + i, a.num_kv_heads - 1);
      const size_t src = page * a.page_stride + slot * a.token_stride + hh * a.head_stride + 8 * sub;
      const size_t ssrc = page * a.scale_page + slot * a.scale_token + hh * a.scale_head;
      kc[i] = *(const u32x2*)(a.k_cache + src);
      vc[i] = *(const u32x2*)(a.v_cache + src);
      ks[i] = a.k_scale[ssrc];
      vs[i] = a.v_scale[ssrc];
    }
  }
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    if (h + i >= a.num_kv_heads) break;
    float x[8];
    const size_t dst = ((size_t)t * a.num_kv_heads + h + i) * TWL_HEAD_DIM + 8 * sub;
    dequantise8<FMT>(kc[i], ks[i], x);
    store8<DT>((void*)a.k_dense, dst, x);
    dequantise8<FMT>(vc[i], vs[i], x);
    store8<DT>((void*)a.v_dense, dst, x);
  }
}

// Checks that both directions share; fills everything but the dense side.
int kv_quant_args(KvQuantArgs& a, uint8_t* k_cache, uint8_t* v_cache, int format, uint64_t page_stride,
                  uint64_t token_stride, uint64_t head_stride, float* k_scale, float* v_scale,
                  uint64_t scale_page, uint64_t scale_token, uint64_t scale_head, uint32_t num_pages,
                  const int32_t* kv_page_indices, const int32_t* kv_page_indptr,
                  const int32_t* kv_last_page_len, const int32_t* token_indptr, uint32_t tokens,
                  uint32_t batch, uint32_t num_kv_heads) {
  if (!k_cache || !v_cache || !k_scale || !v_scale || !kv_page_indices || !kv_page_indptr ||
      !kv_last_page_len || !token_indptr)
    return TWL_ENULL;
  if (format != TWL_I8 && format != TWL_E4M3) return TWL_EDTYPE;
  if (tokens == 0 || batch == 0 || num_kv_heads == 0 || num_pages == 0 || tokens > 0x7FFFFFFFu ||
      num_pages > 0x7FFFFFFFu)
    return TWL_EINVAL;
  if (((uint64_t)tokens * num_kv_heads + 15) / 16 > 0xFFFFFFull) return TWL_EINVAL;   // 2^32 threads
  if ((page_stride | token_stride | head_stride) & 7u) return TWL_EALIGN;
  if ((((uintptr_t)k_cache) | ((uintptr_t)v_cache)) & 7u) return TWL_EALIGN;
  if ((((uintptr_t)k_scale) | ((uintptr_t)v_scale)) & 3u) return TWL_EALIGN;
  a.k_cache = k_cache; a.v_cache = v_cache; a.page_stride = page_stride;
  a.token_stride = token_stride; a.head_stride = head_stride; a.k_scale = k_scale;
  a.v_scale = v_scale; a.scale_page = scale_page; a.scale_token = scale_token;
  a.scale_head = scale_head; a.token_indptr = token_indptr; a.kv_page_indices = kv_page_indices;
  a.kv_page_indptr = kv_page_indptr; a.kv_last_page_len = kv_last_page_len; a.tokens = tokens;
  a.batch = batch; a.num_kv_heads = num_kv_heads; a.num_pages = num_pages;
  return TWL_OK;
}

// Heads per row of 16 lanes, and the grid: four where that leaves half a load of the chip (256 compute units x 4
// workgroups of 16 rows). One head and four, to write and to read: 32768 tokens of 32 heads 189 and 224 us, 166
// and 176; 16384 of 8 heads 31 and 19, 26 and 18; 8192 of 8 17 and 12, 16 and 10; 4096 of 8 10.6 and 7.8, 10.8
// and 7.5.
static bool quant_grid(const KvQuantArgs& a, dim3& grid) {
  const uint64_t four = ((uint64_t)a.tokens * ((a.num_kv_heads + 3) / 4) + 15) / 16;
  const bool bulk = a.num_kv_heads >= 4 && four >= 1024;
  grid = dim3((uint32_t)(bulk ? four : ((uint64_t)a.tokens * a.num_kv_heads + 15) / 16));
  return bulk;
}

}  // namespace twl

extern "C" int twl_kv_quant_append(
    const void* k_new, const void* v_new, int dtype, uint64_t new_token_stride,
    uint64_t new_head_stride, const int32_t* token_indptr, uint32_t tokens, void* k_cache,
    void* v_cache, int format, uint64_t page_stride, uint64_t token_stride, uint64_t head_stride,
    float* k_scale, float* v_scale, uint64_t scale_page_stride, uint64_t scale_token_stride,
    uint64_t scale_head_stride, uint32_t num_pages, const int32_t* kv_page_indices,
    const int32_t* kv_page_indptr, const int32_t* kv_last_page_len, uint32_t batch,
    uint32_t num_kv_heads, void* stream) {
  if (!k_new || !v_new) return TWL_ENULL;
  if (dtype != TWL_F16 && dtype != TWL_BF16) return TWL_EDTYPE;
  twl::KvQuantArgs a{};
  const int rc = twl::kv_quant_args(a, (uint8_t*)k_cache, (uint8_t*)v_cache, format, page_stride,
                                    token_stride, head_stride, k_scale, v_scale, scale_page_stride,
                                    scale_token_stride, scale_head_stride, num_pages,
                                    kv_page_indices, kv_page_indptr, kv_last_page_len, token_indptr,
                                    tokens, batch, num_kv_heads);
  if (rc != TWL_OK) return rc;
  if ((new_token_stride | new_head_stride) & 7u) return TWL_EALIGN;   // 16-byte loads
  if ((((uintptr_t)k_new) | ((uintptr_t)v_new)) & 15u) return TWL_EALIGN;
  a.k_dense = k_new; a.v_dense = v_new; a.dense_token = new_token_stride; a.dense_head = new_head_stride;
  dim3 grid, block(twl::kQuantThreads);
  const bool bulk = twl::quant_grid(a, grid);
#define TWL_APPEND(DT, FMT)                                                                                        \
  do {                                                                                                             \
    if (bulk) hipLaunchKernelGGL((twl::kv_quant_append_kernel<DT, FMT, 4>), grid, block, 0, (hipStream_t)stream, a); \
    else hipLaunchKernelGGL((twl::kv_quant_append_kernel<DT, FMT, 1>), grid, block, 0, (hipStream_t)stream, a);      \
  } while (0)
  if (dtype == TWL_F16) { if (format == TWL_I8) TWL_APPEND(TWL_F16, TWL_I8); else TWL_APPEND(TWL_F16, TWL_E4M3); }
  else { if (format == TWL_I8) TWL_APPEND(TWL_BF16, TWL_I8); else TWL_APPEND(TWL_BF16, TWL_E4M3); }
#undef TWL_APPEND
  return hipGetLastError() == hipSuccess ? TWL_OK : TWL_ELAUNCH;
}

extern "C" int twl_kv_quant_read(
    void* k_out, void* v_out, int dtype, const int32_t* token_indptr, uint32_t tokens,
    const void* k_cache, const void* v_cache, int format, uint64_t page_stride,
    uint64_t token_stride, uint64_t head_stride, const float* k_scale, const float* v_scale,
    uint64_t scale_page_stride, uint64_t scale_token_stride, uint64_t scale_head_stride,
    uint32_t num_pages, const int32_t* kv_page_indices, const int32_t* kv_page_indptr,
    const int32_t* kv_last_page_len, uint32_t batch, uint32_t num_kv_heads, void* stream) {
  if (!k_out || !v_out) return TWL_ENULL;
  if (dtype != TWL_F16 && dtype != TWL_BF16 && dtype != TWL_F32) return TWL_EDTYPE;
  twl::KvQuantArgs a{};
  const int rc = twl::kv_quant_args(a, (uint8_t*)k_cache, (uint8_t*)v_cache, format, page_stride,
                                    token_stride, head_stride, (float*)k_scale, (float*)v_scale,
                                    scale_page_stride, scale_token_stride, scale_head_stride,
                                    num_pages, kv_page_indices, kv_page_indptr, kv_last_page_len,
                                    token_indptr, tokens, batch, num_kv_heads);
  if (rc != TWL_OK) return rc;
  if ((((uintptr_t)k_out) | ((uintptr_t)v_out)) & 15u) return TWL_EALIGN;
  a.k_dense = k_out; a.v_dense = v_out;
  dim3 grid, block(twl::kQuantThreads);
  const bool bulk = twl::quant_grid(a, grid);
#define TWL_READ(DT, FMT)                                                                                        \
  do {                                                                                                           \
    if (bulk) hipLaunchKernelGGL((twl::kv_quant_read_kernel<DT, FMT, 4>), grid, block, 0, (hipStream_t)stream, a); \
    else hipLaunchKernelGGL((twl::kv_quant_read_kernel<DT, FMT, 1>), grid, block, 0, (hipStream_t)stream, a);      \
  } while (0)
#define TWL_READ_DT(FMT)                            \
  if (dtype == TWL_F16) TWL_READ(TWL_F16, FMT);     \
  else if (dtype == TWL_BF16) TWL_READ(TWL_BF16, FMT); \
  else TWL_READ(TWL_F32, FMT)
  if (format == TWL_I8) { TWL_READ_DT(TWL_I8); } else { TWL_READ_DT(TWL_E4M3); }
#undef TWL_READ_DT
#undef TWL_READ
  return hipGetLastError() == hipSuccess ? TWL_OK : TWL_ELAUNCH;
}
