// Paged decode attention over 16-bit or 8-bit pages, for requests in groups that share a prefix.
//
// Request b of group g sees the tokens of the group's prefix pages and then its own:
//     out[b, h] = softmax(sm_scale * q[b, h] . K) V        lse[b, h] = log sum exp(logit)
// A softmax over a set of tokens is the merge of softmaxes over its parts: every part leaves
// (m, l, acc) = (a reference, sum of exp2(s - m), sum of exp2(s - m) V) of its tokens, and parts
// are joined by rescaling to the largest reference. So the prefix is read once per group and kv head,
// with the queries of all its requests as the columns of one matrix product, and the requests' own
// tokens are ordinary parts beside it.
//
// One wavefront works on tiles of 32 tokens (two pages) and 16 query rows, without LDS
// and without moving anything between lanes. With n = lane % 16, kb = lane / 16:
//   S^T = K Q^T   A operand: token n of a page, 8 channels per lane; B operand: query n. A lane of
//                 the result holds query n's logits of tokens 4 kb + i of either page.
//   O^T += V^T P^T   The order of the 32 tokens inside the product is free, so k-slot (kb, i) is
//                 given to exactly the eight tokens whose weights the lane already has: the weights
//                 are the B operand as they stand. The A operand wants the same eight tokens of
//                 one channel: a lane loads 8 channels 8 n .. 8 n + 7 of its eight tokens (a row of
//                 16 lanes covers a token's 128 channels) and transposes 8 x 8 in registers; product
//                 j takes channel 8 n + j of every lane.
// A lane of O^T then holds 32 consecutive channels of ONE query, so maxima, sums and rescaling are
// per-lane scalars. The reference m of a row's weights 2^(s - m) is only raised (and the accumulators rescaled)
// when a logit leaves the room above it, so that most tiles need no reduction across lanes at all. l, the
// accumulators and m belong together, wherever in that room the largest logit lies.
//
// 8-bit pages run on fp16 products (codes are exact in fp16). The scale of K multiplies the logit.
// The scale of V joins the weight, relative to a running power of two that bounds the V scales seen; a bf16
// query is first brought into fp16's range by a power of two of its own.
//
// The weights are rounded to the product's 16-bit type; the sum l takes them before that rounding, in fp32. In
// bf16 that is half a step (2^-8) of each weight. So it is in fp16 (2^-11) down to fp16's normal range, below
// which a weight is off by up to 2^-25 of the product's unit. A token that takes nearly all of the weight and
// has a small V leaves the answer to weights like that, so fp16 products use the range above 1: a row's
// reference is put 12 below its largest logit in base 2 and a logit may exceed it by 14 before it is raised.
// Weights are then below 2^14, also times a V scale (taken below 1), the largest one seen at least 2^12, and what
// is lost below the normal range is 2^-37 of that one (over 8-bit pages 2^-36 of it times the largest V scale
// seen). The smaller room raises references more often: 33 samples over int8 in three groups 39.3 -> 40.4 us, 8
// requests of 32768 int8 tokens 98 before and after.
// bf16 has fp32's range: the reference is the maximum and the room 8.
// What the rounding costs (64 samples of a 32768-token bf16 prompt): out is off by 0.0023 (root mean square) of its
// size, 0.0017 of which is its own rounding to bf16. A second product with what the weights lose leaves that
// 0.0017 and takes 89 us instead of 81. fp16: 0.0003, of which 0.0002.
//
// What bounds it: one read of K and V where few rows share it (8 requests of 32768 int8 tokens, 8 kv heads:
// 554 MB in 93 us, 5.9 TB/s), products and exponentials where many do (256 samples of a 32768-token bf16
// prompt: 137 GFLOP in 170 us, 0.81 PFLOP/s; the exponentials alone take 40 % of the vector pipe), in between
// the parts' partial results (64 samples: 34 MB written and read again) and start and end of the parts.
#include "twl_common.h"

namespace twl {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kPaThreads = 256;
constexpr int kPaWaves = kPaThreads / kWave;
constexpr int kPaTile = 32;                 // tokens of one step of a wavefront
constexpr float kPaNoMax = -3.0e38f;        // reference before the first token
constexpr uint32_t kPaMaxParts = 256;       // of one kind, per row
constexpr float kPaLeastScale = 1.17549435e-38f;   // 2^-126: -inf times it is -inf
constexpr float kLn2 = 0.693147180559945309f;

struct PrefixAttnArgs {
  const uint16_t* q;                        // [batch, num_q_heads, 128]
  void* out;
  float* lse;
  const uint8_t* k;
  const uint8_t* v;
  uint64_t page_bytes, head_bytes;
  uint32_t token_bytes;
  const float* ks;                          // 8-bit pages: one scale per (page, token, kv head)
  const float* vs;
  uint64_t scale_page, scale_head;
  uint32_t scale_token;
  bool scale_vec;                           // the scales of four tokens are one aligned 16-byte load
  uint32_t num_pages;
  const int32_t *p_ids, *p_ptr, *p_last, *g_ptr;   // prefix tables, members of every group
  const int32_t *ids, *ptr, *last;                 // the requests' own pages
  uint32_t batch, num_q_heads, num_kv_heads, G, groups;
  uint32_t max_prefix, max_group, max_tokens;
  uint32_t p_chunk, p_chunks, p_tiles;      // prefix: tokens per part, parts, row tiles per group
  uint32_t chunk, chunks, tiles;            // own tokens: the same
  uint32_t own_blocks;                      // workgroups of the own parts, first in the grid
  float scale_log2, lse_below;
  float* acc;                               // [rows, parts, 128]
  f32x2* ml;                                // [rows, parts]
};

__device__ __forceinline__ float max_over_kb(float x) {
  const uint32_t u = as_u32(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t y = as_u32(fmaxf(as_f32(a[0]), as_f32(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return fmaxf(as_f32(b[0]), as_f32(b[1]));
}
__device__ __forceinline__ float sum_over_kb(float x) {
  const uint32_t u = as_u32(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t y = as_u32(as_f32(a[0]) + as_f32(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return as_f32(b[0]) + as_f32(b[1]);
}

template <int MT>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if (MT == TWL_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                  __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// How far a row's reference lies below its largest logit when it is set, and how far above it a logit may
// come, in base 2 (MT: type of the second product's operands).
template <int MT> constexpr float kPaBelow = MT == TWL_F16 ? 12.0f : 0.0f;
template <int MT> constexpr float kPaRoom = MT == TWL_F16 ? 14.0f : 8.0f;
// What sums leave a part with, so that they are as large as if the reference were the largest logit (2^-below): V
// up to fp32's largest number over the tokens stays finite. lse adds `lse_below` for it.
template <int MT> constexpr float kPaUnit = MT == TWL_F16 ? 1.0f / 4096.0f : 1.0f;

// The reference m raised for a largest logit of `top`. Where the difference is lost in fp32's steps (logits
// beyond 2^26) it is the logit itself.
template <int MT>
__device__ __forceinline__ float raised(float m, float top) {
  const float up = fmaxf(m, top - kPaBelow<MT>);
  return top - up > kPaRoom<MT> ? top : up;
}

template <int MT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {   // one convert for both
  const f32x2 v = {x, y};
  if (MT == TWL_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2_t));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// four 8-bit codes -> four fp16 values
template <int KV>
__device__ __forceinline__ u32x2 widen4(uint32_t w) {
  if (KV == TWL_E4M3) {
    const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false);
    const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
  }
  // 0x6400 | u is the fp16 number 1024 + u; u = code + 128
  const uint32_t u = w ^ 0x80808080u;
  const half2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  const half2_t a = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
  const half2_t b = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
  return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// K and V of a streamed part are read once
template <class T>
__device__ __forceinline__ T load_kv(const uint8_t* p) {
  return __builtin_nontemporal_load((const T*)p);
}

// Tokens of a page list, bounded by what the caller sized the launch for.
__device__ __forceinline__ int list_len(const int32_t* ptr, const int32_t* last, uint32_t i, uint32_t bound) {
  const int64_t np = (int64_t)ptr[i + 1] - ptr[i];
  if (np <= 0) return 0;
  return (int)min((np - 1) * TWL_PAGE + min(max(last[i], 0), TWL_PAGE), (int64_t)bound);
}

// Group of request b: the g with g_ptr[g] <= b < g_ptr[g + 1], or -1. By a whole wavefront.
__device__ __forceinline__ int group_of(const PrefixAttnArgs& a, uint32_t b) {
  int g = -1;
  for (uint32_t g0 = 0; g0 < a.groups; g0 += kWave) {
    const uint32_t i = g0 + lane_id();
    const bool in = i < a.groups && a.g_ptr[i] <= (int)b && (int)b < a.g_ptr[i + 1];
    const uint64_t hit = __ballot(in);
    if (hit) g = (int)g0 + __builtin_ctzll(hit);
  }
  return g;
}

// The queries of a set of 16 rows as the B operand of S^T, and the factor that makes base-2 logits of
// its products. PAIRED: channels in the order in which 16-byte loads of 8-bit K deliver them. TO_F16:
// for products in fp16; a bf16 query goes there by way of a power of two.
template <int QT, bool PAIRED, bool TO_F16>
__device__ __forceinline__ void load_query(const PrefixAttnArgs& a, int row, int kb, u32x4* qf, float& scale) {
  const uint16_t* src = a.q + (size_t)max(row, 0) * TWL_HEAD_DIM;
  // positive, so that the largest product is the largest logit and a masked one stays masked: a negative
  // scale turns the query, a scale of zero clears it
  const bool flat = a.scale_log2 == 0.0f;
  scale = flat ? 1.0f : fabsf(a.scale_log2);
  const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int d = PAIRED ? 64 * (j >> 1) + 16 * kb + 8 * (j & 1) : 32 * j + 8 * kb;
    qf[j] = *(const u32x4*)(src + d);
    if (row < 0 || flat) qf[j] = u32x4{0, 0, 0, 0};
    else qf[j] ^= sign;
  }
  if (TO_F16 && QT == TWL_BF16) {
    float f[4][8];
    int top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unpack8<QT>(qf[j], f[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, as_i32(f[j][i]) & 0x7FFFFFFF);
    }
    top = as_i32(max_over_kb(as_f32(top)));
    // |q| < 2^(e + 15), below fp16's 2^16, so that a channel keeps its 8 bits down to 2^-31 of the largest one
    // (relative to 1 it was 2^-16, and logits can come from channels smaller than that). A query below 2^-60 meets
    // K scales whose products with that would overflow: it comes down to 1. NaN stays NaN
    const int size = (top >> 23) - 127;
    const int e = min(max(size - min(max(size + 74, 0), 14), -126), 126);
    const float down = as_f32((127 - e) << 23);
    scale *= as_f32((127 + e) << 23);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[j][i] = pack2<TWL_F16>(f[j][2 * i] * down, f[j][2 * i + 1] * down);
  }
  scale = fmaxf(scale, kPaLeastScale);
}

// Four channels of a row's part: into the workspace, or, where a row has one part, the answer.
template <int QT>
__device__ __forceinline__ void put_row(const PrefixAttnArgs& a, int row, uint32_t part, uint32_t parts, int c,
                                        f32x4 x, float m, float l) {
  if (parts > 1) {
    const size_t at = (size_t)row * parts + part;
    *(f32x4*)(a.acc + at * TWL_HEAD_DIM + c) = x;
    if (c == 0) a.ml[at] = f32x2{m, l};
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *(u32x2*)((uint16_t*)a.out + (size_t)row * TWL_HEAD_DIM + c) =
      u32x2{pack2<QT>(x[0] * inv, x[1] * inv), pack2<QT>(x[2] * inv, x[3] * inv)};
  if (a.lse && c == 0) a.lse[row] = l == 0.0f ? -__builtin_inff() : m * kLn2 + (logf(l) + a.lse_below);
}

// What the wavefronts of a workgroup exchange at the end of a part.
struct PartLds {
  float o[kPaWaves][16][TWL_HEAD_DIM + 4];
  float m[kPaWaves][16], l[kPaWaves][16], top[16], total[16];
};

// One workgroup's part: tokens [begin, end) of a page list (first id at `ids`, `num_ids` of them)
// for kv head kvh, and 16 query rows; the four wavefronts take every fourth tile each.
// row_of(local row) -> row of q / out, or -1.
template <int QT, int KV, class RowOf>
__device__ __forceinline__ void attend_part(const PrefixAttnArgs& a, const int32_t* ids, int num_ids,
                                            int begin, int end, uint32_t kvh, RowOf row_of,
                                            uint32_t part, uint32_t parts, uint8_t* pool) {
  constexpr bool k8 = KV == TWL_I8 || KV == TWL_E4M3;
  constexpr int MT = k8 ? TWL_F16 : QT;
  constexpr int NKL = k8 ? 2 : 4;           // 16-byte loads of K per lane and page
  const int lane = lane_id(), n = lane & 15, kb = lane >> 4;
  const int wave = threadIdx.x / kWave;

  u32x4 qf[4];
  float row_scale;
  load_query<QT, k8, k8>(a, row_of(n), kb, qf, row_scale);

  f32x4 o[8];
  float m = kPaNoMax, l = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = f32x4{0, 0, 0, 0};
  int vexp = -126;                          // V scales so far are below 2^(vexp + 1)

  const uint8_t* const kbase = a.k + kvh * a.head_bytes;
  const uint8_t* const vbase = a.v + kvh * a.head_bytes;
  const uint32_t koff = n * a.token_bytes + 16 * kb;
  const uint32_t voff = 4 * kb * a.token_bytes + (k8 ? 8 : 16) * n;
  const int tiles = (end - begin + kPaTile - 1) / kPaTile;
  int window = -1, held = 0;
  struct Raw {                              // a tile as it comes from memory
    u32x4 k[2][NKL], v[8];                  // V: eight tokens, 16 bytes (16-bit) or 8 (8-bit) each
    float ks[2][4], vs[2][4];
  };
  auto fetch = [&](int t, Raw& raw) {
    // page ids come 64 at a time, one per lane (32 tiles)
    if ((t >> 5) != window) {
      window = t >> 5;
      const int at = min(begin / TWL_PAGE + window * kWave + lane, num_ids - 1);
      held = (int)min((uint32_t)ids[at], a.num_pages - 1);
    }
    const uint32_t id0 = (uint32_t)__builtin_amdgcn_readlane(held, 2 * (t & 31));
    const uint32_t id1 = (uint32_t)__builtin_amdgcn_readlane(held, 2 * (t & 31) + 1);
    const uint8_t* kp[2] = {kbase + id0 * a.page_bytes, kbase + id1 * a.page_bytes};
    const uint8_t* vp[2] = {vbase + id0 * a.page_bytes, vbase + id1 * a.page_bytes};
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < NKL; ++j) raw.k[p][j] = load_kv<u32x4>(kp[p] + koff + 64 * j);
    if (k8) {
      const float* sk = a.ks + kvh * a.scale_head;
      const float* sv = a.vs + kvh * a.scale_head;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const size_t so = (size_t)(p ? id1 : id0) * a.scale_page + 4 * kb * a.scale_token;
        if (a.scale_vec) {
          const f32x4 x = *(const f32x4*)(sk + so), y = *(const f32x4*)(sv + so);
#pragma unroll
          for (int i = 0; i < 4; ++i) { raw.ks[p][i] = x[i]; raw.vs[p][i] = y[i]; }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            raw.ks[p][i] = sk[so + i * a.scale_token];
            raw.vs[p][i] = sv[so + i * a.scale_token];
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint8_t* p = vp[i >> 2] + voff + (i & 3) * a.token_bytes;
      if (k8) {
        const u32x2 w = load_kv<u32x2>(p);
        raw.v[i].x = w.x;
        raw.v[i].y = w.y;
      } else {
        raw.v[i] = load_kv<u32x4>(p);
      }
    }
  };
  // one tile; only the last one of a part can be cut short by the end of the list
  auto step = [&](int t, const Raw& raw, auto last) {
    constexpr bool cut = decltype(last)::value;
    const int tok0 = begin + t * kPaTile;
    float ks[2][4], vs[2][4];
    u32x4 vr[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ks[i >> 2][i & 3] = raw.ks[i >> 2][i & 3];
      vs[i >> 2][i & 3] = raw.vs[i >> 2][i & 3];
      vr[i] = raw.v[i];
    }

    // ---- logits --------------------------------------------------------------------------------
    f32x4 s[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 kf;
        if (k8) {
          const u32x2 lo = widen4<KV>(raw.k[p][j >> 1][2 * (j & 1)]);
          const u32x2 hi = widen4<KV>(raw.k[p][j >> 1][2 * (j & 1) + 1]);
          kf = u32x4{lo.x, lo.y, hi.x, hi.y};
        } else {
          kf = raw.k[p][j];
        }
        s[p] = mfma16<MT>(kf, qf[j], s[p]);
      }

    if (cut) {
      // slots behind the last token hold whatever was there: their scales and V must not reach a
      // product, not even times zero
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = tok0 + 16 * (i >> 2) + 4 * kb + (i & 3) < end;
        if (k8) {
          ks[i >> 2][i & 3] = in ? ks[i >> 2][i & 3] : 0.0f;
          vs[i >> 2][i & 3] = in ? vs[i >> 2][i & 3] : 0.0f;
        }
        vr[i] = in ? vr[i] : u32x4{0, 0, 0, 0};
      }
    }
    int rise = 0;                           // how far the V exponent has to go up
    if (k8) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(vs[i >> 2][i & 3]));
      const int e = min((as_i32(top) >> 23) - 127, 126);
      if (__any(e > vexp)) {
        const int up = min((as_i32(max_over_kb(top)) >> 23) - 127, 126);
        const int e1 = __builtin_amdgcn_readfirstlane(max(up, vexp));
        rise = e1 - vexp;
        vexp = e1;
      }
      const float down = 0.5f * as_f32((127 - vexp) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) vs[i >> 2][i & 3] *= down;
    }

    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float z = k8 ? s[i >> 2][i & 3] * ks[i >> 2][i & 3] : s[i >> 2][i & 3];
      if (cut) z = tok0 + 16 * (i >> 2) + 4 * kb + (i & 3) < end ? z : -__builtin_inff();
      s[i >> 2][i & 3] = z;
      top = fmaxf(top, z);
    }
    top *= row_scale;
    if (__any(top - m > kPaRoom<MT>)) {
      const float up = raised<MT>(m, max_over_kb(top));
      const float alpha = __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= alpha;
    }
    if (k8 && rise > 0) {
      const float alpha = rise > 126 ? 0.0f : as_f32((127 - rise) << 23);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= alpha;
    }
    float w[8];
    u32x4 pf;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], row_scale, -m));
      l += w[i];
      if (k8) w[i] *= vs[i >> 2][i & 3];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[i] = pack2<MT>(w[2 * i], w[2 * i + 1]);

    // ---- O^T += V^T P^T ------------------------------------------------------------------------
    if (k8) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {         // channels 4 c .. 4 c + 3
        uint32_t by_ch[2][4];               // [tokens 0-3 / 4-7][channel], one byte per token
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t r0 = vr[4 * h][c], r1 = vr[4 * h + 1][c], r2 = vr[4 * h + 2][c], r3 = vr[4 * h + 3][c];
          const uint32_t a01 = __builtin_amdgcn_perm(r1, r0, 0x05010400u);   // r0.0 r1.0 r0.1 r1.1
          const uint32_t b01 = __builtin_amdgcn_perm(r1, r0, 0x07030602u);
          const uint32_t a23 = __builtin_amdgcn_perm(r3, r2, 0x05010400u);
          const uint32_t b23 = __builtin_amdgcn_perm(r3, r2, 0x07030602u);
          by_ch[h][0] = __builtin_amdgcn_perm(a23, a01, 0x05040100u);
          by_ch[h][1] = __builtin_amdgcn_perm(a23, a01, 0x07060302u);
          by_ch[h][2] = __builtin_amdgcn_perm(b23, b01, 0x05040100u);
          by_ch[h][3] = __builtin_amdgcn_perm(b23, b01, 0x07060302u);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x2 lo = widen4<KV>(by_ch[0][j]), hi = widen4<KV>(by_ch[1][j]);
          const u32x4 vf = {lo.x, lo.y, hi.x, hi.y};
          o[4 * c + j] = mfma16<MT>(vf, pf, o[4 * c + j]);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {         // channels 2 c, 2 c + 1
        u32x4 lo, hi;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = __builtin_amdgcn_perm(vr[2 * i + 1][c], vr[2 * i][c], 0x05040100u);
          hi[i] = __builtin_amdgcn_perm(vr[2 * i + 1][c], vr[2 * i][c], 0x07060302u);
        }
        o[2 * c] = mfma16<MT>(lo, pf, o[2 * c]);
        o[2 * c + 1] = mfma16<MT>(hi, pf, o[2 * c + 1]);
      }
    }
  };
  // the next tile is on its way while this one is worked on
  const int whole = (end - begin) / kPaTile;
  Raw cur, next;
  if (wave < tiles) fetch(wave, cur);
  for (int t = wave; t < tiles; t += kPaWaves) {
    if (t + kPaWaves < tiles) fetch(t + kPaWaves, next);
    if (t < whole) step(t, cur, Never{});
    else step(t, cur, Always{});
    cur = next;
  }

  // ---- join the wavefronts that share rows, and leave the part --------------------------------
  const float vfac = kPaUnit<MT> * (k8 ? 2.0f * as_f32((127 + vexp) << 23) : 1.0f);
  auto& lds = *(PartLds*)pool;
  l = sum_over_kb(l) * kPaUnit<MT>;
  if (kb == 0) {
    lds.m[wave][n] = m;
    lds.l[wave][n] = l;
  }
  __syncthreads();
  float top = kPaNoMax, total = 0.0f;
#pragma unroll
  for (int w = 0; w < kPaWaves; ++w) top = fmaxf(top, lds.m[w][n]);
#pragma unroll
  for (int w = 0; w < kPaWaves; ++w) total += lds.l[w][n] * __builtin_amdgcn_exp2f(lds.m[w][n] - top);
  const float f = __builtin_amdgcn_exp2f(m - top) * vfac;
  // every wavefront leaves its rows; 32 threads add and write one
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; j += 4)
      *(f32x4*)&lds.o[wave][n][32 * kb + 8 * i + j] = f32x4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]} * f;
  // the maxima and sums of the joined rows
  if (wave == 0 && kb == 0) {
    lds.top[n] = top;
    lds.total[n] = total;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < 16; r += kPaThreads / 32) {
    const int row = row_of(r);
    if (row < 0) continue;
    const int c = 4 * (threadIdx.x & 31);
    f32x4 x = *(const f32x4*)&lds.o[0][r][c];
#pragma unroll
    for (int w = 1; w < kPaWaves; ++w) x += *(const f32x4*)&lds.o[w][r][c];
    put_row<QT>(a, row, part, parts, c, x, lds.top[r], lds.total[r]);
  }
}

// The same part for many rows: 64 or 128 per workgroup (NQ sets of 16 per wavefront), whose wavefronts take
// every tile of K and V from LDS. Streaming from L2 into every wavefront's registers would need
// 16 KB of L1 traffic per 32 tokens and 32 rows, twice what the products take.
//
// Products and softmax of a tile take 3 us beside 1 us of staging (a 32768-token prompt, 256 rows: 53 us).
// Workgroups of eight wavefronts and 256 rows (half the staging) with V on its way during the softmax took
// 47 us for the prefix, but 10 instead of 4 for short own parts beside it, whose workgroups then fill half
// of a compute unit: 2 to 4 % in all, and lost for int8.
//
// Tiles of 64 tokens, two buffers: while the products of one run, the next one comes into registers; it
// is written to the other buffer after them, one barrier per tile. 8-bit pages are widened to fp16
// on that way, once per workgroup. The V operand comes out of LDS transposed (ds_read_b64_tr_b16: of the
// 4 x 16 elements that 16 lanes name, four consecutive ones each, a lane gets one column), so that
// product c takes channels 16 c .. 16 c + 15. A row of 256 bytes holds its 16 chunks of 16 bytes at place
// c ^ f(row % 16), f(r) = 2 (r % 8) + r / 8: 16 rows of one chunk, which the K operand's loads take, and eight
// rows of two neighbouring chunks, which the transposing ones take, then name every bank once. The
// counter does not go to zero for that: 2.1 M conflict cycles beside 3.2 M of LDS instructions at work (64
// samples of a 32768-token prompt), two per transposing load, whose lanes the hardware groups its own way.
constexpr int kStTile = 64;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
__device__ __forceinline__ int swizzle(int row) { return (row & 7) * 2 + ((row >> 3) & 1); }

struct StagedLds {
  u32x4 k[2][kStTile * 16], v[2][kStTile * 16];
  float ks[2][kStTile], vs[2][kStTile];
};

template <int QT, int KV, int NQ, class RowOf>
__device__ __forceinline__ void attend_staged(const PrefixAttnArgs& a, const int32_t* ids, int num_ids, int begin,
                                              int end, uint32_t kvh, int rows_here, RowOf row_of, uint32_t part,
                                              uint32_t parts, uint8_t* pool) {
  constexpr bool k8 = KV == TWL_I8 || KV == TWL_E4M3;
  constexpr int MT = k8 ? TWL_F16 : QT;
  constexpr int NL = k8 ? 2 : 4;            // 16-byte loads of K (and of V) per thread and tile
  auto& lds = *(StagedLds*)pool;
  const int tx = threadIdx.x, lane = lane_id(), n = lane & 15, kb = lane >> 4, wave = tx / kWave;
  const bool busy = wave * 16 * NQ < rows_here;   // a wavefront without rows only stages

  u32x4 qf[NQ][4];
  float row_scale[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x)
    load_query<QT, false, k8>(a, row_of((wave * NQ + x) * 16 + n), kb, qf[x], row_scale[x]);

  f32x4 o[NQ][8];
  float m[NQ], l[NQ];
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    m[x] = kPaNoMax;
    l[x] = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[x][j] = f32x4{0, 0, 0, 0};
  }
  int vexp = -126;

  const uint8_t* const kbase = a.k + kvh * a.head_bytes;
  const uint8_t* const vbase = a.v + kvh * a.head_bytes;
  const int tiles = (end - begin + kStTile - 1) / kStTile;
  // a thread's place in a page: 16-bit, one page per load; 8-bit, two pages per load
  const int tok = k8 ? (tx >> 3) & 15 : tx >> 4, chunk = k8 ? tx & 7 : tx & 15;
  const uint32_t off = tok * a.token_bytes + 16 * chunk;
  int window = -1, held = 0;
  u32x4 kraw[NL], vraw[NL];
  float sc = 0.0f;                          // wavefront 0: a scale of K, wavefront 1: of V

  // Tile t into registers, and from there into LDS.
  auto fetch = [&](int t) {
    if ((t >> 4) != window) {               // 64 page ids, 16 tiles
      window = t >> 4;
      const int at = min(begin / TWL_PAGE + window * kWave + lane, num_ids - 1);
      held = (int)min((uint32_t)ids[at], a.num_pages - 1);
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int pg = k8 ? 2 * i + __builtin_amdgcn_readfirstlane(tx >> 7) : i;
      const uint64_t id = (uint32_t)__builtin_amdgcn_readlane(held, 4 * (t & 15) + pg);
      kraw[i] = *(const u32x4*)(kbase + id * a.page_bytes + off);
      vraw[i] = *(const u32x4*)(vbase + id * a.page_bytes + off);
    }
    if (k8 && wave < 2) {                   // one scale per lane
      const uint64_t id = (uint32_t)__shfl(held, 4 * (t & 15) + (lane >> 4));
      sc = (wave ? a.vs : a.ks)[id * a.scale_page + (lane & 15) * (size_t)a.scale_token + kvh * a.scale_head];
    }
  };
  auto stage = [&](int t) {
    const int left = end - begin - t * kStTile, buf = t & 1;
    if (left < kStTile) {
      // slots behind the last token hold whatever was there and must not reach a product
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (16 * (k8 ? 2 * i + (tx >> 7) : i) + tok >= left) kraw[i] = vraw[i] = u32x4{0, 0, 0, 0};
      if (lane >= left) sc = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = 16 * (k8 ? 2 * i + (tx >> 7) : i) + tok;
      if (k8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = row * 16 + ((2 * chunk + h) ^ swizzle(tok));
          const u32x2 k0 = widen4<KV>(kraw[i][2 * h]), k1 = widen4<KV>(kraw[i][2 * h + 1]);
          lds.k[buf][at] = u32x4{k0.x, k0.y, k1.x, k1.y};
          const u32x2 v0 = widen4<KV>(vraw[i][2 * h]), v1 = widen4<KV>(vraw[i][2 * h + 1]);
          lds.v[buf][at] = u32x4{v0.x, v0.y, v1.x, v1.y};
        }
      } else {
        lds.k[buf][row * 16 + (chunk ^ swizzle(tok))] = kraw[i];
        lds.v[buf][row * 16 + (chunk ^ swizzle(tok))] = vraw[i];
      }
    }
    if (k8 && wave < 2) (wave ? lds.vs : lds.ks)[buf][lane] = sc;
  };

  // the products of 32 tokens: pages 2 h and 2 h + 1 of tile t
  auto products = [&](int t, int h, auto last) {
    constexpr bool cut = decltype(last)::value;
    const int left = end - begin - t * kStTile - 32 * h, buf = t & 1;
    const u32x4* const kt = lds.k[buf] + 512 * h;
    const u32x4* const vt = lds.v[buf] + 512 * h;
    f32x4 s[NQ][2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int x = 0; x < NQ; ++x) s[x][p] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x4 kf = kt[(16 * p + n) * 16 + ((4 * j + kb) ^ swizzle(n))];
#pragma unroll
        for (int x = 0; x < NQ; ++x) s[x][p] = mfma16<MT>(kf, qf[x][j], s[x][p]);
      }
    }
    f32x4 ks[2], vs[2];
    int rise = 0;
    if (k8) {
      const float top = wave_allreduce<OpMax>(fabsf(lds.vs[buf][32 * h + (lane & 31)]));
      const int e = max(min((as_i32(top) >> 23) - 127, 126), vexp);
      rise = e - vexp;
      vexp = e;
      const float down = 0.5f * as_f32((127 - vexp) << 23);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        ks[p] = *(const f32x4*)&lds.ks[buf][32 * h + 16 * p + 4 * kb];
        vs[p] = *(const f32x4*)&lds.vs[buf][32 * h + 16 * p + 4 * kb] * down;
      }
    }
    u32x4 pf[NQ];
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float z = k8 ? s[x][i >> 2][i & 3] * ks[i >> 2][i & 3] : s[x][i >> 2][i & 3];
        if (cut) z = 16 * (i >> 2) + 4 * kb + (i & 3) < left ? z : -__builtin_inff();
        s[x][i >> 2][i & 3] = z;
        top = fmaxf(top, z);
      }
      top *= row_scale[x];
      if (__any(top - m[x] > kPaRoom<MT>)) {
        const float up = raised<MT>(m[x], max_over_kb(top));
        const float alpha = __builtin_amdgcn_exp2f(m[x] - up);
        m[x] = up;
        l[x] *= alpha;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[x][j] *= alpha;
      }
      if (k8 && rise > 0) {
        const float alpha = rise > 126 ? 0.0f : as_f32((127 - rise) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[x][j] *= alpha;
      }
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(fmaf(s[x][i >> 2][i & 3], row_scale[x], -m[x]));
        l[x] += w[i];
        if (k8) w[i] *= vs[i >> 2][i & 3];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[x][i] = pack2<MT>(w[2 * i], w[2 * i + 1]);
    }
    // lane n names channels 16 c + 4 (n % 4) .. + 3 of token 4 kb + n / 4 of either page
    const int vrow = 4 * kb + (n >> 2), half = n & 1;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int at = vrow * 16 + ((2 * c + ((n >> 1) & 1)) ^ swizzle(vrow));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)((const uint8_t*)(vt + at) + 8 * half));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)((const uint8_t*)(vt + 256 + at) + 8 * half));
      const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
      const u32x4 vf = {l2.x, l2.y, h2.x, h2.y};
#pragma unroll
      for (int x = 0; x < NQ; ++x) o[x][c] = mfma16<MT>(vf, pf[x], o[x][c]);
    }
  };

  // tile t + 2 is asked for as soon as t + 1 has left the registers: it has a whole tile's products to arrive
  fetch(0);
  stage(0);
  if (tiles > 1) fetch(1);
  __syncthreads();
  // all tiles but the last are whole, and a tile follows them
  for (int t = 0; t + 1 < tiles; ++t) {
    if (busy) {
      products(t, 0, Never{});
      products(t, 1, Never{});
    }
    stage(t + 1);
    if (t + 2 < tiles) fetch(t + 2);
    __syncthreads();
  }
  if (busy) {
    products(tiles - 1, 0, Always{});
    products(tiles - 1, 1, Always{});
  }

  const float vfac = kPaUnit<MT> * (k8 ? 2.0f * as_f32((127 + vexp) << 23) : 1.0f);
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const float total = sum_over_kb(l[x]) * kPaUnit<MT>;
    const int row = row_of((wave * NQ + x) * 16 + n);
    if (row < 0) continue;
#pragma unroll
    for (int c = 0; c < 8; ++c) put_row<QT>(a, row, part, parts, 16 * c + 4 * kb, o[x][c] * vfac, m[x], total);
  }
}

// Kernels by the rows of a kv head that may share a prefix part: up to 16 rows are streamed, above that the
// rows that a group really has decide (a 32768-token prompt, bf16 and int8):
//   up to 16   streaming (16 rows: 36 and 27 us, through LDS 36 and 30)
//   up to 64   through LDS, 16 rows a wavefront, so that none is without rows where half of 128 are (32 rows:
//              38 and 34 us, streamed in two sets of 16 40 and 34; 48 rows: 40 and 35, with 32 rows a
//              wavefront 42 and 42)
//   above      through LDS, 32 rows a wavefront (96 rows: 47 and 44 us, in tiles of 64 46 and 52; 64 samples
//              of four q heads with up to 600 tokens of their own: 84 us and 96)
enum PrefixMode { kStream, kStaged };
constexpr int mode_rows(int mode) { return mode == kStream ? 16 : 128; }
constexpr size_t mode_lds(int mode) {
  return mode == kStream || sizeof(PartLds) > sizeof(StagedLds) ? sizeof(PartLds) : sizeof(StagedLds);
}

// Grid: the own parts (kv head, request, row tile, part: the parts that only long requests have come last),
// then the prefix parts (eight of (kv head, part, group), row tile, the next eight, ...: the row tiles of a
// part run side by side on one XCD and find its K and V in that L2). Own parts wait for memory where
// prefix parts compute, so each compute unit's first prefix part overlaps with its last own ones (64 samples
// of a 32768-token prompt, up to 4000 tokens of their own: 202 us with the prefix first, 183 so; 4 samples
// of 16384, up to 1000: 40 and 35.5; 20 of 16384, up to 100: 32 and 30).
template <int QT, int KV, int MODE>
__global__ __launch_bounds__(kPaThreads, 2) void prefix_attn_kernel(PrefixAttnArgs a) {
  __shared__ __align__(16) uint8_t pool[mode_lds(MODE)];
  const uint32_t parts = a.p_chunks + a.chunks;
  uint32_t id = blockIdx.x;
  if (id >= a.own_blocks) {
    id -= a.own_blocks;
    const uint32_t tile = (id >> 3) % a.p_tiles;
    id = (id >> 3) / a.p_tiles * 8 + (id & 7);
    const uint32_t kvh = id % a.num_kv_heads;
    id /= a.num_kv_heads;
    const uint32_t c = id % a.p_chunks, g = id / a.p_chunks;
    if (g >= a.groups) return;              // the last eight may be short
    const int first = max(a.g_ptr[g], 0);
    const int members = min(min((int)a.batch, a.g_ptr[g + 1]) - first, (int)a.max_group);
    const int rows = members * (int)a.G, row0 = (int)tile * mode_rows(MODE);
    const int len = list_len(a.p_ptr, a.p_last, g, a.max_prefix);
    const int begin = (int)(c * a.p_chunk), end = min(len, begin + (int)a.p_chunk);
    if (begin >= end || row0 >= rows) return;
    auto row_of = [&](int r) {
      const int lr = row0 + r;
      if (lr >= rows) return -1;
      const int b = lr / (int)a.G;
      return (int)((first + b) * a.num_q_heads + kvh * a.G) + lr - b * (int)a.G;
    };
    const int32_t* ids = a.p_ids + a.p_ptr[g];
    const int num_ids = a.p_ptr[g + 1] - a.p_ptr[g];
    const int here = rows - row0;
    if (MODE == kStream || here <= 16)
      attend_part<QT, KV>(a, ids, num_ids, begin, end, kvh, row_of, c, parts, pool);
    else if (here <= 64)
      attend_staged<QT, KV, 1>(a, ids, num_ids, begin, end, kvh, here, row_of, c, parts, pool);
    else
      attend_staged<QT, KV, 2>(a, ids, num_ids, begin, end, kvh, here, row_of, c, parts, pool);
  } else {
    const uint32_t kvh = id % a.num_kv_heads;
    id /= a.num_kv_heads;
    const uint32_t b = id % a.batch;
    id /= a.batch;
    const uint32_t tile = id % a.tiles, c = id / a.tiles;
    if (c >= a.chunks) return;              // the last eight may be short
    const int row0 = (int)(tile * 16);
    const int len = list_len(a.ptr, a.last, b, a.max_tokens);
    const int begin = (int)(c * a.chunk), end = min(len, begin + (int)a.chunk);
    auto row_of = [&](int r) {
      return row0 + r < (int)a.G ? (int)(b * a.num_q_heads + kvh * a.G) + row0 + r : -1;
    };
    if (begin >= end) {
      // a row of one part has nobody else to say that it sees no token
      if (parts == 1)
        for (int r = threadIdx.x >> 5; r < 16; r += kPaThreads / 32)
          if (row_of(r) >= 0)
            put_row<QT>(a, row_of(r), 0, 1, 4 * (threadIdx.x & 31), f32x4{0, 0, 0, 0}, 0.0f, 0.0f);
      return;
    }
    attend_part<QT, KV>(a, a.ids + a.ptr[b], a.ptr[b + 1] - a.ptr[b], begin, end, kvh, row_of,
                        a.p_chunks + c, parts, pool);
  }
}

// Joins the parts of a row: one workgroup per row, 32 threads per part (four channels each), eight parts
// at a time, so that the parts of a long context are not fetched one after another. Which parts exist
// follows from the lengths alone, so the workspace needs no initial contents. Where a row has at most
// one part (a prefix of one part and no own tokens, or neither) it only writes the rows that see no token.
// 4 to 5 us, a chain of loads, up to some hundred rows; 2048 rows of 33 parts (34 MB) 10 us. Asking for the
// parts before the lengths are known was no faster.
template <int QT>
__global__ __launch_bounds__(kPaThreads) void prefix_attn_merge_kernel(PrefixAttnArgs a) {
  constexpr int kLists = kPaThreads / 32;
  __shared__ float weight[2 * kPaMaxParts];
  __shared__ f32x4 sums[kLists][32];
  const uint32_t row = blockIdx.x, b = row / a.num_q_heads, parts = a.p_chunks + a.chunks;
  const int lane = lane_id(), list = threadIdx.x >> 5, c = threadIdx.x & 31;
  int np = 0;
  if (a.p_chunks) {
    const int g = group_of(a, b);
    if (g >= 0 && (int)b - max(a.g_ptr[g], 0) < (int)a.max_group)
      np = (list_len(a.p_ptr, a.p_last, g, a.max_prefix) + (int)a.p_chunk - 1) / (int)a.p_chunk;
  }
  const int no = a.chunks ? (list_len(a.ptr, a.last, b, a.max_tokens) + (int)a.chunk - 1) / (int)a.chunk : 0;
  const int count = np + no;
  if (parts <= 1 && count > 0) return;      // the part has written the row
  const size_t at = (size_t)row * parts;
  auto slot = [&](int i) { return i < np ? i : (int)a.p_chunks + i - np; };
  // every wavefront finds the maximum and the sum for itself; the first one shares the weights
  float top = kPaNoMax;
  for (int i = lane; i < count; i += kWave) top = fmaxf(top, a.ml[at + slot(i)].x);
  top = wave_allreduce<OpMax>(top);
  float l = 0.0f;
  for (int i = lane; i < count; i += kWave) {
    const f32x2 ml = a.ml[at + slot(i)];
    const float w = __builtin_amdgcn_exp2f(ml.x - top);
    l += w * ml.y;
    if (threadIdx.x < kWave) weight[i] = w;
  }
  l = wave_allreduce<OpSum>(l);
  __syncthreads();
  f32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (int i = list; i < count; i += kLists)
    acc += *(const f32x4*)(a.acc + (at + slot(i)) * TWL_HEAD_DIM + 4 * c) * weight[i];
  sums[list][c] = acc;
  __syncthreads();
  if (list > 0) return;
#pragma unroll
  for (int i = 1; i < kLists; ++i) acc += sums[i][c];
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *(u32x2*)((uint16_t*)a.out + (size_t)row * TWL_HEAD_DIM + 4 * c) =
      u32x2{pack2<QT>(acc[0] * inv, acc[1] * inv), pack2<QT>(acc[2] * inv, acc[3] * inv)};
  if (a.lse && c == 0) a.lse[row] = l == 0.0f ? -__builtin_inff() : top * kLn2 + (logf(l) + a.lse_below);
}

// How a call is cut into workgroups: from the sizes alone, the same for the workspace and the launch.
struct PrefixPlan {
  int mode;
  uint32_t p_chunk, p_chunks, p_tiles, chunk, chunks, tiles;
};

static void cut_tokens(uint32_t tokens, uint64_t others, uint32_t target, uint32_t most, uint32_t* chunk,
                       uint32_t* chunks) {
  const uint32_t least = kPaWaves * kPaTile;
  *chunk = 0;
  *chunks = 0;
  if (tokens == 0 || others == 0) return;
  uint64_t want = (target + others - 1) / others;
  if (want > kPaMaxParts) want = kPaMaxParts;
  if (want < 1) want = 1;
  uint64_t c = (tokens + want - 1) / want;
  if (c > most && (tokens + most - 1) / most <= kPaMaxParts) c = most;
  c = (c + least - 1) / least * least;
  *chunk = (uint32_t)c;
  *chunks = (uint32_t)((tokens + c - 1) / c);
}

static PrefixPlan prefix_plan(uint32_t batch, uint32_t num_q_heads, uint32_t num_kv_heads,
                              uint32_t groups, uint32_t max_prefix, uint32_t max_group,
                              uint32_t max_tokens) {
  PrefixPlan p{};
  const uint32_t G = num_q_heads / num_kv_heads;
  const uint64_t rows = (uint64_t)max_group * G;
  p.mode = rows <= 16 ? kStream : kStaged;
  p.p_tiles = (uint32_t)((rows + mode_rows(p.mode) - 1) / mode_rows(p.mode));
  p.tiles = (G + 15) / 16;
  // Prefix tokens: two workgroups per compute unit, one full load of the chip (64 samples of a 32768-token bf16
  // prompt: 256 of them 87 us, 512 73, 1024 84; 12 samples 36, 41 and 47, but 16 of int8 41 and 38, and 44
  // int8 rows of three prompts 62, 45 and 41 where their lengths differ, 80, 54 and 59 where not)
  cut_tokens(groups ? max_prefix : 0, (uint64_t)num_kv_heads * groups * p.p_tiles, 512, 1u << 24, &p.p_chunk,
             &p.p_chunks);
  // Own tokens: about two workgroups per compute unit (at 32k tokens, 8 requests, 8 kv heads: 512 of them
  // 98 us, 1024 106, 2048 105; a workgroup's start and end cost what it does not stream), but where the
  // requests alone are half of that, parts of 2048 tokens at most, since their lengths may differ (16
  // requests of up to 8191 tokens, 32 kv heads: 144 -> 121 us). Without a prefix, up to 1024 tokens are
  // one part: the merge is a launch of its own (1000 tokens: 20.6 -> 17.9 us). Beside prefix parts it runs
  // in any case and few requests are cut like longer ones (4 samples of 16384 tokens, up to 1000 of their
  // own: 35.5 -> 27 us), but 256 lists fill the chip as they are (264 of up to 300: 50.5 -> 47.5).
  const uint64_t lists = (uint64_t)num_kv_heads * batch * p.tiles;
  const bool whole = p.p_chunks ? lists >= 256 : max_tokens <= 1024;
  cut_tokens(max_tokens, whole ? 512 : lists, 512, lists < 256 ? 1u << 24 : 2048, &p.chunk, &p.chunks);
  return p;
}

template <int QT, int KV>
static void launch_prefix(const PrefixAttnArgs& a, const PrefixPlan& p, uint32_t blocks, hipStream_t st) {
#define TWL_PA(MODE) \
  hipLaunchKernelGGL((prefix_attn_kernel<QT, KV, MODE>), dim3(blocks), dim3(kPaThreads), 0, st, a)
  if (a.p_chunks == 0 || p.mode == kStream) TWL_PA(kStream);
  else TWL_PA(kStaged);
#undef TWL_PA
}

}  // namespace twl

extern "C" uint64_t twl_prefix_attn_workspace_bytes(uint32_t batch, uint32_t num_q_heads,
                                                    uint32_t num_kv_heads, uint32_t groups,
                                                    uint32_t max_prefix_tokens,
                                                    uint32_t max_group_size, uint32_t max_tokens) {
  if (batch == 0 || num_kv_heads == 0 || num_q_heads == 0 || num_q_heads % num_kv_heads != 0) return 0;
  const twl::PrefixPlan p = twl::prefix_plan(batch, num_q_heads, num_kv_heads, groups,
                                             max_prefix_tokens, max_group_size, max_tokens);
  const uint64_t parts = (uint64_t)p.p_chunks + p.chunks;
  if (parts <= 1) return 0;
  return (uint64_t)batch * num_q_heads * parts * (TWL_HEAD_DIM + 2) * sizeof(float);
}

extern "C" int twl_prefix_attn(
    const void* q, void* out, int dtype, const void* k_cache, const void* v_cache, int format,
    uint64_t page_stride, uint64_t token_stride, uint64_t head_stride, const float* k_scale,
    const float* v_scale, uint64_t scale_page_stride, uint64_t scale_token_stride,
    uint64_t scale_head_stride, uint32_t num_pages, const int32_t* prefix_page_indices,
    const int32_t* prefix_page_indptr, const int32_t* prefix_last_page_len,
    const int32_t* group_indptr, uint32_t groups, uint32_t max_prefix_tokens,
    uint32_t max_group_size, const int32_t* kv_page_indices, const int32_t* kv_page_indptr,
    const int32_t* kv_last_page_len, uint32_t max_tokens, uint32_t batch, uint32_t num_q_heads,
    uint32_t num_kv_heads, float sm_scale, float* lse_out, void* workspace,
    uint64_t workspace_bytes, void* stream) {
  const bool k8 = format == TWL_I8 || format == TWL_E4M3;
  if (!q || !out || !k_cache || !v_cache || (max_tokens && !kv_page_indices) || !kv_page_indptr || !kv_last_page_len)
    return TWL_ENULL;
  if (groups && ((max_prefix_tokens && !prefix_page_indices) || !prefix_page_indptr || !prefix_last_page_len ||
                 !group_indptr))
    return TWL_ENULL;
  if (k8 && (!k_scale || !v_scale)) return TWL_ENULL;
  if (dtype != TWL_F16 && dtype != TWL_BF16) return TWL_EDTYPE;
  if (!k8 && format != dtype) return TWL_EDTYPE;
  if (batch == 0 || num_q_heads == 0 || num_kv_heads == 0 || num_q_heads % num_kv_heads != 0 ||
      num_pages == 0 || num_pages > 0x7FFFFFFFu)
    return TWL_EINVAL;
  if ((uint64_t)batch * num_q_heads > 65535u || groups > batch) return TWL_EINVAL;
  if (groups && (max_group_size == 0 || max_group_size > batch)) return TWL_EINVAL;
  if (max_tokens > (1u << 24) || max_prefix_tokens > (1u << 24)) return TWL_EINVAL;
  if (token_stride > (1u << 24) || scale_token_stride > (1u << 24)) return TWL_EINVAL;
  if (!(sm_scale - sm_scale == 0.0f)) return TWL_EINVAL;   // infinite or NaN
  const uint64_t align = k8 ? 15u : 7u;     // 16-byte loads of a token's channels
  if ((page_stride | token_stride | head_stride) & align) return TWL_EALIGN;
  if ((((uintptr_t)q) | ((uintptr_t)k_cache) | ((uintptr_t)v_cache) | ((uintptr_t)workspace)) & 15u)
    return TWL_EALIGN;
  if ((((uintptr_t)out) & 7u) || ((((uintptr_t)k_scale) | ((uintptr_t)v_scale) | ((uintptr_t)lse_out)) & 3u))
    return TWL_EALIGN;
  if (!groups) { max_prefix_tokens = 0; max_group_size = 0; }
  const twl::PrefixPlan p = twl::prefix_plan(batch, num_q_heads, num_kv_heads, groups,
                                             max_prefix_tokens, max_group_size, max_tokens);
  const uint64_t need = twl_prefix_attn_workspace_bytes(batch, num_q_heads, num_kv_heads, groups,
                                                        max_prefix_tokens, max_group_size, max_tokens);
  if (need && !workspace) return TWL_ENULL;
  if (workspace_bytes < need) return TWL_EINVAL;
  const uint64_t p_blocks = ((uint64_t)num_kv_heads * p.p_chunks * groups + 7) / 8 * 8 * p.p_tiles;
  const uint64_t own_blocks = ((uint64_t)num_kv_heads * p.chunks * batch * p.tiles + 7) / 8 * 8;
  const uint64_t blocks = p_blocks + own_blocks;
  if (blocks > 0xFFFFFFull) return TWL_EINVAL;   // 2^32 threads
  const uint64_t parts = (uint64_t)p.p_chunks + p.chunks, rows = (uint64_t)batch * num_q_heads;
  twl::PrefixAttnArgs a{};
  const uint64_t eb = k8 ? 1 : 2;
  a.q = (const uint16_t*)q; a.out = out; a.lse = lse_out; a.k = (const uint8_t*)k_cache;
  a.v = (const uint8_t*)v_cache; a.page_bytes = page_stride * eb; a.head_bytes = head_stride * eb;
  a.token_bytes = (uint32_t)(token_stride * eb); a.ks = k_scale; a.vs = v_scale;
  a.scale_page = scale_page_stride; a.scale_head = scale_head_stride;
  a.scale_token = (uint32_t)scale_token_stride;
  a.scale_vec = scale_token_stride == 1 && ((scale_page_stride | scale_head_stride) & 3u) == 0 &&
                ((((uintptr_t)k_scale) | ((uintptr_t)v_scale)) & 15u) == 0;
  a.num_pages = num_pages;
  a.p_ids = prefix_page_indices; a.p_ptr = prefix_page_indptr; a.p_last = prefix_last_page_len;
  a.g_ptr = group_indptr; a.ids = kv_page_indices; a.ptr = kv_page_indptr; a.last = kv_last_page_len;
  a.batch = batch; a.num_q_heads = num_q_heads; a.num_kv_heads = num_kv_heads;
  a.G = num_q_heads / num_kv_heads; a.groups = groups; a.max_prefix = max_prefix_tokens;
  a.max_group = max_group_size; a.max_tokens = max_tokens; a.p_chunk = p.p_chunk;
  a.p_chunks = p.p_chunks; a.p_tiles = p.p_tiles; a.chunk = p.chunk; a.chunks = p.chunks;
  a.tiles = p.tiles; a.own_blocks = (uint32_t)own_blocks;
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.lse_below = (k8 || dtype == TWL_F16 ? twl::kPaBelow<TWL_F16> : twl::kPaBelow<TWL_BF16>) * twl::kLn2;
  a.acc = (float*)workspace;
  a.ml = (twl::f32x2*)((float*)workspace + rows * parts * TWL_HEAD_DIM);
  hipStream_t st = (hipStream_t)stream;
  if (blocks) {
    if (dtype == TWL_F16) {
      if (format == TWL_I8) twl::launch_prefix<TWL_F16, TWL_I8>(a, p, (uint32_t)blocks, st);
      else if (format == TWL_E4M3) twl::launch_prefix<TWL_F16, TWL_E4M3>(a, p, (uint32_t)blocks, st);
      else twl::launch_prefix<TWL_F16, TWL_F16>(a, p, (uint32_t)blocks, st);
    } else {
      if (format == TWL_I8) twl::launch_prefix<TWL_BF16, TWL_I8>(a, p, (uint32_t)blocks, st);
      else if (format == TWL_E4M3) twl::launch_prefix<TWL_BF16, TWL_E4M3>(a, p, (uint32_t)blocks, st);
      else twl::launch_prefix<TWL_BF16, TWL_BF16>(a, p, (uint32_t)blocks, st);
    }
    if (hipGetLastError() != hipSuccess) return TWL_ELAUNCH;
  }
  if (p.p_chunks == 0 && p.chunks == 1) return TWL_OK;   // every row is written by its one part
  const dim3 mgrid((uint32_t)rows);
  if (dtype == TWL_F16)
    hipLaunchKernelGGL((twl::prefix_attn_merge_kernel<TWL_F16>), mgrid, dim3(twl::kPaThreads), 0, st, a);
  else
    hipLaunchKernelGGL((twl::prefix_attn_merge_kernel<TWL_BF16>), mgrid, dim3(twl::kPaThreads), 0, st, a);
  return hipGetLastError() == hipSuccess ? TWL_OK : TWL_ELAUNCH;
}
