// The next token of every row of logits, drawn with one given uniform number.
//
// Tokens are ranked by logit, the larger first and equal ones by index. With T the temperature and
// x* the largest logit, w = exp((x - x*) / T). A token is kept if
//   top-k   its rank is below k,
//   top-p   the summed w of the better ranks is below p times the summed w of the top-k,
//   min-p   w >= min_p,
// in this order; the first rank always is. The answer is the first token, in the order of the
// vocabulary, whose running sum of kept w exceeds u times the sum of all kept w.
//
// Sums decide, so they must not depend on their order: w is computed in 64 bits and held as a
// multiple of 2^-45 in 64-bit integers, whose sums are exact (2^18 tokens of weight 1 fill 63
// bits). What is lost is below 2^-46 of the best token's weight, per token: a token more than 32 T
// below the best weighs nothing.
//
// No row is sorted. Three launches, the first two with several workgroups (slices) per row so that a
// small batch fills the chip (w costs about twenty 64-bit operations per token, which a single
// compute unit would be at for most of the time):
//   hist  Every slice finds its largest logit and, relative to that, adds up w (top-p, in 32 bits) or
//         counts tokens (top-k) in 512 bins of width T / 16. A bin is floor(16 x / T), so bins of
//         different slices are the same intervals and the slices' sums join after one rescaling each.
//   keep  Every slice joins its row's bins and finds the one that holds the cut. With top-p these are
//         approximate sums: where a bin ends within their error of the cut, the next one may hold it too.
//         Tokens above are kept: their w goes into sums over 512 consecutive tokens, and the tokens of
//         the cut's bin or bins become candidates. On the way every w, relative to the row's best token, is
//         added up exactly: what top-p reaches for. With top-k, all tokens down to the cut bin are
//         candidates.
//   pick  One workgroup per row finds the exact cut among the candidates, digit by digit of the logit's
//         ordered bit pattern (then of the index, where equal logits are cut), adds the kept ones to
//         the sums and draws.
// A row whose candidates do not fit (more than kSmpMaxCand tokens within T / 16 of the cut) is done by
// pick alone, digit by digit over the whole row.
//
// Not bound by memory (64 bf16 rows of 128256: 16 MB, 3 us): hist by the atomics and the weights of every token (11
// us there, 14 with weights in 64 bits), keep by their 64-bit weights (19.5; 18 when it weighed kept tokens only
// and took the mass to reach from the bins, so that the cut could depend on how a batch is sliced), pick by
// its chain of sums and by fetching code that is used once (14 us). One row of 32000: 4, 7 and 7 us. Logits
// read a second time in a loop, instead of kept in registers through unrolled code, cost hist and keep 1 and 2
// us; copies of hist's bins against atomics on one address changed nothing.
#include "twl_common.h"

namespace twl {

constexpr int kSmpThreads = 512;
constexpr int kSmpWaves = kSmpThreads / kWave;
constexpr uint32_t kSmpMaxVocab = 1u << 18;
constexpr double kSmpOne = 35184372088832.0;   // 2^45: the weight 1
constexpr int kSmpBins = 512;
constexpr int kSmpSeg = 512;                   // tokens of one running sum: a wavefront, 8 a lane
constexpr int kSmpStep = kSmpThreads * 8;      // tokens of one pass of a workgroup
constexpr uint32_t kSmpMaxCand = 8192;
constexpr double kSmpHistError = 1.0 / (1 << 18);   // of a row's mass, what the bins' sums may be off by,
constexpr double kSmpSumError = 1.0 / (1ull << 45); // and in 64 bits: some 80 roundings of 2^-53

struct SampleArgs {
  const void* logits;
  uint64_t row_stride;
  uint32_t rows, vocab;
  const float* u;
  const float* temperature;   // [rows] or NULL: the value below for every row
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* tokens;
  // workspace
  uint32_t slices, iters;     // slices of iters * kSmpStep tokens
  uint64_t* best;             // [rows, slices]  key, then the lowest index
  uint64_t* hist;             // [rows, slices, kSmpBins]
  uint64_t* seg;              // [rows, segments]
  uint64_t* cand;             // [rows, cand_stride]  key, then the complement of the index
  uint32_t cand_stride;       // min(kSmpMaxCand, vocab)
  struct SampleCut* cut;      // [rows]
  uint32_t* cand_count;       // [rows]
  uint64_t* mass;             // [rows, slices, 2]  summed w of all tokens, and of those above the cut's bin
};

// What keep leaves for pick. Tokens from `keep` up are kept, those from `cand` up to there are
// candidates (a NaN: there are none).
struct SampleCut {
  float keep, cand;
};

// NaN counts as masked; -0 ranks as +0
__device__ __forceinline__ float masked_logit(float x) { return fmaxf(x, -__builtin_inff()) + 0.0f; }
template <int DT>
__device__ __forceinline__ float logit_at(const SampleArgs& a, uint32_t row, uint32_t i) {
  float x;
  if (DT == TWL_F32) x = ((const float*)a.logits)[row * a.row_stride + i];
  else x = bits16_to_f32<DT>(((const uint16_t*)a.logits)[row * a.row_stride + i]);
  return masked_logit(x);
}
// Eight consecutive logits from i on; -inf behind the vocabulary.
template <int DT>
__device__ __forceinline__ void logits8(const SampleArgs& a, uint32_t row, uint32_t i, float* x) {
  constexpr int kBytes = DT == TWL_F32 ? 4 : 2;
  const uint8_t* p = (const uint8_t*)a.logits + (row * a.row_stride + i) * kBytes;
  if (i + 8 <= a.vocab && (((uintptr_t)p) & 15u) == 0) {
    if (DT == TWL_F32) {
      const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) { x[j] = lo[j]; x[4 + j] = hi[j]; }
    } else {
      unpack8<DT>(*(const u32x4*)p, x);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = masked_logit(x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < a.vocab ? logit_at<DT>(a, row, i + j) : -__builtin_inff();
  }
}
// order-preserving bit pattern, and back
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = as_u32(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return as_f32(key ^ (~(uint32_t)((int32_t)key >> 31) | 0x80000000u));
}
constexpr uint32_t kKeyNone = 0x007FFFFFu;     // key_of(-inf)

// ---- 64-bit values across a wavefront, by DPP (a scan step is a few cycles; through LDS it is a
// hundred) ------------------------------------------------------------------------------------
template <int CTRL, int ROW_MASK, class T>
__device__ __forceinline__ T dpp64(T v) {        // 0 where there is no source
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)dpp<CTRL, ROW_MASK>(0, (int)(uint32_t)u);
  const uint32_t hi = (uint32_t)dpp<CTRL, ROW_MASK>(0, (int)(uint32_t)(u >> 32));
  return __builtin_bit_cast(T, ((uint64_t)hi << 32) | lo);
}
template <class T>
__device__ __forceinline__ T lane63(T v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __builtin_bit_cast(T, ((uint64_t)hi << 32) | lo);
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {    // inclusive, in lane order
  T t;
  t = dpp64<0x111, 0xF>(v); v += t;
  t = dpp64<0x112, 0xF>(v); v += t;
  t = dpp64<0x114, 0xF>(v); v += t;
  t = dpp64<0x118, 0xF>(v); v += t;
  t = dpp64<kDppBcast15, 0xA>(v); v += t;
  t = dpp64<kDppBcast31, 0xC>(v); v += t;
  return v;
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return lane63(wave_scan(v)); }
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  v = max(v, dpp64<0x111, 0xF>(v));
  v = max(v, dpp64<0x112, 0xF>(v));
  v = max(v, dpp64<0x114, 0xF>(v));
  v = max(v, dpp64<0x118, 0xF>(v));
  v = max(v, dpp64<kDppBcast15, 0xA>(v));
  v = max(v, dpp64<kDppBcast31, 0xC>(v));
  return lane63(v);
}
__device__ __forceinline__ uint32_t wave_max32(uint32_t v) {
  v = max(v, (uint32_t)dpp<0x111>(0, (int)v));
  v = max(v, (uint32_t)dpp<0x112>(0, (int)v));
  v = max(v, (uint32_t)dpp<0x114>(0, (int)v));
  v = max(v, (uint32_t)dpp<0x118>(0, (int)v));
  v = max(v, (uint32_t)dpp<kDppBcast15, 0xA>(0, (int)v));
  v = max(v, (uint32_t)dpp<kDppBcast31, 0xC>(0, (int)v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// How a row is filtered.
struct RowFilter {
  double T, p, min_p;
  int32_t k;
  bool greedy, by_rank, by_mass;   // the best token only; top-k cuts; top-p cuts (and no top-k)
  bool fine;                       // bins are summed in 64 bits
};
__device__ __forceinline__ RowFilter row_filter(const SampleArgs& a, uint32_t row) {
  RowFilter f;
  const float T = a.temperature ? a.temperature[row] : a.temperature_all;
  f.T = fmin((double)T, 1e300);                 // finite: a masked logit has weight 0 at every T
  f.p = a.top_p ? a.top_p[row] : a.top_p_all;
  f.min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  f.k = a.top_k ? a.top_k[row] : a.top_k_all;
  f.greedy = !(T > 0.0f) || f.k == 1;
  f.by_rank = f.k > 0 && (uint32_t)f.k < a.vocab;
  f.by_mass = !f.by_rank && f.p < 1.0;
  // temperatures whose reciprocal 32 bits do not hold, or no longer times a masked logit, and cuts so near the end
  // that the bins' error in 32 bits would make candidates of the whole tail
  f.fine = !(f.T > 1e-18 && f.T < 1e18) || f.p > 0.9999;
  return f;
}

// a * b + c with c a constant of the scalar registers (the compiler takes the two-address form and
// refills its accumulator with the constant each time)
__device__ __forceinline__ double fma_const(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// w in units of 2^-45 and its fixed-point form, for logits relative to `top`. With
// z = 64 (x - top) log2(e) / T:
//   2^(z / 64) = 2^(n >> 6) * 2^((n & 63) / 64) * 2^(f / 64),   n = rint(z),  |f| <= 1/2
// with the middle factor from a table and the last from its series to the fifth power in f
// (next term (ln 2 / 128)^6 / 720 < 4e-17).
struct Weigher {
  const double* table;        // LDS, 2^(45 + i / 64)
  double top, per;            // per = 64 log2(e) / T
  bool endless;               // the largest logit is infinite: it weighs 1, the others nothing
  __device__ __forceinline__ Weigher(const double* t, float best, double T)
      : table(t), top(best), per(92.3324826168936580 / T), endless(best == __builtin_inff()) {}
  // any x where `endless` is not set. Rounding by adding 1.5 * 2^52 and scaling in the exponent field:
  // the instructions made for either run at a quarter of an addition's rate
  __device__ __forceinline__ double scaled(float x) const {
    const double z = fmax(((double)x - top) * per, -4096.0);   // 2^-19 units for all that is further down
    const double t = z + 6755399441055744.0;
    const uint32_t i = (uint32_t)__builtin_bit_cast(uint64_t, t);
    const double f = z - (t - 6755399441055744.0);
    constexpr double c = 0.693147180559945309417 / 64;
    double y = fma_const(f, c * c * c * c * c / 120, c * c * c * c / 24);
    y = fma_const(f, y, c * c * c / 6);
    y = fma_const(f, y, c * c / 2);
    y = fma_const(f, y, c);
    y = fma(f, y, 1.0) * table[i & 63];
    const uint64_t b = __builtin_bit_cast(uint64_t, y);
    return __builtin_bit_cast(double, ((uint64_t)((uint32_t)(b >> 32) + ((i & ~63u) << 14)) << 32) | (uint32_t)b);
  }
  __device__ __forceinline__ double weight(float x) const {     // in units of 2^-45
    if (endless) return x == __builtin_inff() ? kSmpOne : 0.0;
    return scaled(x);
  }
  static __device__ __forceinline__ uint64_t fixed(double w) {
    // adding 2^52 leaves the nearest integer in the low bits
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) - 0x4330000000000000ull;
  }
  __device__ __forceinline__ uint64_t mass(float x) const { return fixed(weight(x)); }
};
__device__ const double kPow2[64] = {   // 2^(i / 64), rounded to nearest
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};
__device__ __forceinline__ void fill_table(double* table) {
  if (threadIdx.x < 64) table[threadIdx.x] = kPow2[threadIdx.x] * kSmpOne;
}

// Bins of width T / 16 from the best token's down: monotone in x, the same intervals for every slice.
struct Binner {
  float per;
  __device__ __forceinline__ int bin(float x) const {
    int b;                                        // floor and conversion in one; saturates
    asm("v_cvt_flr_i32_f32 %0, %1" : "=v"(b) : "v"(x * per));
    return b;
  }
  // The least logit of bin b or above (NaN: no logit is), so that a pass over the tokens compares instead
  // of binning: by halving, on the ordered bit patterns, an interval around the quotient or else all
  __device__ __forceinline__ float edge(int64_t b) const {
    if (b > 0x7FFFFFFFll) return __builtin_nanf("");
    uint32_t lo = key_of(-__FLT_MAX__), hi = key_of(__FLT_MAX__);
    if (b <= -0x80000000ll || bin(key_value(lo)) >= (int)b) return -__FLT_MAX__;
    if (bin(key_value(hi)) < (int)b) return __builtin_inff();
    const uint32_t near = key_of(fminf(fmaxf((float)b / per, -1e38f), 1e38f));
    if (bin(key_value(near - 32)) < (int)b && bin(key_value(near + 32)) >= (int)b) {
      lo = near - 32;
      hi = near + 32;
    }
    while (hi - lo > 1) {                 // bin(lo) < b <= bin(hi)
      const uint32_t mid = lo + (hi - lo) / 2;
      if (bin(key_value(mid)) >= (int)b) hi = mid;
      else lo = mid;
    }
    return key_value(hi);
  }
  // bins from the best token's down: a huge number, as unsigned, where the difference leaves 32 bits
  __device__ __forceinline__ uint32_t below(int top_bin, float x) const { return (uint32_t)top_bin - (uint32_t)bin(x); }
};
__device__ __forceinline__ Binner binner(const RowFilter& f) {
  // bounded away from 0 and infinity, either of which could make a NaN of a logit
  return Binner{fminf(fmaxf((float)(16.0 / f.T), 1e-37f), 1e30f)};
}

// ---- first launch ------------------------------------------------------------------------------
template <int DT, int ITERS>
__global__ __launch_bounds__(kSmpThreads) void sample_hist_kernel(SampleArgs a) {
  __shared__ uint64_t hist[kSmpBins];
  __shared__ uint32_t wbest[kSmpWaves], wat[kSmpWaves];
  __shared__ double table[64];
  const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const uint32_t first = slice * (ITERS * kSmpStep) + threadIdx.x * 8;
  float x[ITERS][8];
#pragma unroll
  for (int t = 0; t < ITERS; ++t) logits8<DT>(a, row, first + t * kSmpStep, x[t]);
  const RowFilter f = row_filter(a, row);
  for (int i = threadIdx.x; i < kSmpBins; i += kSmpThreads) hist[i] = 0;
  fill_table(table);
  float m = -__builtin_inff();
#pragma unroll
  for (int t = 0; t < ITERS; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, x[t][j]);
  const uint32_t mine = wave_max32(key_of(m));
  if (lane_id() == 0) wbest[threadIdx.x / kWave] = mine;
  __syncthreads();
  uint32_t key = 0;
#pragma unroll
  for (int w = 0; w < kSmpWaves; ++w) key = max(key, wbest[w]);
  const size_t out = (size_t)row * a.slices + slice;
  if (f.greedy) {
    // where it is first
    uint32_t at = 0xFFFFFFFFu;
#pragma unroll
    for (int t = ITERS - 1; t >= 0; --t)
#pragma unroll
      for (int j = 7; j >= 0; --j)
        if (key_of(x[t][j]) == key) at = first + t * kSmpStep + j;
    const uint32_t inv = wave_max32(0xFFFFFFFFu - at);
    if (lane_id() == 0) wat[threadIdx.x / kWave] = inv;
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t b = 0;
      for (int w = 0; w < kSmpWaves; ++w) b = max(b, wat[w]);
      a.best[out] = ((uint64_t)key << 32) | b;
    }
    return;
  }
  if (threadIdx.x == 0) {
    a.best[out] = (uint64_t)key << 32;
    if (slice == 0) a.cand_count[row] = 0;
  }
  if (!(f.by_rank || f.by_mass) || key <= kKeyNone) return;
  const float top = key_value(key);
  const Weigher wt(table, top, f.T);
  const Binner bn = binner(f);
  const int top_bin = bn.bin(top);
  if (f.by_rank || wt.endless || f.fine) {
#pragma unroll
    for (int t = 0; t < ITERS; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t rel = bn.below(top_bin, x[t][j]);
        if (rel < kSmpBins && x[t][j] > -__builtin_inff())
          atomicAdd((unsigned long long*)&hist[rel], f.by_rank ? 1ull : (unsigned long long)wt.mass(x[t][j]));
      }
  } else {
    // w in 32 bits, as a multiple of 2^-45. Off by 1.5 |z| 2^-23 ln 2 + 2^-22 of itself, z = log2 w: the roundings of
    // the difference, the factor and the product, and the exponential's. |z| averages at most log2 of the
    // tokens over the mass of a row, 18, so that sums are off by 21 * 2^-23 of the row's mass (kSmpHistError)
    const float per = (float)(1.44269504088896341 / f.T);
#pragma unroll
    for (int t = 0; t < ITERS; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t rel = bn.below(top_bin, x[t][j]);
        const float w = __builtin_amdgcn_exp2f((x[t][j] - top) * per) * (float)kSmpOne;
        const uint64_t v = Weigher::fixed((double)w);
        if (rel < kSmpBins) atomicAdd((unsigned long long*)&hist[rel], (unsigned long long)v);
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kSmpBins; i += kSmpThreads) a.hist[out * kSmpBins + i] = hist[i];
}

// the best token of slice `lane` of a row (0: no such slice); there are at most kWave
__device__ __forceinline__ uint64_t slice_best(const SampleArgs& a, uint32_t row) {
  const uint32_t s = lane_id();
  return s < a.slices ? a.best[(size_t)row * a.slices + s] : 0ull;
}

// ---- second launch -----------------------------------------------------------------------------
// 128 registers at most, or a compute unit holds one workgroup instead of two (64 rows of 128256: 26 us so, 19.5)
template <int DT, int ITERS>
__global__ __launch_bounds__(kSmpThreads, 4) void sample_keep_kernel(SampleArgs a) {
  static_assert(kSmpBins == kSmpThreads, "one bin per thread");
  __shared__ uint64_t list[kSmpMaxCand];
  __shared__ double wsum[kSmpWaves], table[64];
  __shared__ int slice_shift[64];
  __shared__ double slice_weight[64];
  __shared__ uint64_t wmass[kSmpWaves][2];
  __shared__ int cut_bin, sure_bin;         // the last bin that the cut may be in, and the first
  __shared__ float cut_keep, cut_cand;
  __shared__ uint32_t list_n, list_at;
  const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
  const uint32_t first = slice * (ITERS * kSmpStep) + threadIdx.x * 8;
  float x[ITERS][8];
#pragma unroll
  for (int t = 0; t < ITERS; ++t) logits8<DT>(a, row, first + t * kSmpStep, x[t]);
  const uint64_t mine_best = slice_best(a, row);
  fill_table(table);
  const RowFilter f = row_filter(a, row);
  const uint32_t top_key = (uint32_t)(wave_max(mine_best) >> 32);
  if (f.greedy || top_key <= kKeyNone) return;
  const float top = key_value(top_key);
  const Binner bn = binner(f);
  const int top_bin = bn.bin(top);
  if (threadIdx.x == 0) {
    list_n = 0;
    cut_bin = sure_bin = kSmpBins - 1;
    cut_keep = -__FLT_MAX__;              // without a cut: everything but -inf, and no candidates
    cut_cand = __builtin_nanf("");
  }
  __syncthreads();
  const Weigher wt(table, top, f.T);
  if (f.by_rank || f.by_mass) {
    // this thread's bin of the row, from the slices in order: their shifts and weights first, by one
    // thread each, so that the loads of the bins do not wait for one another
    if (threadIdx.x < a.slices) {
      const uint32_t key = (uint32_t)(mine_best >> 32);
      const float stop = key_value(key);
      const bool used = key > kKeyNone;
      slice_shift[threadIdx.x] = used ? (int)min(bn.below(top_bin, stop), (uint32_t)kSmpBins) : kSmpBins;
      slice_weight[threadIdx.x] = !used ? 0.0 : f.by_rank ? 1.0 : wt.weight(stop) / kSmpOne;
    }
    __syncthreads();
    double v = 0.0;
    const uint64_t* const bins = a.hist + (size_t)row * a.slices * kSmpBins;
    // eight loads at a time; every one is used, if with weight 0, or the compiler makes branches of them
    // that wait for one another (one row of 128256 in 32 slices: 33 us so, 27 like this)
    for (uint32_t s0 = 0; s0 < a.slices; s0 += 8) {
      uint64_t h[8];
      double w[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t s = min(s0 + j, a.slices - 1);
        const int mine = (int)threadIdx.x - slice_shift[s];
        h[j] = bins[s * kSmpBins + max(mine, 0)];
        w[j] = mine >= 0 && s0 + j < a.slices ? slice_weight[s] : 0.0;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v += (double)h[j] * w[j];
    }
    const int wave = threadIdx.x / kWave;
    const double incl = wave_scan(v);
    if (lane_id() == kWave - 1) wsum[wave] = incl;
    __syncthreads();
    double off = 0.0, total = 0.0;
#pragma unroll
    for (int w = 0; w < kSmpWaves; ++w) {
      if (w < wave) off += wsum[w];
      total += wsum[w];
    }
    // the first bin whose running sum reaches the goal. Counts are exact; with masses, the first that may and the
    // first that surely does. Two units per token are the roundings of its w here and in the exact sums
    const double goal = f.by_mass ? f.p * total : (double)f.k, after = off + incl;
    const double off_by = !f.by_mass ? 0.0 : total * (f.fine ? kSmpSumError : kSmpHistError) + 2.0 * (double)a.vocab;
    const uint64_t sure = __ballot(after >= goal - off_by && v > 0.0);
    const uint64_t hit = __ballot(after >= goal + off_by && v > 0.0);
    if (sure && lane_id() == __builtin_ctzll(sure)) atomicMin(&sure_bin, (int)threadIdx.x);
    if (hit && lane_id() == __builtin_ctzll(hit)) atomicMin(&cut_bin, (int)threadIdx.x);
    __syncthreads();
    if (threadIdx.x < 2) {
      const float e = bn.edge((int64_t)top_bin - (threadIdx.x == 0 ? cut_bin : sure_bin - 1));
      if (threadIdx.x == 0) cut_cand = e;
      else cut_keep = f.by_rank ? __builtin_nanf("") : e;
    }
    __syncthreads();
  }
  const float keep = cut_keep, cand = cut_cand;
  if (slice == 0 && threadIdx.x == 0) a.cut[row] = SampleCut{keep, cand};
  // candidates first: their place in the row's list is a round trip that the weights can hide
  uint32_t hits[ITERS];                   // bit j: token j of the eight is a candidate
#pragma unroll
  for (int t = 0; t < ITERS; ++t) {
    hits[t] = 0;
    if (cand == cand) {
#pragma unroll
      for (int j = 0; j < 8; ++j) hits[t] |= x[t][j] >= cand && !(x[t][j] >= keep) ? 1u << j : 0u;
      if (__any(hits[t] != 0)) {
        const int n = __builtin_popcount(hits[t]), incl = wave_inclusive_scan(n);
        int base = 0;
        if (lane_id() == kWave - 1) base = (int)atomicAdd(&list_n, (uint32_t)incl);
        uint32_t at = (uint32_t)(__builtin_amdgcn_readlane(base, kWave - 1) + incl - n);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (hits[t] & (1u << j)) {
            if (at < kSmpMaxCand)
              list[at] = ((uint64_t)key_of(x[t][j]) << 32) | (0xFFFFFFFFu - (first + t * kSmpStep + j));
            ++at;
          }
      }
    }
  }
  __syncthreads();
  const uint32_t n = list_n;
  uint32_t row_at = 0;
  if (threadIdx.x == 0 && n > 0) row_at = atomicAdd(&a.cand_count[row], n);
  if (!f.by_rank) {
    const double min_w = f.min_p > 0.0 ? f.min_p * kSmpOne : -1.0;
    const uint32_t segs = (a.vocab + kSmpSeg - 1) / kSmpSeg;
    // FILTERED: min-p is in use, and the mass above the cut's bin is not that of the kept tokens
    auto sums = [&](auto weigh, auto filtered) {
      constexpr bool FILTERED = decltype(filtered)::value;
      uint64_t all = 0, above = 0;
#pragma unroll
      for (int t = 0; t < ITERS; ++t) {
        uint64_t mine = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float y = x[t][j];
          asm("" : "+v"(y));                // or what the three uses share is computed before them and fills registers
          const double w = weigh(y);
          const uint64_t v = Weigher::fixed(w);
          all += v;
          if (FILTERED) above += y >= keep ? v : 0;
          mine += y >= keep && (!FILTERED || w >= min_w || y == top) ? v : 0;
        }
        const uint64_t s = wave_sum(mine);
        const uint32_t g = (first + t * kSmpStep) / kSmpSeg;
        if (lane_id() == 0 && g < segs) a.seg[(size_t)row * segs + g] = s;
        if (!FILTERED) above += s;
      }
      all = wave_sum(all);
      if (FILTERED) above = wave_sum(above);
      if (lane_id() == 0) {
        wmass[threadIdx.x / kWave][0] = all;
        wmass[threadIdx.x / kWave][1] = above;
      }
    };
    if (wt.endless) sums([&](float y) { return wt.weight(y); }, Always{});
    else if (f.min_p > 0.0) sums([&](float y) { return wt.scaled(y); }, Always{});
    else sums([&](float y) { return wt.scaled(y); }, Never{});
  }
  if (threadIdx.x == 0) list_at = row_at;
  __syncthreads();
  if (f.by_mass && threadIdx.x < 2) {
    uint64_t sum = 0;
#pragma unroll
    for (int w = 0; w < kSmpWaves; ++w) sum += wmass[w][threadIdx.x];
    a.mass[((size_t)row * a.slices + slice) * 2 + threadIdx.x] = sum;
  }
  for (uint32_t i = threadIdx.x; i < min(n, kSmpMaxCand); i += kSmpThreads)
    if (list_at + i < a.cand_stride) a.cand[(size_t)row * a.cand_stride + list_at + i] = list[i];
}

// ---- third launch ------------------------------------------------------------------------------
// Sums by digit are kept in copies, one per lane of 16: equal logits are common (a bf16 logit near 4 has 16
// of them per unit) and atomics on one address go one after another.
constexpr int kSmpDigitBits = 7, kSmpCopies = 16, kSmpSlots = kSmpCopies << kSmpDigitBits;
struct SampleShared {
  uint64_t list[kSmpMaxCand];           // key, then the complement of the index: larger is better ranked
  uint64_t seg[kSmpMaxVocab / kWave];   // generic: measure of every 64 tokens; else of every kSmpSeg
  uint64_t hist[kSmpSlots];
  uint32_t count[kSmpSlots];
  uint64_t left[kWave][2], before[kWave];
  uint64_t wsum[kSmpWaves], wmin[kSmpWaves];
  double table[64];
  uint32_t word[2], members;
  uint64_t wide[2];
};
// Sum of measure(i) over the row, by 64 tokens in sh.seg.
template <class F>
__device__ __forceinline__ uint64_t measure_row(SampleShared& sh, uint32_t vocab, F measure) {
  const int wave = threadIdx.x / kWave;
  uint64_t mine = 0;
  for (uint32_t i0 = 0; i0 < vocab; i0 += kSmpThreads) {
    const uint32_t i = i0 + threadIdx.x;
    const uint64_t s = wave_sum(i < vocab ? measure(i) : 0ull);
    if (lane_id() == 0 && i < vocab) sh.seg[i / kWave] = s;
    mine += s;
  }
  if (lane_id() == 0) sh.wsum[wave] = mine;
  __syncthreads();
  uint64_t total = 0;
  for (int w = 0; w < kSmpWaves; ++w) total += sh.wsum[w];
  __syncthreads();
  return total;
}
// First i whose running measure exceeds `target` (< the total), after measure_row.
template <class F>
__device__ __forceinline__ uint32_t first_beyond(SampleShared& sh, uint32_t vocab, uint64_t target, F measure) {
  const uint32_t segs = (vocab + kWave - 1) / kWave;
  const int wave = threadIdx.x / kWave;
  uint64_t before = 0;                  // measure of the segments in front of these
  for (uint32_t s0 = 0; s0 < segs; s0 += kSmpThreads) {
    const uint32_t s = s0 + threadIdx.x;
    const uint64_t m = s < segs ? sh.seg[s] : 0ull;
    const uint64_t incl = wave_scan(m);
    if (lane_id() == kWave - 1) sh.wsum[wave] = incl;
    __syncthreads();
    uint64_t off = before, all = before;
    for (int w = 0; w < kSmpWaves; ++w) {
      if (w < wave) off += sh.wsum[w];
      all += sh.wsum[w];
    }
    if (off + incl > target && off + incl - m <= target) {   // one thread of the row
      sh.word[0] = s;
      sh.wide[0] = off + incl - m;
    }
    __syncthreads();
    before = all;
    if (all > target) break;
  }
  if (wave == 0) {
    const uint32_t i = sh.word[0] * kWave + lane_id();
    const uint64_t m = i < vocab ? measure(i) : 0ull;
    const uint64_t incl = wave_scan(m) + sh.wide[0];
    const uint64_t beyond = __ballot(incl > target);
    if (lane_id() == 0) sh.word[1] = sh.word[0] * kWave + (beyond ? __builtin_ctzll(beyond) : 0);
  }
  __syncthreads();
  const uint32_t got = sh.word[1];
  __syncthreads();
  return got;
}

// The key at which the running measure, from the largest key down, first reaches `target` (>= 1,
// <= the total), and the measure of the keys above it. measure(i, key): 0 for tokens left out.
template <class F>
__device__ __forceinline__ uint32_t key_reaching(SampleShared& sh, uint32_t vocab, uint64_t target, F measure,
                                                 uint64_t& above) {
  uint32_t prefix = 0;
  above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) sh.hist[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < vocab; i += kSmpThreads) {
      uint32_t key;
      const uint64_t m = measure(i, key);
      if (m && (shift == 24 || (key >> (shift + 8)) == prefix))
        atomicAdd((unsigned long long*)&sh.hist[(key >> shift) & 255], (unsigned long long)m);
    }
    __syncthreads();
    if (threadIdx.x < kWave) {          // lane 0 holds the four largest digits
      const int lane = lane_id();
      uint64_t m[4], s = 0;
      for (int j = 0; j < 4; ++j) s += m[j] = sh.hist[255 - (4 * lane + j)];
      uint64_t run = wave_scan(s) - s + above;
      for (int j = 0; j < 4; ++j) {
        if (run < target && run + m[j] >= target) {
          sh.word[0] = 255 - (4 * lane + j);
          sh.wide[0] = run;
        }
        run += m[j];
      }
    }
    __syncthreads();
    prefix = (prefix << 8) | sh.word[0];
    above = sh.wide[0];
    __syncthreads();
  }
  return prefix;
}

// The whole of a row by one workgroup, without candidates.
template <int DT, class Aim>
__device__ uint32_t pick_from_row(SampleShared& sh, const SampleArgs& a, uint32_t row, const RowFilter& f,
                                  const Weigher& wt, uint32_t top_key, Aim aim) {
  const uint32_t V = a.vocab;
  // ---- cuts by rank: keys above `cut` are kept, and of those equal to it the first `ties` --------
  uint32_t cut = 0, ties = V;
  uint64_t above = 0;
  if (f.by_rank) {
    cut = key_reaching(sh, V, (uint64_t)f.k, [&](uint32_t i, uint32_t& key) {
      key = key_of(logit_at<DT>(a, row, i));
      return 1ull;
    }, above);
    ties = (uint32_t)((uint64_t)f.k - above);
  }
  if (f.p < 1.0) {
    const uint64_t tie_mass = cut ? wt.mass(key_value(cut)) : 0;
    uint64_t total = measure_row(sh, V, [&](uint32_t i) {
      const float x = logit_at<DT>(a, row, i);
      return key_of(x) > cut ? wt.mass(x) : 0ull;
    });
    total += tie_mass * (cut ? ties : 0);
    const double goal = f.p * (double)total;
    const uint64_t target = goal > 1.0 ? (uint64_t)ceil(goal) : 1ull;
    // the last kept token is the one whose running mass reaches the target. Equal keys weigh the
    // same, so all tokens of the cut's key may count here: those beyond `ties` come after the goal
    const uint32_t pcut = key_reaching(sh, V, target, [&](uint32_t i, uint32_t& key) {
      const float x = logit_at<DT>(a, row, i);
      key = key_of(x);
      return key >= cut ? wt.mass(x) : 0ull;
    }, above);
    const uint64_t each = wt.mass(key_value(pcut));
    const uint64_t want = (target - above + each - 1) / each;
    if (pcut > cut) ties = (uint32_t)min(want, (uint64_t)V);
    else ties = (uint32_t)min(want, (uint64_t)ties);
    cut = pcut;
  }
  // index of the last kept token among those equal to the cut
  uint32_t last_tie = V;
  if (cut) {
    auto tie = [&](uint32_t i) { return key_of(logit_at<DT>(a, row, i)) == cut ? 1ull : 0ull; };
    const uint64_t all = measure_row(sh, V, tie);
    if (ties < all) last_tie = first_beyond(sh, V, ties - 1, tie);
  }

  // ---- the draw ---------------------------------------------------------------------------------
  auto kept = [&](uint32_t i) {
    const float x = logit_at<DT>(a, row, i);
    const uint32_t key = key_of(x);
    if (key < cut || (key == cut && i > last_tie)) return 0ull;
    const double w = wt.weight(x);
    if (key != top_key && w < f.min_p * kSmpOne) return 0ull;
    return (unsigned long long)Weigher::fixed(w);
  };
  const uint64_t total = measure_row(sh, V, kept);
  return first_beyond(sh, V, aim(total), kept);
}

// Exclusive running sum of v over the threads, and the sum of all.
__device__ __forceinline__ uint64_t block_scan(SampleShared& sh, uint64_t v, uint64_t& total) {
  const int wave = threadIdx.x / kWave;
  const uint64_t incl = wave_scan(v);
  if (lane_id() == kWave - 1) sh.wsum[wave] = incl;
  __syncthreads();
  uint64_t off = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSmpWaves; ++w) {
    if (w < wave) off += sh.wsum[w];
    total += sh.wsum[w];
  }
  __syncthreads();
  return off + incl - v;
}

// Among the entries of sh.list in [lo, hi] (no two alike), the one at which the running measure, from the
// largest entry down, first reaches `target` (>= 1), or 0 where the total does not. A digit at a time, of
// the bounds and then of the range that is in use, until at most a wavefront's worth is left, which is
// ranked directly. Expects and leaves the digits' sums, the members and their ranks cleared. Loops are not
// unrolled: a workgroup goes through this code once, and fetching it is what takes the time (with the
// entries in registers it was 62 KB and 2 to 4 us slower).
template <class F>
__device__ __forceinline__ uint64_t entry_reaching(SampleShared& sh, uint32_t entries, F meas, uint64_t target,
                                                   uint64_t lo, uint64_t hi) {
  uint64_t above = 0;
#pragma unroll 1
  for (int digits = 0; digits < 11; ++digits) {   // a digit is 7 of 64 bits, the first one of the bounds
    if (digits > 0) {
      uint64_t mx = 0, nmn = 0;
#pragma unroll 1
      for (uint32_t i = threadIdx.x; i < entries; i += kSmpThreads) {
        const uint64_t e = sh.list[i];
        if (e >= lo && e <= hi) {
          mx = max(mx, e);
          nmn = max(nmn, ~e);
        }
      }
      mx = wave_max(mx);
      nmn = wave_max(nmn);
      if (lane_id() == 0) {
        sh.wsum[threadIdx.x / kWave] = mx;
        sh.wmin[threadIdx.x / kWave] = nmn;
      }
      __syncthreads();
      hi = 0;
      lo = 0;
#pragma unroll
      for (int w = 0; w < kSmpWaves; ++w) {
        hi = max(hi, sh.wsum[w]);
        lo = max(lo, sh.wmin[w]);
      }
      lo = ~lo;
      if (lo >= hi) {
        __syncthreads();
        return hi;
      }
    }
    uint32_t n = 0;
    if (entries > kWave) {                  // few entries are ranked as they are (2 of them: pick 7.4 -> 6.4 us)
      const int shift = max(0, 64 - __builtin_clzll(hi - lo) - kSmpDigitBits);
#pragma unroll 1
      for (uint32_t i = threadIdx.x; i < entries; i += kSmpThreads) {
        const uint64_t e = sh.list[i];
        if (e >= lo && e <= hi) {
          const uint32_t at = (uint32_t)((hi - e) >> shift) * kSmpCopies + lane_id() % kSmpCopies;
          atomicAdd((unsigned long long*)&sh.hist[at], (unsigned long long)meas(e));
          atomicAdd(&sh.count[at], 1u);
        }
      }
      __syncthreads();
      // a digit's copies are read by four neighbouring lanes
      static_assert(kSmpSlots == 4 * kSmpThreads && kSmpCopies == 16, "four slots a thread, four threads a digit");
      uint64_t s = 0, total;
      uint32_t c = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s += sh.hist[4 * threadIdx.x + j];
        c += sh.count[4 * threadIdx.x + j];
        sh.hist[4 * threadIdx.x + j] = 0;
        sh.count[4 * threadIdx.x + j] = 0;
      }
      s += dpp64<kDppXor1, 0xF>(s);
      s += dpp64<kDppXor2, 0xF>(s);
      c += (uint32_t)dpp<kDppXor1>(0, (int)c);
      c += (uint32_t)dpp<kDppXor2>(0, (int)c);
      const bool lead = threadIdx.x % 4 == 0;
      const uint64_t run = block_scan(sh, lead ? s : 0, total) + above;
      if (digits == 0 && total < target) return 0;
      if (lead && run < target && run + s >= target) {
        sh.word[0] = threadIdx.x / 4;
        sh.word[1] = c;
        sh.wide[0] = run;
      }
      __syncthreads();
      const uint64_t digit = sh.word[0];
      n = sh.word[1];
      above = sh.wide[0];
      hi -= digit << shift;
      const uint64_t width = (1ull << shift) - 1;
      const uint64_t least = hi > width ? hi - width : 0;   // one type on both sides of max, or it is the double's
      lo = max(lo, least);
    }
    if (n <= kWave) {
#pragma unroll 1
      for (uint32_t i = threadIdx.x; i < entries; i += kSmpThreads) {
        const uint64_t e = sh.list[i];
        if (e >= lo && e <= hi) {
          const uint32_t at = atomicAdd(&sh.members, 1u);
          sh.left[at][0] = e;
          sh.left[at][1] = meas(e);
        }
      }
      if (threadIdx.x == 0) sh.wide[1] = 0;
      __syncthreads();
      n = sh.members;
      // the measure in front of every member, an eighth of the members per wavefront
      const uint32_t member = threadIdx.x % kWave, first = threadIdx.x / kWave * (kWave / kSmpWaves);
      if (member < n) {
        const uint64_t mine = sh.left[member][0];
        uint64_t before = 0;
#pragma unroll
        for (uint32_t i = 0; i < kWave / kSmpWaves; ++i) {
          const uint64_t e = sh.left[first + i][0], w = sh.left[first + i][1];
          before += first + i < n && e > mine ? w : 0;
        }
        if (before) atomicAdd((unsigned long long*)&sh.before[member], (unsigned long long)before);
      }
      __syncthreads();
      if (threadIdx.x < n) {
        const uint64_t before = above + sh.before[threadIdx.x];
        sh.before[threadIdx.x] = 0;
        if (before < target && before + sh.left[threadIdx.x][1] >= target) sh.wide[1] = sh.left[threadIdx.x][0];
      }
      __syncthreads();
      if (threadIdx.x == 0) sh.members = 0;
      const uint64_t got = sh.wide[1];
      __syncthreads();
      return got;
    }
    __syncthreads();
  }
  return hi;
}

template <int DT>
__global__ __launch_bounds__(kSmpThreads) void sample_pick_kernel(SampleArgs a) {
  __shared__ SampleShared sh;
  const uint32_t row = blockIdx.x, V = a.vocab, segs = (V + kSmpSeg - 1) / kSmpSeg;
  // everything that does not depend on anything first: one round trip
  uint64_t best = slice_best(a, row);
  const uint32_t n = a.cand_count[row];
  const SampleCut c = a.cut[row];
  uint64_t mass[2] = {0, 0};
  if (lane_id() < a.slices) {
    const uint64_t* const m = a.mass + ((size_t)row * a.slices + lane_id()) * 2;
    mass[0] = m[0];
    mass[1] = m[1];
  }
  uint64_t seg = threadIdx.x < segs ? a.seg[(size_t)row * segs + threadIdx.x] : 0;
  const uint64_t* const cand = a.cand + (size_t)row * a.cand_stride;
  const uint64_t first = threadIdx.x < a.cand_stride ? cand[threadIdx.x] : 0;
  const float u = a.u[row];
  const RowFilter f = row_filter(a, row);
  fill_table(sh.table);
  for (int i = threadIdx.x; i < kSmpSlots; i += kSmpThreads) {
    sh.hist[i] = 0;
    sh.count[i] = 0;
  }
  if (threadIdx.x < kWave) sh.before[threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.members = 0;
  best = wave_max(best);
  const uint32_t top_key = (uint32_t)(best >> 32);
  if (f.greedy || top_key <= kKeyNone) {
    if (threadIdx.x == 0) a.tokens[row] = top_key <= kKeyNone ? -1 : (int64_t)(0xFFFFFFFFu - (uint32_t)best);
    return;
  }
  const float top = key_value(top_key);
  const Weigher wt(sh.table, top, f.T);
  auto aim = [&](uint64_t total) {
    const double at = (u > 0.0f ? fmin((double)u, 1.0) : 0.0) * (double)total;
    return min((uint64_t)at, total - 1);
  };
  __syncthreads();
  if (n > kSmpMaxCand) {
    const uint32_t token = pick_from_row<DT>(sh, a, row, f, wt, top_key, aim);
    if (threadIdx.x == 0) a.tokens[row] = token;
    return;
  }
  sh.list[threadIdx.x] = first;
#pragma unroll 4
  for (uint32_t i = threadIdx.x + kSmpThreads; i < n; i += kSmpThreads) sh.list[i] = cand[i];
  if (threadIdx.x < segs) sh.seg[threadIdx.x] = f.by_rank ? 0 : seg;
  __syncthreads();
  auto mass_of = [&](uint64_t e) { return wt.mass(key_value((uint32_t)(e >> 32))); };
  // candidates from `cut` up are kept. All of them lie between the edges of the cut's bin, or (top-k) up to
  // the best
  const uint64_t least = (uint64_t)key_of(c.cand) << 32;
  const uint64_t most = c.keep == c.keep ? ((uint64_t)key_of(c.keep) << 32) - 1 : ((uint64_t)top_key << 32) | 0xFFFFFFFFu;
  uint64_t cut = 0;
#pragma unroll 1
  for (int by_mass = 0; by_mass < 2; ++by_mass) {
    uint64_t target = (uint64_t)f.k;
    if (by_mass) {
      if (!(f.p < 1.0) || n == 0) break;
      uint64_t total, above = 0;
      if (f.by_rank) {
        uint64_t mine = 0;
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < n; i += kSmpThreads) mine += sh.list[i] >= cut ? mass_of(sh.list[i]) : 0;
        block_scan(sh, mine, total);
      } else {
        total = wave_sum(mass[0]);
        above = wave_sum(mass[1]);
      }
      const double goal = f.p * (double)total;
      target = goal > 1.0 ? (uint64_t)ceil(goal) : 1ull;
      target = target > above ? target - above : 1ull;
    } else if (!f.by_rank || (uint32_t)f.k >= n) {
      continue;
    }
    const uint64_t reached = entry_reaching(sh, n, [&](uint64_t e) { return by_mass ? mass_of(e) : 1ull; }, target,
                                            max(cut, least), most);
    cut = max(cut, reached);
  }
  // ---- sums over kSmpSeg tokens, and the draw -------------------------------------------------
  const double min_w = f.min_p > 0.0 ? f.min_p * kSmpOne : -1.0;
  auto passes = [&](uint32_t k, double w) { return k == top_key || w >= min_w; };
#pragma unroll 1
  for (uint32_t i = threadIdx.x; i < n; i += kSmpThreads) {
    const uint64_t e = sh.list[i];
    const uint32_t k = (uint32_t)(e >> 32);
    const double w = wt.weight(key_value(k));
    if (e >= cut && passes(k, w))
      atomicAdd((unsigned long long*)&sh.seg[(0xFFFFFFFFu - (uint32_t)e) / kSmpSeg],
                (unsigned long long)Weigher::fixed(w));
  }
  __syncthreads();
  seg = threadIdx.x < segs ? sh.seg[threadIdx.x] : 0;
  uint64_t total;
  const uint64_t off = block_scan(sh, seg, total);
  const uint64_t target = aim(total);
  if (off <= target && off + seg > target) {
    sh.word[0] = threadIdx.x;
    sh.wide[0] = off;
  }
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  const uint32_t i0 = sh.word[0] * kSmpSeg + lane_id() * 8;
  float x[8];
  logits8<DT>(a, row, i0, x);
  uint64_t m[8], sum = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t k = key_of(x[j]);
    const uint64_t e = ((uint64_t)k << 32) | (0xFFFFFFFFu - (i0 + j));
    const bool in = x[j] >= c.keep || (x[j] >= c.cand && e >= cut);
    const double w = wt.weight(x[j]);
    m[j] = in && passes(k, w) ? Weigher::fixed(w) : 0;
    sum += m[j];
  }
  uint64_t run = sh.wide[0] + wave_scan(sum) - sum;
  int found = -1;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (found < 0 && run + m[j] > target && run <= target) found = j;
    run += m[j];
  }
  if (found >= 0) a.tokens[row] = i0 + found;
}

struct SamplePlan {
  uint32_t slices, iters;
  uint64_t best, hist, seg, cand, mass, cut, count, bytes;   // offsets into the workspace
};
// Slices of 4096, 8192 or 16384 tokens: as large as leaves a workgroup per compute unit, or two where a row
// has few slices. Every slice reads the bins of all the row's slices, which is what many of them cost (63
// rows of 128256: 504 workgroups of 8 slices a row 49 us, 1008 of 16 55; 24 rows: 38 and 48; but 128 rows of
// 32000: 256 workgroups of 2 slices a row 37 us, 512 of 4 35).
static SamplePlan sample_plan(uint32_t rows, uint32_t vocab) {
  SamplePlan p{};
  for (p.iters = 4;; p.iters >>= 1) {
    p.slices = (vocab + p.iters * kSmpStep - 1) / (p.iters * kSmpStep);
    const uint64_t groups = (uint64_t)rows * p.slices;
    if (p.iters == 1 || groups >= 512 || (groups >= 256 && p.slices >= 4)) break;
  }
  const uint64_t r = rows, segs = (vocab + kSmpSeg - 1) / kSmpSeg;
  p.best = 0;
  p.hist = p.best + r * p.slices * 8;
  p.seg = p.hist + r * p.slices * kSmpBins * 8;
  p.cand = p.seg + r * segs * 8;
  p.mass = p.cand + r * (vocab < kSmpMaxCand ? vocab : kSmpMaxCand) * 8;
  p.cut = p.mass + r * p.slices * 16;
  p.count = p.cut + r * sizeof(SampleCut);
  p.bytes = p.count + r * 4;
  return p;
}

template <int DT>
static void launch_sample(const SampleArgs& a, hipStream_t st) {
  const dim3 grid(a.rows * a.slices), block(kSmpThreads);
#define TWL_SMP(ITERS)                                                                  \
  do {                                                                                  \
    hipLaunchKernelGGL((sample_hist_kernel<DT, ITERS>), grid, block, 0, st, a);         \
    hipLaunchKernelGGL((sample_keep_kernel<DT, ITERS>), grid, block, 0, st, a);         \
  } while (0)
  if (a.iters == 1) TWL_SMP(1);
  else if (a.iters == 2) TWL_SMP(2);
  else TWL_SMP(4);
#undef TWL_SMP
  hipLaunchKernelGGL((sample_pick_kernel<DT>), dim3(a.rows), block, 0, st, a);
}

}  // namespace twl

extern "C" uint64_t twl_sample_tokens_workspace_bytes(uint32_t rows, uint32_t vocab) {
  if (rows == 0 || vocab == 0 || vocab > twl::kSmpMaxVocab) return 0;
  return twl::sample_plan(rows, vocab).bytes;
}

extern "C" int twl_sample_tokens(const void* logits, int dtype, uint64_t row_stride, uint32_t rows,
                                 uint32_t vocab, const float* u, const float* temperature_arr,
                                 float temperature, const int32_t* top_k_arr, int32_t top_k,
                                 const float* top_p_arr, float top_p, const float* min_p_arr,
                                 float min_p, int64_t* tokens, void* workspace,
                                 uint64_t workspace_bytes, void* stream) {
  if (!logits || !u || !tokens || !workspace) return TWL_ENULL;
  if (dtype != TWL_F16 && dtype != TWL_BF16 && dtype != TWL_F32) return TWL_EDTYPE;
  if (rows == 0 || vocab == 0 || vocab > twl::kSmpMaxVocab || rows > 65535u) return TWL_EINVAL;
  if (temperature != temperature || top_p != top_p || min_p != min_p) return TWL_EINVAL;
  if (((uintptr_t)logits) & (dtype == TWL_F32 ? 3u : 1u)) return TWL_EALIGN;
  if ((((uintptr_t)u) | ((uintptr_t)temperature_arr) | ((uintptr_t)top_k_arr) | ((uintptr_t)top_p_arr) |
       ((uintptr_t)min_p_arr)) & 3u)
    return TWL_EALIGN;
  if ((((uintptr_t)tokens) | ((uintptr_t)workspace)) & 7u) return TWL_EALIGN;
  const twl::SamplePlan p = twl::sample_plan(rows, vocab);
  if (workspace_bytes < p.bytes) return TWL_EINVAL;
  twl::SampleArgs a{};
  a.logits = logits; a.row_stride = row_stride; a.rows = rows; a.vocab = vocab; a.u = u;
  a.temperature = temperature_arr; a.top_k = top_k_arr; a.top_p = top_p_arr; a.min_p = min_p_arr;
  a.temperature_all = temperature; a.top_k_all = top_k; a.top_p_all = top_p; a.min_p_all = min_p;
  a.tokens = tokens;
  uint8_t* const ws = (uint8_t*)workspace;
  a.slices = p.slices; a.iters = p.iters; a.best = (uint64_t*)(ws + p.best); a.hist = (uint64_t*)(ws + p.hist);
  a.seg = (uint64_t*)(ws + p.seg); a.cand = (uint64_t*)(ws + p.cand); a.cut = (twl::SampleCut*)(ws + p.cut);
  a.cand_count = (uint32_t*)(ws + p.count); a.mass = (uint64_t*)(ws + p.mass);
  a.cand_stride = vocab < twl::kSmpMaxCand ? vocab : twl::kSmpMaxCand;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == TWL_F16) twl::launch_sample<TWL_F16>(a, st);
  else if (dtype == TWL_BF16) twl::launch_sample<TWL_BF16>(a, st);
  else twl::launch_sample<TWL_F32>(a, st);
  return hipGetLastError() == hipSuccess ? TWL_OK : TWL_ELAUNCH;
}
