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
// bits). What is lost is below 2^-46 of the best token's weight, per token.
//
// One workgroup per row. The cuts by rank are found digit by digit of the logit's ordered bit
// pattern (count or mass per digit in LDS); the tokens that share the last kept value are kept in
// index order.
#include "twl_common.h"

namespace twl {

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
};

constexpr int kSmpThreads = 1024;
constexpr int kSmpWaves = kSmpThreads / kWave;
constexpr uint32_t kSmpMaxVocab = 1u << 18;
constexpr double kSmpOne = 35184372088832.0;   // 2^45: the weight 1

template <int DT>
__device__ __forceinline__ float logit_at(const SampleArgs& a, uint32_t row, uint32_t i) {
  float x;
  if (DT == TWL_F32) x = ((const float*)a.logits)[row * a.row_stride + i];
  else x = bits16_to_f32<DT>(((const uint16_t*)a.logits)[row * a.row_stride + i]);
  return x != x ? -__builtin_inff() : x + 0.0f;   // NaN counts as masked; -0 ranks as +0
}
// order-preserving bit pattern
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = as_u32(x);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {   // inclusive, in lane order
  const int lane = lane_id();
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint64_t x = __shfl_up(v, d);
    if (lane >= d) v += x;
  }
  return v;
}

struct SampleShared {
  uint64_t seg[kSmpMaxVocab / kWave];   // measure of every 64 tokens
  uint64_t mass[256];
  uint32_t count[256];
  uint64_t wsum[kSmpWaves];
  uint32_t word[8];
  uint64_t wide[4];
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
  uint64_t before = 0;                  // measure of the segments in front of this round
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
    if (threadIdx.x < 256) sh.mass[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < vocab; i += kSmpThreads) {
      uint32_t key;
      const uint64_t m = measure(i, key);
      if (m && (shift == 24 || (key >> (shift + 8)) == prefix))
        atomicAdd((unsigned long long*)&sh.mass[(key >> shift) & 255], (unsigned long long)m);
    }
    __syncthreads();
    if (threadIdx.x < kWave) {          // lane 0 holds the four largest digits
      const int lane = lane_id();
      uint64_t m[4], s = 0;
      for (int j = 0; j < 4; ++j) s += m[j] = sh.mass[255 - (4 * lane + j)];
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

template <int DT>
__global__ __launch_bounds__(kSmpThreads) void sample_kernel(SampleArgs a) {
  __shared__ SampleShared sh;
  const uint32_t row = blockIdx.x, V = a.vocab;
  const int wave = threadIdx.x / kWave;
  const float T0 = a.temperature ? a.temperature[row] : a.temperature_all;
  const double T = fmin((double)T0, 1e300);   // finite: a masked logit has weight 0 at every T
  const double p = a.top_p ? a.top_p[row] : a.top_p_all;
  const double min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  const int32_t k = a.top_k ? a.top_k[row] : a.top_k_all;

  // ---- the best token ---------------------------------------------------------------------------
  uint64_t best = 0;                    // key, then the lowest index
  for (uint32_t i = threadIdx.x; i < V; i += kSmpThreads)
    best = max(best, ((uint64_t)key_of(logit_at<DT>(a, row, i)) << 32) | (0xFFFFFFFFu - i));
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) best = max(best, (uint64_t)__shfl_xor(best, d));
  if (lane_id() == 0) sh.wsum[wave] = best;
  __syncthreads();
  for (int w = 0; w < kSmpWaves; ++w) best = max(best, sh.wsum[w]);
  __syncthreads();
  const uint32_t top_key = (uint32_t)(best >> 32), top_at = 0xFFFFFFFFu - (uint32_t)best;
  if (top_key <= key_of(-__builtin_inff()) || !(T0 > 0.0f) || k == 1) {
    if (threadIdx.x == 0) a.tokens[row] = top_key <= key_of(-__builtin_inff()) ? -1 : (int64_t)top_at;
    return;
  }
  const double top = logit_at<DT>(a, row, top_at);
  auto weight = [&](float x) { return (double)x == top ? 1.0 : exp(((double)x - top) / T); };
  auto mass = [&](float x) { return (uint64_t)(weight(x) * kSmpOne + 0.5); };

  // ---- cuts by rank: keys above `cut` are kept, and of those equal to it the first `ties` --------
  uint32_t cut = 0, ties = V;
  uint64_t above = 0;
  if (k > 0 && (uint32_t)k < V) {
    cut = key_reaching(sh, V, (uint64_t)k, [&](uint32_t i, uint32_t& key) {
      key = key_of(logit_at<DT>(a, row, i));
      return 1ull;
    }, above);
    ties = (uint32_t)((uint64_t)k - above);
  }
  auto key_value = [](uint32_t key) { return as_f32(key ^ (~(uint32_t)((int32_t)key >> 31) | 0x80000000u)); };
  if (p < 1.0) {
    const uint64_t tie_mass = cut ? mass(key_value(cut)) : 0;
    uint64_t total = measure_row(sh, V, [&](uint32_t i) {
      const float x = logit_at<DT>(a, row, i);
      return key_of(x) > cut ? mass(x) : 0ull;
    });
    total += tie_mass * (cut ? ties : 0);
    const double goal = p * (double)total;
    const uint64_t target = goal > 1.0 ? (uint64_t)ceil(goal) : 1ull;
    // the last kept token is the one whose running mass reaches the target. Equal keys weigh the
    // same, so all tokens of the cut's key may count here: those beyond `ties` come after the goal
    const uint32_t pcut = key_reaching(sh, V, target, [&](uint32_t i, uint32_t& key) {
      const float x = logit_at<DT>(a, row, i);
      key = key_of(x);
      return key >= cut ? mass(x) : 0ull;
    }, above);
    const uint64_t each = mass(key_value(pcut));
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
    const double w = weight(x);
    if (key != top_key && w < min_p) return 0ull;
    return (unsigned long long)(w * kSmpOne + 0.5);
  };
  const uint64_t total = measure_row(sh, V, kept);
  const float u = a.u[row];
  const double at = (u > 0.0f ? fmin((double)u, 1.0) : 0.0) * (double)total;
  const uint64_t target = min((uint64_t)at, total - 1);
  const uint32_t token = first_beyond(sh, V, target, kept);
  if (threadIdx.x == 0) a.tokens[row] = token;
}

}  // namespace twl

extern "C" int twl_sample_tokens(const void* logits, int dtype, uint64_t row_stride, uint32_t rows,
                                 uint32_t vocab, const float* u, const float* temperature_arr,
                                 float temperature, const int32_t* top_k_arr, int32_t top_k,
                                 const float* top_p_arr, float top_p, const float* min_p_arr,
                                 float min_p, int64_t* tokens, void* stream) {
  if (!logits || !u || !tokens) return TWL_ENULL;
  if (dtype != TWL_F16 && dtype != TWL_BF16 && dtype != TWL_F32) return TWL_EDTYPE;
  if (rows == 0 || vocab == 0 || vocab > twl::kSmpMaxVocab || rows > 0x7FFFFFFFu) return TWL_EINVAL;
  if (temperature != temperature || top_p != top_p || min_p != min_p) return TWL_EINVAL;
  if (((uintptr_t)logits) & (dtype == TWL_F32 ? 3u : 1u)) return TWL_EALIGN;
  if ((((uintptr_t)u) | ((uintptr_t)temperature_arr) | ((uintptr_t)top_k_arr) | ((uintptr_t)top_p_arr) |
       ((uintptr_t)min_p_arr)) & 3u)
    return TWL_EALIGN;
  if (((uintptr_t)tokens) & 7u) return TWL_EALIGN;
  twl::SampleArgs a{};
  a.logits = logits; a.row_stride = row_stride; a.rows = rows; a.vocab = vocab; a.u = u;
  a.temperature = temperature_arr; a.top_k = top_k_arr; a.top_p = top_p_arr; a.min_p = min_p_arr;
  a.temperature_all = temperature; a.top_k_all = top_k; a.top_p_all = top_p; a.min_p_all = min_p;
  a.tokens = tokens;
  const dim3 grid(rows), block(twl::kSmpThreads);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == TWL_F16) hipLaunchKernelGGL((twl::sample_kernel<TWL_F16>), grid, block, 0, st, a);
  else if (dtype == TWL_BF16) hipLaunchKernelGGL((twl::sample_kernel<TWL_BF16>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((twl::sample_kernel<TWL_F32>), grid, block, 0, st, a);
  return hipGetLastError() == hipSuccess ? TWL_OK : TWL_ELAUNCH;
}
