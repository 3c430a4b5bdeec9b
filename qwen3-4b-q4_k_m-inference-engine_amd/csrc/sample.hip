// The next token of each row by temperature, top-k, top-p and min-p from a
// given uniform: one workgroup per row.
//
// Values are ranked by a 32-bit key whose unsigned order is the order of the
// logits (NaN and -inf: 0, never drawn). top-k and top-p are the same search:
// the largest key K whose measure of {key >= K} reaches a target, the measure
// being a count or a sum of weights; it is found digit by digit (11, 11, 10
// bits) from a histogram of the values that share the digits found so far.
// Weights are fixed-point integers, rint(exp((z - max) / T) * 2^shift) of a
// 64-bit exponential with 2^shift * vocabulary < 2^62, so every sum is exact
// and no order of additions can change a result.
#include "qk_device.hpp"
#include "qk_launch.hpp"
#include "serving.hpp"

namespace qk {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 2048;

__device__ __forceinline__ uint32_t rank_key(float v) {
  if (!(v > -__builtin_inff())) return 0;
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);  // -0 -> +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __builtin_bit_cast(float, (key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}

struct Weigher {
  double max, inv_t, one;
  __device__ __forceinline__ double ratio(uint32_t key) const {
    const double z = key_value(key);
    return z == max ? 1.0 : exp((z - max) * inv_t);
  }
  __device__ __forceinline__ uint64_t fixed(uint32_t key) const {
    return key == 0 ? 0 : static_cast<uint64_t>(rint(ratio(key) * one));
  }
};

struct Shared {
  uint64_t bins[kBins];
  uint64_t wave[16];
  uint64_t found[3];
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
__device__ uint64_t group_sum(uint64_t v, Shared& sh) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t t = 0;
  for (int i = 0; i < kThreads / 64; ++i) t += sh.wave[i];
  return t;
}

// The largest key whose measure of {key >= it} reaches target (1 <= target <=
// the measure of all), and in `above` the measure of the larger ones.
template <class F>
__device__ uint32_t descend(const float* x, int n, uint64_t target, F measure, uint64_t& above, Shared& sh) {
  uint32_t prefix = 0;
  above = 0;
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint32_t key = rank_key(x[i]);
      if (digit == 0 || key >> (shift + bits) == prefix) {
        const uint64_t m = measure(key);
        if (m) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(key >> shift) & ((1u << bits) - 1)]), m);
      }
    }
    __syncthreads();
    // bins from the top: thread t has bins n-1-2t and n-2-2t
    const int count = 1 << bits, hi = count - 1 - 2 * static_cast<int>(threadIdx.x);
    const uint64_t b0 = hi >= 0 ? sh.bins[hi] : 0, b1 = hi >= 1 ? sh.bins[hi - 1] : 0;
    uint64_t run = b0 + b1;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint64_t other = __shfl_up(run, off);
      if (lane >= off) run += other;
    }
    if (lane == 63) sh.wave[threadIdx.x >> 6] = run;
    __syncthreads();
    uint64_t before = above;
    for (int i = 0; i < static_cast<int>(threadIdx.x >> 6); ++i) before += sh.wave[i];
    before += run - (b0 + b1);
    if (before < target && before + b0 + b1 >= target) {
      const bool upper = before + b0 >= target;
      sh.found[0] = static_cast<uint64_t>(upper ? hi : hi - 1);
      sh.found[1] = upper ? before : before + b0;
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<uint32_t>(sh.found[0]);
    above = sh.found[1];
  }
  return prefix;
}

// Index of the first element, in index order, at which the running sum of
// measure exceeds `beyond`; n if it never does.
template <class F>
__device__ int walk(const float* x, int n, uint64_t beyond, F measure, Shared& sh) {
  // each wave a contiguous run of the row
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int span = ((n + kThreads - 1) / kThreads) * 64;
  const int lo = min(n, wave * span), hi = min(n, lo + span);
  uint64_t sum = 0;
  for (int i = lo + lane; i < hi; i += 64) sum += measure(rank_key(x[i]), i);
  sum = wave_sum(sum);
  __syncthreads();
  if (lane == 0) sh.wave[wave] = sum;
  if (threadIdx.x == 0) sh.found[0] = static_cast<uint64_t>(n);
  __syncthreads();
  uint64_t before = 0;
  for (int i = 0; i < wave; ++i) before += sh.wave[i];
  if (before <= beyond && before + sum > beyond) {
    for (int base = lo; base < hi; base += 64) {
      const int i = base + lane;
      uint64_t run = i < hi ? measure(rank_key(x[i]), i) : 0;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint64_t other = __shfl_up(run, off);
        if (lane >= off) run += other;
      }
      const uint64_t crossed = __ballot(before + run > beyond);
      if (crossed) {
        if (lane == 0) sh.found[0] = static_cast<uint64_t>(base + __builtin_ctzll(crossed));
        break;
      }
      before += __shfl(run, 63);
    }
  }
  __syncthreads();
  return static_cast<int>(sh.found[0]);
}

__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs a, int shift) {
  __shared__ Shared sh;
  const int row = static_cast<int>(blockIdx.x), n = a.vocabulary;
  const float* x = a.logits + row * a.row_stride;
  const float heat = a.temperature[row];
  uint64_t best = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint32_t key = rank_key(x[i]);
    const uint64_t c = key ? (static_cast<uint64_t>(key) << 32) | (0xFFFFFFFFu - i) : 0;
    best = c > best ? c : best;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t other = __shfl_xor(best, off);
    best = other > best ? other : best;
  }
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = best;
  __syncthreads();
  for (int i = 0; i < kThreads / 64; ++i) best = sh.wave[i] > best ? sh.wave[i] : best;
  if (!(heat > 0.0f) || best == 0) {
    if (threadIdx.x == 0) {
      a.token[row] = best ? 0xFFFFFFFFu - static_cast<uint32_t>(best) : 0xFFFFFFFFu;
      if (a.probability) a.probability[row] = best ? 1.0f : 0.0f;
    }
    return;
  }
  const uint32_t top = static_cast<uint32_t>(best >> 32);
  const Weigher w{static_cast<double>(key_value(top)), 1.0 / heat, static_cast<double>(uint64_t{1} << shift)};

  // kept: keys above `least`, and of those equal to it the ones up to index
  // `last`
  uint32_t least = 1;
  int last = n;
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < n) {
    uint64_t mine = 0, above;
    for (int i = threadIdx.x; i < n; i += kThreads) mine += rank_key(x[i]) != 0;
    if (group_sum(mine, sh) > static_cast<uint64_t>(k)) {
      least = descend(x, n, k, [](uint32_t key) { return key ? uint64_t{1} : 0; }, above, sh);
      last = walk(x, n, k - above - 1, [=](uint32_t key, int) { return key == least ? uint64_t{1} : 0; }, sh);
    }
  }
  const auto weigh = [&](uint32_t key, int i) {
    return key > least || (key == least && i <= last) ? w.fixed(key) : 0;
  };
  const double p = a.top_p ? static_cast<double>(a.top_p[row]) : 1.0;
  if (p < 1.0) {
    uint64_t mine = 0, above;
    for (int i = threadIdx.x; i < n; i += kThreads) mine += weigh(rank_key(x[i]), i);
    const uint64_t total = group_sum(mine, sh);
    const double goal = ceil(p * static_cast<double>(total));
    const uint64_t target = goal < 1.0 ? 1 : min(total, static_cast<uint64_t>(goal));
    // equal keys beyond `last` weigh more than their share here; the search
    // then ends at `least` itself, and the count below is cut to `last`
    const uint32_t key = descend(x, n, target, [&](uint32_t q) { return q >= least ? w.fixed(q) : 0; }, above, sh);
    const uint64_t each = w.fixed(key), keep = (target - above + each - 1) / each;
    const int upto = walk(x, n, keep - 1, [=](uint32_t q, int) { return q == key ? uint64_t{1} : 0; }, sh);
    if (key > least) {
      least = key;
      last = upto;
    } else {
      last = min(last, upto);
    }
  }
  const double floor_w = a.min_p ? static_cast<double>(a.min_p[row]) : 0.0;
  const auto kept = [&](uint32_t key, int i) -> uint64_t {
    if (key < least || (key == least && i > last)) return 0;
    return key == top || w.ratio(key) >= floor_w ? w.fixed(key) : 0;
  };
  uint64_t mine = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) mine += kept(rank_key(x[i]), i);
  const uint64_t total = group_sum(mine, sh);
  const double aim = static_cast<double>(a.uniform[row]) * static_cast<double>(total);
  const uint64_t beyond = aim >= 0.0 ? (aim < static_cast<double>(total) ? static_cast<uint64_t>(aim) : total - 1) : 0;
  const int index = walk(x, n, min(beyond, total - 1), kept, sh);
  if (threadIdx.x == 0) {
    a.token[row] = static_cast<uint32_t>(index);
    if (a.probability) a.probability[row] = static_cast<float>(static_cast<double>(kept(rank_key(x[index]), index)) / static_cast<double>(total));
  }
}

}  // namespace

size_t sample_workspace(int64_t, int64_t) { return 0; }

hipError_t launch_sample(const SampleArgs& a, void*, hipStream_t stream) {
  int shift = 62;
  while ((int64_t{1} << (62 - shift)) < a.vocabulary) --shift;
  sample_kernel<<<a.rows, kThreads, 0, stream>>>(a, shift);
  note("sample_kernel", a.rows);
  return hipGetLastError();
}

}  // namespace qk
