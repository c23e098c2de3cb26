// One token id from each row of logits and one given uniform number a row
// (gfx950): temperature, top-k, top-p, min-p.
//
//   w_i = exp((x_i - max x) / T); ids ordered by (x descending, id ascending);
//   top-k keeps the first k, top-p of those the ones with less than p of their
//   weight before them, min-p those with w_i >= min_p (w of the best is 1); the
//   token is the first id, in ascending order, whose kept weight up to and with
//   it exceeds u times the kept weight.  T <= 0: the best id.
//
// All three rules keep a prefix of one order, so what is kept is one key (the
// order key of x), how many ids of that key, and min-p's bound.
//
// Weights.  A draw falls between two words' shares; with f32 weights the border
// is off by 1e-7 of the row's weight and one draw in a few hundred over 32000
// words would give the neighbour.  So w is 2^y with y in 64 bits, from the series of
// exp to the tenth power (|z| <= ln 2 / 2: 3e-13), held as an integer of 2^-44
// units: sums of integers have no order, so that histograms by atomics give the
// same bits each time; 2^18 words sum to less than 2^62.
#include "abi.h"
#include "common.h"

namespace moc {
namespace {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmBits = 44;
constexpr int64_t kSmMaxVocab = 1 << 18;

struct SampleArgs {
  const void* x;
  int64_t ld;
  int vocab;
  const float *u, *temp, *top_p, *min_p;  // per row, or null: the number below
  const int32_t* top_k;
  float temp1, top_p1, min_p1;
  int top_k1;
  int64_t* out;
};

template <bool BF16>
__device__ __forceinline__ float logit(const SampleArgs& a, int64_t row, int i) {
  const float x = BF16 ? bf16_to_f32(static_cast<const uint16_t*>(a.x)[row * a.ld + i])
                       : static_cast<const float*>(a.x)[row * a.ld + i];
  return x != x ? -INFINITY : x;  // NaN is never drawn
}

struct Weights {
  float max;
  double c;  // log2(e) / T
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (x == max) return 1ull << kSmBits;
    const double y = (static_cast<double>(x) - static_cast<double>(max)) * c;
    if (!(y > -46.0)) return 0;
    const double n = rint(y), z = (y - n) * 0.69314718055994530942;
    double p = 1.0 / 3628800.0;
    p = fma(p, z, 1.0 / 362880.0);
    p = fma(p, z, 1.0 / 40320.0);
    p = fma(p, z, 1.0 / 5040.0);
    p = fma(p, z, 1.0 / 720.0);
    p = fma(p, z, 1.0 / 120.0);
    p = fma(p, z, 1.0 / 24.0);
    p = fma(p, z, 1.0 / 6.0);
    p = fma(p, z, 0.5);
    p = fma(p, z, 1.0);
    p = fma(p, z, 1.0);
    return static_cast<uint64_t>(rint(ldexp(p, static_cast<int>(n) + kSmBits)));
  }
};

struct Lds {
  uint64_t mass[256];
  uint32_t count[256];
  uint64_t wave[kSmWaves];
  float fmax[kSmWaves];
  int imin[kSmWaves];
  uint64_t r64[2];
  int r32[4];
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(static_cast<unsigned long long>(v), o);
  return v;
}

// Sum of v over the lanes before this one.
__device__ __forceinline__ uint64_t wave_before64(uint64_t v) {
  const int lane = threadIdx.x & 63;
  uint64_t s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t t = __shfl_up(static_cast<unsigned long long>(s), o);
    if (lane >= o) s += t;
  }
  return s - v;
}

template <bool BF16>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleArgs a) {
  __shared__ Lds lds;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab;
  const float T = a.temp ? a.temp[row] : a.temp1;
  const int k = a.top_k ? a.top_k[row] : a.top_k1;
  const float p = a.top_p ? a.top_p[row] : a.top_p1, min_p = a.min_p ? a.min_p[row] : a.min_p1;

  // the best, lowest id first
  float best = -INFINITY;
  int at = V;
  for (int i = tid; i < V; i += kSmThreads) {
    const float x = logit<BF16>(a, row, i);
    if (x > best) {
      best = x;
      at = i;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float x = __shfl_xor(best, o);
    const int j = __shfl_xor(at, o);
    if (x > best || (x == best && j < at)) {
      best = x;
      at = j;
    }
  }
  if (lane == 0) {
    lds.fmax[wave] = best;
    lds.imin[wave] = at;
  }
  __syncthreads();
  for (int w = 0; w < kSmWaves; ++w) {
    const float x = lds.fmax[w];
    const int j = lds.imin[w];
    if (x > best || (x == best && j < at)) {
      best = x;
      at = j;
    }
  }
  if (best == -INFINITY) {  // nothing to draw
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (!(T > 0.f)) {
    if (tid == 0) a.out[row] = at;
    return;
  }
  const Weights weight{best, 1.4426950408889634074 / static_cast<double>(T)};

  // kept so far: keys above `key`, and the first `ties` ids of that key
  uint32_t key = 0;
  int ties = V;
  // One digit of the order key at a time: the digit where the ids above
  // (`before`) reach the rule's amount.
  auto descend = [&](bool by_mass, uint64_t target, double share) {
    uint32_t prefix = 0, mask = 0;
    uint64_t above_mass = 0;
    int above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) {
        lds.mass[tid] = 0;
        lds.count[tid] = 0;
      }
      __syncthreads();
      for (int i = tid; i < V; i += kSmThreads) {
        const float x = logit<BF16>(a, row, i);
        const uint32_t q = f32_order_key(__float_as_uint(x));
        if ((q & mask) != prefix || q < key) continue;
        const int b = (q >> shift) & 255;
        atomicAdd(&lds.count[b], 1u);
        if (by_mass) atomicAdd(reinterpret_cast<unsigned long long*>(&lds.mass[b]), weight(x));
      }
      __syncthreads();
      if (tid == 0) {
        int b = 255;
        for (; b > 0; --b) {
          // the ids of this bin exhaust the rule?
          uint32_t n = lds.count[b];
          if (by_mass ? static_cast<double>(above_mass + lds.mass[b]) >= share
                      : static_cast<uint64_t>(above) + n >= target)
            break;
          above += n;
          above_mass += lds.mass[b];
        }
        lds.r32[0] = b;
        lds.r32[1] = above;
        lds.r64[0] = above_mass;
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(lds.r32[0]) << shift;
      mask |= 255u << shift;
      above = lds.r32[1];
      above_mass = lds.r64[0];
    }
    int n = static_cast<int>(lds.count[prefix & 255]);
    if (prefix == key) n = min(n, ties);
    if (by_mass) {  // of equal weights, those with less than the share before them
      const uint64_t w = n > 0 ? lds.mass[prefix & 255] / lds.count[prefix & 255] : 0;
      int c = 0;
      while (c < n && static_cast<double>(above_mass + w * static_cast<uint64_t>(c)) < share) ++c;
      n = c;
    } else {
      n = min(n, static_cast<int>(target) - above);
    }
    key = prefix;
    ties = n;
    __syncthreads();
  };
  if (k > 0 && k < V) descend(false, static_cast<uint64_t>(k), 0.0);

  // A thread owns a run of ids, so that the ids of one key are met in order.
  const int run = (V + kSmThreads - 1) / kSmThreads, i0 = min(tid * run, V), i1 = min(i0 + run, V);
  auto totals = [&](uint64_t floor, uint64_t& before, uint64_t& total, int& rank) {
    int mine = 0;
    for (int i = i0; i < i1; ++i) mine += f32_order_key(__float_as_uint(logit<BF16>(a, row, i))) == key;
    __syncthreads();
    const uint64_t rb = wave_before64(static_cast<uint64_t>(mine));
    if (lane == 63) lds.wave[wave] = rb + mine;
    __syncthreads();
    uint64_t r = rb;
    for (int w = 0; w < wave; ++w) r += lds.wave[w];
    rank = static_cast<int>(r);
    int seen = rank;
    uint64_t s = 0;
    for (int i = i0; i < i1; ++i) {
      const float x = logit<BF16>(a, row, i);
      const uint32_t q = f32_order_key(__float_as_uint(x));
      if (q < key || (q == key && seen++ >= ties)) continue;
      const uint64_t w = weight(x);
      if (w >= floor) s += w;
    }
    __syncthreads();
    const uint64_t sb = wave_before64(s);
    if (lane == 63) lds.wave[wave] = sb + s;
    __syncthreads();
    before = sb;
    total = 0;
    for (int w = 0; w < kSmWaves; ++w) {
      if (w < wave) before += lds.wave[w];
      total += lds.wave[w];
    }
  };
  uint64_t before, total;
  int rank;
  if (p < 1.f) {
    totals(0, before, total, rank);
    const double share = fmax(static_cast<double>(p), 0.0) * static_cast<double>(total);
    if (share > 0.0) {
      descend(true, 0, share);
    } else {  // the best alone
      key = f32_order_key(__float_as_uint(best));
      ties = 1;
    }
    if (ties < 1) ties = 1;
  }
  uint64_t floor = 1;
  if (min_p > 0.f) floor = static_cast<uint64_t>(ceil(ldexp(fmin(static_cast<double>(min_p), 1.0), kSmBits)));
  totals(floor, before, total, rank);
  const float u = a.u[row];
  const double target = (u > 0.f ? static_cast<double>(fminf(u, 1.f)) : 0.0) * static_cast<double>(total);
  // u >= 1: the last id with weight
  uint64_t sum = before;
  int seen = rank, got = -1, last = -1;
  for (int i = i0; i < i1; ++i) {
    const float x = logit<BF16>(a, row, i);
    const uint32_t q = f32_order_key(__float_as_uint(x));
    if (q < key || (q == key && seen++ >= ties)) continue;
    const uint64_t w = weight(x);
    if (w < floor) continue;
    last = i;
    if (got < 0 && static_cast<double>(sum) <= target && static_cast<double>(sum + w) > target) got = i;
    sum += w;
  }
  if (got >= 0) a.out[row] = got;
  if (static_cast<double>(total) <= target && last >= 0 && sum == total) a.out[row] = last;
}

}  // namespace
}  // namespace moc

using namespace moc;

extern "C" int moc_sample_tokens(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t ld, const float* u,
                                 const float* temperature, float temperature1, const int32_t* top_k, int top_k1,
                                 const float* top_p, float top_p1, const float* min_p, float min_p1, int64_t* out,
                                 void* stream) {
  MOC_REQUIRE(dtype == MOC_BF16 || dtype == MOC_F32, "moc_sample_tokens: logits must be bf16 or f32");
  MOC_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= kSmMaxVocab && ld >= 0 && rows < (1LL << 31),
              "moc_sample_tokens: 1 to %lld words a row", (long long)kSmMaxVocab);
  if (rows == 0) return MOC_OK;
  MOC_REQUIRE(logits && u && out, "moc_sample_tokens: null pointer");
  const SampleArgs a{logits, ld, static_cast<int>(vocab), u, temperature, top_p, min_p, top_k,
                     temperature1, top_p1, min_p1, top_k1, out};
  const dim3 grid(static_cast<unsigned>(rows));
  if (dtype == MOC_BF16) sample_kernel<true><<<grid, kSmThreads, 0, as_stream(stream)>>>(a);
  else sample_kernel<false><<<grid, kSmThreads, 0, as_stream(stream)>>>(a);
  return check_launch("sample_kernel");
}
