// One token id from each row of logits and one given uniform number a row
// (gfx950): temperature, top-k, top-p, min-p.
//
//   w_i = exp((x_i - max x) / T); ids ordered by (x descending, id ascending);
//   top-k keeps the first k, top-p of those the ones with less than p of their
//   weight before them, min-p those with w_i >= min_p (w of the best is 1); the
//   token is the first id, in ascending order, whose kept weight up to and with
//   it exceeds u times the kept weight.  T <= 0: the best id.
//
// Weights.  A draw falls between two words' shares; with f32 weights the border
// is off by 1e-7 of the row's weight and one draw in a few hundred over 32000
// words would give the neighbour.  So w = 2^y with y in 64 bits: a table of
// 2^(i/64) and the series of 2^r to the fourth power (|r| <= 2^-7: 4e-14), held
// in units of 2^-44.  Sums of these are sums of integers (2^18 words: less than
// 2^62) and have no order, so histograms by atomics give the same bits each time.
//
// Rules.  Top-k and top-p keep a prefix of one order, so what is kept is its last
// word, (key, id).  It is found with a histogram over the distance from the best
// in 1/88 octaves of weight (numbers of words for top-k, their weights for top-p;
// 4096 bins reach 46.5 octaves, below which a weight is 0) and then among the
// words of the bin where the rule's amount is reached, each against all others;
// where they are too many (equal logits), digit by digit of the order key.
// A top-k of up to a few hundred words goes on as a list in LDS.
//
// One workgroup a row: the largest value of each block of words (16 bytes a lane of
// a wave) and of the row, a histogram for each rule in use, the weights by blocks,
// the block and then the lane of the draw.  The row is read again for each pass
// (128 KB of 32000 words from L2 at 64 B a clock: under a microsecond), blocks
// whose largest value is below the cut are not.  Bound by the 64-bit arithmetic of
// the weights, 18 instructions a word, and for few words by the chain of passes
// and barriers.
#include <type_traits>

#include "abi.h"
#include "common.h"

namespace moc {
namespace {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / 64;
constexpr int kSmBins = 4 * kSmThreads;
constexpr double kSmBinsPerOctave = 88.0;
constexpr int64_t kSmMaxVocab = 1 << 18;
constexpr int kSmBlocks = kSmMaxVocab / 256;  // blocks of f32 words
constexpr int kSmList = 512;                  // words compared each with all
constexpr int kSmFew = 256;                   // top-k that goes on as a list

struct SampleArgs {
  const void* x;
  int64_t ld;
  int vocab;
  bool wide;  // rows in 16-byte loads
  const float *u, *temp, *top_p, *min_p;  // per row, or null: the number below
  const int32_t* top_k;
  float temp1, top_p1, min_p1;
  int top_k1;
  int64_t* out;
};

struct SampleLds {
  uint64_t hist[kSmBins];    // weights; as uint32_t: numbers of words
  uint64_t block[kSmBlocks];  // kept weight of each block of words
  float high[kSmBlocks];      // its largest value
  double pow2[64];
  uint32_t key[kSmList];
  int id[kSmList];
  uint64_t w[kSmList];
  uint64_t wave[kSmWaves];
  float top[kSmWaves];
  int first;
  int n;
  uint32_t cut_key;
  int cut_id;
  int bin;
  uint64_t above, held;
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return __shfl_xor(static_cast<unsigned long long>(v), o);
}

template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  return dpp_u32<CTRL>(static_cast<uint32_t>(v)) | (static_cast<uint64_t>(dpp_u32<CTRL>(static_cast<uint32_t>(v >> 32))) << 32);
}

// Sum over the 64 lanes, returned to every lane.
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
  v += dpp_u64<0xB1>(v);
  v += dpp_u64<0x4E>(v);
  v += dpp_u64<0x141>(v);
  v += dpp_u64<0x140>(v);
  uint64_t s = 0;
#pragma unroll
  for (int r = 0; r < 64; r += 16)
    s += wave_read_lane(static_cast<uint32_t>(v), r) |
         (static_cast<uint64_t>(wave_read_lane(static_cast<uint32_t>(v >> 32), r)) << 32);
  return s;
}

__device__ __forceinline__ float wave_max_f32(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  v = fmaxf(v, dpp_f32<0x140>(v));
  const float a = __uint_as_float(wave_read_lane(__float_as_uint(v), 0)), b = __uint_as_float(wave_read_lane(__float_as_uint(v), 16));
  const float c = __uint_as_float(wave_read_lane(__float_as_uint(v), 32)), d = __uint_as_float(wave_read_lane(__float_as_uint(v), 48));
  return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// Sum of v over the lanes up to and with this one.
__device__ __forceinline__ uint64_t wave_upto64(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t t = __shfl_up(static_cast<unsigned long long>(v), o);
    if (lane >= o) v += t;
  }
  return v;
}

// Sum of v over the threads before this one; total over all.
__device__ __forceinline__ uint64_t block_before64(uint64_t v, uint64_t* wave_lds, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t upto = wave_upto64(v);
  __syncthreads();
  if (lane == 63) wave_lds[wave] = upto;
  __syncthreads();
  uint64_t before = upto - v;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSmWaves; ++w) {
    const uint64_t t = wave_lds[w];
    if (w < wave) before += t;
    total += t;
  }
  return before;
}

__device__ __forceinline__ uint32_t key_of(float x) { return f32_order_key(__float_as_uint(x)); }

// Weights relative to the best, in units of 2^-44, and bins.
struct Scale {
  float top;
  double c;  // log2(e) / T
  float cf;  // bins per unit of x
  const double* pow2;

  // 2^44 for the best, 0 below 2^-45 of it (and for -infinity at T = infinity).
  __device__ __forceinline__ uint64_t weight(float x) const {
    const double y = fmax((static_cast<double>(x) - static_cast<double>(top)) * c, -60.0);
    // to the nearest 1/64: the low bits of y + 1.5 2^46 hold 64 y
    const double t = y + 105553116266496.0;
    const int n = static_cast<int>(__double_as_longlong(t));
    const double r = y - (t - 105553116266496.0);
    double q = fma(r, 9.618129107628477e-3, 5.550410866482158e-2);  // ln2^4 / 24, ln2^3 / 6
    q = fma(q, r, 2.402265069591007e-1);                            // ln2^2 / 2
    q = fma(q, r, 6.931471805599453e-1);                            // ln2
    const double b = pow2[n & 63];
    const int64_t w = __double_as_longlong(fma(q * r, b, b)) + (static_cast<int64_t>(n >> 6) << 52);
    // 256 + w has units of 2^-44
    const uint64_t i = static_cast<uint64_t>(__double_as_longlong(256.0 + __longlong_as_double(w)));
    return i - 0x4070000000000000ull;
  }
  // The bin of x; kSmBins or more: no weight.  Never lower for a smaller x.
  __device__ __forceinline__ int bin(float x) const {
    const float y = (top - x) * cf;
    return y < static_cast<float>(kSmBins) ? static_cast<int>(y) : kSmBins;
  }
};

// f(block, first id, words of this lane) over those of the row's blocks that want()
// names, each wave its own, four loads in flight; words past the row and NaN are
// -infinity, infinity the largest finite number.
template <bool BF16, typename W, typename F>
__device__ __forceinline__ void each_block(const SampleArgs& a, int64_t row, int first, int stride, int blocks, W want,
                                           F f) {
  constexpr int kPer = BF16 ? 8 : 4, kAhead = 4;
  const int lane = threadIdx.x & 63;
  const uint16_t* p16 = static_cast<const uint16_t*>(a.x) + row * a.ld;
  const float* p32 = static_cast<const float*>(a.x) + row * a.ld;
  for (int b0 = first; b0 < blocks; b0 += kAhead * stride) {
    uint4 raw[kAhead];
    bool wanted[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int b = b0 + j * stride, i = (b * 64 + lane) * kPer;
      raw[j] = BF16 ? make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u)
                    : make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
      wanted[j] = b < blocks && want(b);
      if (!wanted[j] || i >= a.vocab) continue;
      if (a.wide && i + kPer <= a.vocab) {
        raw[j] = BF16 ? *reinterpret_cast<const uint4*>(p16 + i) : *reinterpret_cast<const uint4*>(p32 + i);
      } else {
        uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (i + e >= a.vocab) continue;
          if (BF16)
            w[e / 2] = (e & 1) ? (w[e / 2] & 0xFFFFu) | (static_cast<uint32_t>(p16[i + e]) << 16)
                               : (w[e / 2] & 0xFFFF0000u) | p16[i + e];
          else
            w[e & 3] = __float_as_uint(p32[i + e]);
        }
        raw[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int b = b0 + j * stride;
      if (!wanted[j]) continue;
      const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
      float x[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        x[e] = __uint_as_float(BF16 ? ((e & 1) ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16) : w[e & 3]);
        x[e] = fminf(fmaxf(x[e], -INFINITY), 3.4028234663852886e38f);
      }
      f(b, (b * 64 + lane) * kPer, x);
    }
  }
}

template <bool BF16>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleArgs a) {
  constexpr int kPer = BF16 ? 8 : 4;
  __shared__ SampleLds s;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int blocks = (a.vocab + 64 * kPer - 1) / (64 * kPer);
  const float T = a.temp ? a.temp[row] : a.temp1;
  const int k = a.top_k ? a.top_k[row] : a.top_k1;
  const float p = a.top_p ? a.top_p[row] : a.top_p1, min_p = a.min_p ? a.min_p[row] : a.min_p1;
  const float u = a.u[row];
  // blocks with a value of at least `floor`
  auto pass = [&](float floor, auto f) {
    each_block<BF16>(a, row, wave, kSmWaves, blocks, [&](int b) { return s.high[b] >= floor; }, f);
  };

  // the best
  float top = -INFINITY;
  each_block<BF16>(a, row, wave, kSmWaves, blocks, [](int) { return true; }, [&](int b, int, const float(&x)[kPer]) {
    float m = x[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) m = fmaxf(m, x[e]);
    m = wave_max_f32(m);
    if (lane == 0) s.high[b] = m;
    top = fmaxf(top, m);
  });
  if (lane == 0) s.top[wave] = top;
  if (tid < 64) s.pow2[tid] = exp2(tid / 64.0);
  if (tid == 0) s.first = a.vocab;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSmWaves; ++w) top = fmaxf(top, s.top[w]);
  if (top == -INFINITY) {  // nothing to draw
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (!(T > 0.f) || k == 1 || p <= 0.f) {  // the best alone: its lowest id
    int at = a.vocab;
    pass(top, [&](int, int i, const float(&x)[kPer]) {
#pragma unroll
      for (int e = kPer - 1; e >= 0; --e)
        if (x[e] == top) at = min(at, i + e);
    });
    if (at < a.vocab) atomicMin(&s.first, at);
    __syncthreads();
    if (tid == 0) a.out[row] = s.first;
    return;
  }
  const double c = 1.4426950408889634074 / static_cast<double>(T);
  const Scale sc{top, c, static_cast<float>(fmin(c * kSmBinsPerOctave, 3e38)), s.pow2};
  // words from here on have weight
  const float reach = static_cast<float>(static_cast<double>(top) - 47.0 / c);
  const uint64_t least =
      min_p > 0.f ? static_cast<uint64_t>(ceil(ldexp(fmin(static_cast<double>(min_p), 1.0), 44))) : 1;
  uint32_t cut_key = 0;
  int cut_id = a.vocab;
  float floor = reach;
  auto kept = [&](uint32_t key, int id) { return key > cut_key || (key == cut_key && id <= cut_id); };
  uint32_t* const count = reinterpret_cast<uint32_t*>(s.hist);

  // The bin where a rule's amount is reached (BY false: `words` words; true:
  // `share` of the kept weight, made a weight here): s.bin, s.above = what lies in
  // the bins before it, s.held = in it.  False if the rule keeps all with weight.
  auto reached = [&](auto by, uint64_t t, uint32_t words, double share) {
    return decltype(by)::value ? static_cast<double>(t) >= share : t >= words;
  };
  auto find_bin = [&](auto by, uint32_t words, double& share) -> bool {
    constexpr bool BY = decltype(by)::value;
    __syncthreads();
    for (int i = tid; i < kSmBins; i += kSmThreads) {
      if (BY) s.hist[i] = 0;
      else count[i] = 0;
    }
    if (tid == 0) s.n = 0;
    __syncthreads();
    const bool all = cut_key == 0;
    pass(floor, [&](int, int i, const float(&x)[kPer]) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int b = sc.bin(x[e]);
        if (BY) {
          if (b < kSmBins && (all || kept(key_of(x[e]), i + e)))
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[b]), sc.weight(x[e]));
        } else if (b < kSmBins) {
          atomicAdd(&count[b], 1u);
        }
      }
    });
    __syncthreads();
    uint64_t v[4], sum = 0, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = BY ? s.hist[4 * tid + j] : count[4 * tid + j];
      sum += v[j];
    }
    uint64_t before = block_before64(sum, s.wave, total);
    if (BY) share *= static_cast<double>(total);
    if (!reached(by, total, words, share) || (!BY && total == words)) return false;
    if (!reached(by, before, words, share) && reached(by, before + sum, words, share)) {
      int j = 0;
      while (!reached(by, before + v[j], words, share)) before += v[j++];
      s.bin = 4 * tid + j;
      s.above = before;
      s.held = v[j];
    }
    __syncthreads();
    return true;
  };
  // x of the first word behind a bin, about: blocks below hold nothing of it
  auto bin_floor = [&](int bin) {
    return fmaxf(reach, static_cast<float>(static_cast<double>(top) - (bin + 2) / (c * kSmBinsPerOctave)));
  };

  // The last word that a rule keeps: the one whose amount before it is the last
  // below the rule's.
  auto cut = [&](auto by, uint32_t words, double share) {
    constexpr bool BY = decltype(by)::value;
    const int bin = s.bin;
    const uint64_t above = s.above;
    auto reached = [&](uint64_t t) { return BY ? static_cast<double>(t) >= share : t >= words; };
    const float low = bin_floor(bin);
    pass(low, [&](int, int i, const float(&x)[kPer]) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (sc.bin(x[e]) != bin) continue;
        const uint32_t key = key_of(x[e]);
        if (!kept(key, i + e)) continue;
        const int at = atomicAdd(&s.n, 1);
        if (at < kSmList) {
          s.key[at] = key;
          s.id[at] = i + e;
          s.w[at] = BY ? sc.weight(x[e]) : 1;
        }
      }
    });
    __syncthreads();
    uint64_t total;
    const int n = s.n;
    if (n <= kSmList) {
      // 2^g threads for each word, its own share of the others each
      const int g = n <= 1 ? 6 : min(6, 10 - (32 - __clz(n - 1))), e = tid >> g;
      uint64_t b = 0;
      if (e < n) {
        const uint32_t key = s.key[e];
        const int id = s.id[e];
        for (int o = tid & ((1 << g) - 1); o < n; o += 1 << g)
          if (s.key[o] > key || (s.key[o] == key && s.id[o] < id)) b += s.w[o];
      }
      for (int o = 1; o < (1 << g); o <<= 1) b += shfl_xor64(b, o);
      if (e < n && (tid & ((1 << g) - 1)) == 0 && !reached(above + b) && reached(above + b + s.w[e])) {
        s.cut_key = s.key[e];
        s.cut_id = s.id[e];
      }
    } else {
      // the order key of the word where the amount is reached, a digit at a time
      uint32_t prefix = 0;
      uint64_t high = above;
      for (int shift = 24; shift >= 0; shift -= 8) {
        const uint32_t mask = shift == 24 ? 0 : ~0u << (shift + 8);
        __syncthreads();
        if (tid < 256) s.hist[tid] = 0;
        __syncthreads();
        pass(low, [&](int, int i, const float(&x)[kPer]) {
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const uint32_t key = key_of(x[e]);
            if (sc.bin(x[e]) != bin || (key & mask) != prefix || !kept(key, i + e)) continue;
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[(key >> shift) & 255]),
                      BY ? sc.weight(x[e]) : 1ull);
          }
        });
        __syncthreads();
        // thread t: digit 255 - t
        const uint64_t mine = tid < 256 ? s.hist[255 - tid] : 0;
        const uint64_t ahead = high + block_before64(mine, s.wave, total);
        if (!reached(ahead) && reached(ahead + mine)) {
          s.bin = 255 - tid;
          s.above = ahead;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(s.bin) << shift;
        high = s.above;
      }
      // of the equal words, the one where it is reached: one block of words at a time
      for (int b = tid; b < kSmBlocks; b += kSmThreads) s.block[b] = 0;
      __syncthreads();
      auto mine_of = [&](int i, const float(&x)[kPer]) {
        uint64_t m = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (key_of(x[e]) == prefix && kept(prefix, i + e)) m += BY ? sc.weight(x[e]) : 1;
        return m;
      };
      pass(low, [&](int b, int i, const float(&x)[kPer]) {
        const uint64_t m = wave_sum64(mine_of(i, x));
        if (lane == 0) s.block[b] = m;
      });
      __syncthreads();
      uint64_t m = tid < blocks ? s.block[tid] : 0;
      uint64_t ahead = high + block_before64(m, s.wave, total);
      if (!reached(ahead) && reached(ahead + m)) {
        s.bin = tid;
        s.above = ahead;
      }
      __syncthreads();
      if (wave == 0) {
        const uint64_t from = s.above;
        each_block<BF16>(a, row, s.bin, kSmBlocks, min(blocks, s.bin + 1), [](int) { return true; }, [&](int, int i, const float(&x)[kPer]) {
          uint64_t at = from + wave_upto64(mine_of(i, x)) - mine_of(i, x);
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            if (key_of(x[e]) != prefix || !kept(prefix, i + e)) continue;
            const uint64_t w = BY ? sc.weight(x[e]) : 1;
            if (!reached(at) && reached(at + w)) {
              s.cut_key = prefix;
              s.cut_id = i + e;
            }
            at += w;
          }
        });
      }
    }
    __syncthreads();
    cut_key = s.cut_key;
    cut_id = s.cut_id;
    floor = low;
  };

  double share = static_cast<double>(p);
  if (k > 0 && k < a.vocab && find_bin(std::false_type(), static_cast<uint32_t>(k), share)) {
    if (k > kSmFew || s.above + s.held > kSmList) {
      cut(std::false_type(), static_cast<uint32_t>(k), share);
    } else {
      // few words: all of the bins up to this one as a list, 2^g threads a word
      const int bin = s.bin, n = static_cast<int>(s.above + s.held);
      pass(bin_floor(bin), [&](int, int i, const float(&x)[kPer]) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (sc.bin(x[e]) > bin) continue;
          const int at = atomicAdd(&s.n, 1);
          s.key[at & (kSmList - 1)] = key_of(x[e]);
          s.id[at & (kSmList - 1)] = i + e;
          s.w[at & (kSmList - 1)] = sc.weight(x[e]);
        }
      });
      __syncthreads();
      const int g = n <= 16 ? 6 : 10 - (32 - __clz(n - 1)), e = tid >> g, sub = tid & ((1 << g) - 1);
      const bool mine = e < n && sub == 0;
      const uint32_t key = e < n ? s.key[e] : 0;
      const int id = e < n ? s.id[e] : 0;
      uint64_t w = e < n ? s.w[e] : 0, total, b = 0;
      int rank = 0;
      for (int o = sub; o < n && e < n; o += 1 << g)
        if (s.key[o] > key || (s.key[o] == key && s.id[o] < id)) {
          b += s.w[o];
          ++rank;
        }
      for (int o = 1; o < (1 << g); o <<= 1) {
        b += shfl_xor64(b, o);
        rank += __shfl_xor(rank, o);
      }
      if (rank >= k) w = 0;
      if (p < 1.f) {
        block_before64(mine ? w : 0, s.wave, total);
        if (!(static_cast<double>(b) < share * static_cast<double>(total))) w = 0;
      }
      if (w < least) w = 0;
      block_before64(mine ? w : 0, s.wave, total);
      if (mine) s.w[e] = w;
      __syncthreads();
      const double target = (u > 0.f ? static_cast<double>(u) : 0.0) * static_cast<double>(total);
      b = 0;
      for (int o = sub; o < n && e < n; o += 1 << g)
        if (s.id[o] < id) b += s.w[o];
      for (int o = 1; o < (1 << g); o <<= 1) b += shfl_xor64(b, o);
      if (mine && w > 0 && (target < static_cast<double>(total)
                                ? static_cast<double>(b) <= target && static_cast<double>(b + w) > target
                                : b + w == total))
        a.out[row] = id;
      return;
    }
  }
  if (p < 1.f && find_bin(std::true_type(), 0, share)) cut(std::true_type(), 0, share);

  // kept weight of each block of words
  const bool all = cut_key == 0;
  auto weights = [&](int i, const float(&x)[kPer], uint64_t(&w)[kPer]) {
    uint64_t sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      w[e] = 0;
      if (!__any(x[e] >= floor)) continue;
      const uint64_t t = sc.weight(x[e]);
      if (t >= least && (all || kept(key_of(x[e]), i + e))) w[e] = t;
      sum += w[e];
    }
    return sum;
  };
  __syncthreads();
  for (int b = tid; b < blocks; b += kSmThreads) s.block[b] = 0;
  __syncthreads();
  pass(floor, [&](int b, int i, const float(&x)[kPer]) {
    uint64_t w[kPer];
    const uint64_t sum = wave_sum64(weights(i, x, w));
    if (lane == 0) s.block[b] = sum;
  });
  __syncthreads();
  const uint64_t mine = tid < blocks ? s.block[tid] : 0;
  uint64_t total;
  const uint64_t before = block_before64(mine, s.wave, total);
  const double target = (u > 0.f ? static_cast<double>(u) : 0.0) * static_cast<double>(total);
  const bool inside = target < static_cast<double>(total);  // else the last word with weight
  if (mine > 0 && (inside ? static_cast<double>(before) <= target && static_cast<double>(before + mine) > target
                          : before + mine == total)) {
    s.bin = tid;
    s.above = before;
  }
  __syncthreads();
  if (wave != 0) return;
  each_block<BF16>(a, row, s.bin, kSmBlocks, s.bin + 1, [](int) { return true; }, [&](int, int i, const float(&x)[kPer]) {
    uint64_t w[kPer];
    const uint64_t sum = weights(i, x, w);
    uint64_t at = s.above + wave_upto64(sum) - sum;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (w[e] > 0 && (inside ? static_cast<double>(at) <= target && static_cast<double>(at + w[e]) > target
                              : at + w[e] == total))
        a.out[row] = i + e;
      at += w[e];
    }
  });
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
  const bool wide = aligned16(logits) && (rows == 1 || ld % (dtype == MOC_BF16 ? 8 : 4) == 0);
  const SampleArgs a{logits, ld, static_cast<int>(vocab), wide, u, temperature, top_p, min_p, top_k,
                     temperature1, top_p1, min_p1, top_k1, out};
  const dim3 grid(static_cast<unsigned>(rows));
  if (dtype == MOC_BF16) sample_kernel<true><<<grid, kSmThreads, 0, as_stream(stream)>>>(a);
  else sample_kernel<false><<<grid, kSmThreads, 0, as_stream(stream)>>>(a);
  return check_launch("sample_kernel");
}
