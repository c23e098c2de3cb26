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
// words would give the neighbour.  So w = 2^y with y in 64 bits, 2^f by a
// polynomial of the eighth degree (the least largest relative error on |f| <= 1/2
// with value 1 at 0: 8.14e-13), held in units of 2^-44.  Sums of these are sums of
// integers (2^18 words: at most 2^62) and have no order, so histograms by atomics
// give the same bits each time.  A weight is off by 8.2e-13 of itself and half a
// unit (2^-45 of the best's, below which it is 0), a sum by at most 8.2e-13 of it
// and 2^-45 for each word (2^18 words: 2^-27): the id is that of exact arithmetic
// unless one of its borders, the draw's, top-p's or min-p's, lies as near as that.  A table of 2^(i/64) takes three
// multiplications fewer and an LDS read, which the histogram's atomics leave no
// time for.
//
// Rules.  Top-k and top-p keep a prefix of one order, so what is kept is its last
// word, (key, id).  It is found with a histogram over the distance from the best
// in 1/88 octaves of weight (numbers of words for top-k, their weights for top-p;
// 4096 bins reach 46.5 octaves, below which a weight is 0) and then among the
// words of the bin where the rule's amount is reached, each against all others;
// where they are too many (equal logits), digit by digit of the order key.  A
// top-k of a few hundred words takes its bin from the largest values of the
// blocks of words: k of them are at or above it.  What lies there goes on as a
// list in LDS.
//
// One workgroup a row: the largest value of each block (16 bytes a lane of a wave),
// the rules, the weights by blocks, the block and then the lane of the draw.  The
// row is read again for each pass (128 KB of 32000 words from L2 at 64 B a clock:
// under a microsecond), blocks whose largest value is below the cut are not.  A row
// that no top-k shortens is bound by the 64-bit arithmetic of its weights, 20
// instructions a word: of 128256 words with top-p 0.95 alone, 78 us, VALU
// instructions issue in two thirds of its CU's clocks, waits for loads, atomics and
// barriers take the rest.  A call of many rows is bound by such rows, a CU each: of
// 256 with settings of their own (106 us; 25 to read them once) the CUs work 40 % of
// the time and issue VALU instructions in 18 % of the clocks, 256 equal ones 99 us,
// 89 % and 50 %.  Few words are bound by the chain of passes and barriers: 16 rows
// of 32000 bf16 words with top-p 27 us, one with top-k 50 12.3.
// Few long rows are spread over several workgroups (below).
#include <algorithm>
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
constexpr int kSmBlocks = kSmMaxVocab / 256;  // blocks of f32 words: 64 a wave
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
  char* ws;  // SampleWs of each row
};

// What the workgroups of a row hand on.
struct SampleWs {
  uint64_t hist[kSmBins];        // top-p's weights by bin
  uint64_t sums[kSmBlocks / 4];  // kept weight of each group of four blocks, without top-p's bin
  uint64_t w[kSmList];           // the words of top-p's bin
  float x[kSmList];
  int id[kSmList];
  float high[kSmBlocks], odd[kSmBlocks];  // of a block: its largest value; 1: it holds NaN or infinity
  int n, unused[3];                       // words of top-p's bin
};

struct SampleLds {
  uint64_t hist[kSmBins];     // weights; as uint32_t: numbers of words
  uint64_t sums[kSmBlocks / 4];  // kept weight of each group of four blocks
  float x[kSmList];
  int id[kSmList];
  uint64_t w[kSmList];
  uint64_t wave[2][kSmWaves];
  float best[kSmWaves], odd[kSmWaves];
  int first;
  int n;
  float cut_x;
  int cut_id;
  int bin;
  uint64_t above, held;
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return __shfl_xor(static_cast<unsigned long long>(v), o);
}

template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
  return dpp_u32<CTRL, ROW_MASK>(static_cast<uint32_t>(v)) |
         (static_cast<uint64_t>(dpp_u32<CTRL, ROW_MASK>(static_cast<uint32_t>(v >> 32))) << 32);
}

__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  return wave_read_lane(static_cast<uint32_t>(v), lane) |
         (static_cast<uint64_t>(wave_read_lane(static_cast<uint32_t>(v >> 32), lane)) << 32);
}

// Sum over the 64 lanes, returned to every lane.
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
  v += dpp_u64<0xB1>(v);
  v += dpp_u64<0x4E>(v);
  v += dpp_u64<0x141>(v);
  v += dpp_u64<0x140>(v);
  return (lane_u64(v, 0) + lane_u64(v, 16)) + (lane_u64(v, 32) + lane_u64(v, 48));
}

// Sum over the lanes up to and with this one (wave_inclusive_scan's steps).
__device__ __forceinline__ uint64_t wave_upto64(uint64_t v) {
  v += dpp_u64<0x111>(v);
  v += dpp_u64<0x112>(v);
  v += dpp_u64<0x114>(v);
  v += dpp_u64<0x118>(v);
  v += dpp_u64<0x142, 0xA>(v);
  v += dpp_u64<0x143, 0xC>(v);
  return v;
}

// Sum over the 64 lanes, returned to every lane.
__device__ __forceinline__ double wave_sum_f64(double v) {
  auto dpp = [](auto ctrl, double x) {
    return __longlong_as_double(static_cast<long long>(dpp_u64<decltype(ctrl)::value>(static_cast<uint64_t>(__double_as_longlong(x)))));
  };
  v += dpp(std::integral_constant<int, 0xB1>(), v);
  v += dpp(std::integral_constant<int, 0x4E>(), v);
  v += dpp(std::integral_constant<int, 0x141>(), v);
  v += dpp(std::integral_constant<int, 0x140>(), v);
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  auto lane = [&](int l) { return __longlong_as_double(static_cast<long long>(lane_u64(b, l))); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// A sum of weights of at most 512 in units of 2^-44.
__device__ __forceinline__ uint64_t units(double s) {
  const double hi = floor(s);
  return (static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 44) +
         (static_cast<uint64_t>(__double_as_longlong(256.0 + (s - hi))) - 0x4070000000000000ull);
}

__device__ __forceinline__ float wave_max_f32(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  v = fmaxf(v, dpp_f32<0x140>(v));
  const float a = __uint_as_float(wave_read_lane(__float_as_uint(v), 0));
  const float b = __uint_as_float(wave_read_lane(__float_as_uint(v), 16));
  const float c = __uint_as_float(wave_read_lane(__float_as_uint(v), 32));
  const float d = __uint_as_float(wave_read_lane(__float_as_uint(v), 48));
  return fmaxf(fmaxf(a, b), fmaxf(c, d));
}

// Sum of v over the threads before this one; total over all.  One barrier:
// calls in a row take turns with the two buffers of the waves' sums.
__device__ __forceinline__ uint64_t block_before64(uint64_t v, uint64_t (&lds)[2][kSmWaves], int& turn, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t upto = wave_upto64(v);
  turn ^= 1;
  if (lane == 63) lds[turn][wave] = upto;
  __syncthreads();
  uint64_t w = lane < kSmWaves ? lds[turn][lane] : 0;
  w += dpp_u64<0x111>(w);
  w += dpp_u64<0x112>(w);
  w += dpp_u64<0x114>(w);
  w += dpp_u64<0x118>(w);
  total = lane_u64(w, kSmWaves - 1);
  return upto - v + (wave > 0 ? lane_u64(w, wave - 1) : 0);
}

__device__ __forceinline__ uint32_t key_of(float x) { return f32_order_key(__float_as_uint(x)); }
__device__ __forceinline__ float of_key(uint32_t q) {
  return __uint_as_float(q & 0x80000000u ? q & 0x7FFFFFFFu : ~q);
}

// True in all lanes if in any.
__device__ __forceinline__ bool any_lane(bool b) { return __builtin_amdgcn_ballot_w64(b) != 0; }

// a b + c with c in scalar registers: the compiler copies c for its two-operand form.
__device__ __forceinline__ double fma_s(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}

// Weights relative to the best, in units of 2^-44, and bins.
struct Scale {
  float top;
  double c;  // log2(e) / T
  float cf;  // bins per unit of x

  // For words of the bins: 256 and the weight, which 256 gives units of 2^-44.
  __device__ __forceinline__ double weight256(float x) const {
    const double y = (static_cast<double>(x) - static_cast<double>(top)) * c;
    const double t = y + 6755399441055744.0;  // 1.5 2^52: y to the nearest integer, in the low bits
    const double f = y - (t - 6755399441055744.0);
    double p = fma_s(f, 1.317893594751445e-06, 1.530915606856033e-05);
    p = fma_s(p, f, 0.00015403825447588072);
    p = fma_s(p, f, 0.0013333454860892282);
    p = fma_s(p, f, 0.009618128616147829);
    p = fma_s(p, f, 0.055504109352659786);
    p = fma_s(p, f, 0.24022650698110454);
    p = fma_s(p, f, 0.6931471805482117);
    p = fma(p, f, 1.0);
    return 256.0 + __builtin_amdgcn_ldexp(p, static_cast<int>(__double_as_longlong(t)));
  }
  // In units of 2^-44: 2^44 for the best, 0 below 2^-45 of it.
  __device__ __forceinline__ uint64_t weight(float x) const {
    return static_cast<uint64_t>(__double_as_longlong(weight256(x))) - 0x4070000000000000ull;
  }
  // As a number; sums of up to 512 of these are exact.
  __device__ __forceinline__ double weight_f64(float x) const { return weight256(x) - 256.0; }
  // The bin of x; kSmBins or more: no weight.  Never lower for a smaller x.
  __device__ __forceinline__ int bin(float x) const {
    const float y = (top - x) * cf;
    return y < static_cast<float>(kSmBins) ? static_cast<int>(y) : kSmBins;
  }
};

// Blocks of a wave: four in a row, then the next four 64 on; bit l of a set and
// lane l stand for block block_of(l, wave).  A group of four is a row of s.sums.
__device__ __forceinline__ int block_of(int l, int wave) { return (l >> 2) * (4 * kSmWaves) + 4 * wave + (l & 3); }

// A row in blocks of 16 bytes a lane.
template <bool BF16>
struct Row {
  static constexpr int kPer = BF16 ? 8 : 4;
  const uint16_t* p16;
  const float* p32;
  int vocab;
  bool wide;

  __device__ __forceinline__ int first(int b) const { return (b * 64 + (threadIdx.x & 63)) * kPer; }
  // Words past the row are -infinity.
  __device__ __forceinline__ uint4 load(int b) const {
    const int i = first(b);
    const uint32_t none = BF16 ? 0xFF80FF80u : 0xFF800000u;
    if (wide && i + kPer <= vocab)
      return BF16 ? *reinterpret_cast<const uint4*>(p16 + i) : *reinterpret_cast<const uint4*>(p32 + i);
    uint32_t w[4] = {none, none, none, none};
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (i + e >= vocab) continue;
      if (BF16)
        w[e / 2] = (e & 1) ? (w[e / 2] & 0xFFFFu) | (static_cast<uint32_t>(p16[i + e]) << 16)
                           : (w[e / 2] & 0xFFFF0000u) | p16[i + e];
      else
        w[e & 3] = __float_as_uint(p32[i + e]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // NaN is -infinity, infinity the largest finite number (PLAIN: the row has neither).
  template <bool PLAIN = false>
  __device__ __forceinline__ void words(const uint4& raw, float (&x)[kPer]) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float v = __uint_as_float(BF16 ? ((e & 1) ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16) : w[e & 3]);
      x[e] = PLAIN ? v : __builtin_amdgcn_fmed3f(v >= -INFINITY ? v : -INFINITY, -INFINITY, 3.4028234663852886e38f);
    }
  }
  // f(block, first id, words of this lane, the block's bit) over this wave's blocks
  // in `set` (block_of), then done(group) after the last of a group of four, whose
  // loads are in flight together.
  template <bool PLAIN = false, typename F, typename G>
  __device__ __forceinline__ void each(uint64_t set, int wave, F f, G done) const {
    while (set != 0) {
      const int group = __builtin_ctzll(set) >> 2;
      const uint32_t four = static_cast<uint32_t>(set >> (4 * group)) & 15u;
      set &= ~(15ull << (4 * group));
      uint4 raw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((four >> j) & 1) raw[j] = load(block_of(4 * group + j, wave));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!((four >> j) & 1)) continue;
        float x[kPer];
        words<PLAIN>(raw[j], x);
        const int b = block_of(4 * group + j, wave);
        f(b, first(b), x, 4 * group + j);
      }
      done(group * kSmWaves + wave);
    }
  }
  template <bool PLAIN = false, typename F>
  __device__ __forceinline__ void each(uint64_t set, int wave, F f) const {
    each<PLAIN>(set, wave, f, [](int) {});
  }
};

// The settings of a row, and whether its weights are summed by several workgroups:
// with top-k the words that count are few, without temperature there is one.
struct Settings {
  float T, p, min_p;
  int k;
  __device__ __forceinline__ Settings(const SampleArgs& a, int64_t row)
      : T(a.temp ? a.temp[row] : a.temp1), p(a.top_p ? a.top_p[row] : a.top_p1),
        min_p(a.min_p ? a.min_p[row] : a.min_p1), k(a.top_k ? a.top_k[row] : a.top_k1) {}
  __device__ __forceinline__ bool best_alone() const { return !(T > 0.f) || k == 1 || p <= 0.f; }
  __device__ __forceinline__ bool shared(int vocab) const { return !best_alone() && !(k > 0 && k < vocab); }
  __device__ __forceinline__ double least() const {
    return min_p > 0.f ? fmin(static_cast<double>(min_p), 1.0) : 0.0;
  }
};

__device__ __forceinline__ Scale scale_of(float top, double c) {
  return Scale{top, c, static_cast<float>(fmin(c * kSmBinsPerOctave, 3e38))};
}
// Words from here on have weight.
__device__ __forceinline__ float reach_of(float top, double c) {
  return fmaxf(static_cast<float>(static_cast<double>(top) - 47.0 / c), -3.4028234663852886e38f);
}
// No word behind a bin is as large.
__device__ __forceinline__ float floor_of_bin(float top, double c, float reach, int bin) {
  return fmaxf(reach, static_cast<float>(static_cast<double>(top) - (bin + 2) / (c * kSmBinsPerOctave)));
}
// Words below have less than min-p.
__device__ __forceinline__ float need_of(float top, double c, float floor, double least) {
  return least > 0.0 ? fmaxf(floor, static_cast<float>(static_cast<double>(top) + (log2(least) - 0.01) / c)) : floor;
}

// ------------------------------------------------- several workgroups a row
// For few long rows: the passes over the whole row by workgroups of four waves, each
// wave groups of four blocks: the blocks' largest values, top-p's histogram, the
// groups' kept weights; sample_kernel takes what they left instead of its own passes.
constexpr int kSmPart = 256;

template <bool BF16>
__global__ __launch_bounds__(kSmPart) void sample_high_kernel(SampleArgs a) {
  constexpr int kPer = BF16 ? 8 : 4;
  const int64_t row = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = (a.vocab + 256 * kPer - 1) / (256 * kPer), stride = 4 * gridDim.x;
  SampleWs& ws = reinterpret_cast<SampleWs*>(a.ws)[row];
  const Row<BF16> words{static_cast<const uint16_t*>(a.x) + row * a.ld, static_cast<const float*>(a.x) + row * a.ld,
                        a.vocab, a.wide};
  for (int i = blockIdx.x * kSmPart + tid; i < kSmBins; i += gridDim.x * kSmPart) ws.hist[i] = 0;
  if (blockIdx.x == 0 && tid == 0) ws.n = 0;
  for (int g = 4 * blockIdx.x + wave; g < groups; g += stride) {
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = words.load(4 * g + j);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[kPer], m = -INFINITY;
      words.template words<true>(raw[j], x);
      bool odd = false;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        odd |= !(x[e] < INFINITY);
        m = fmaxf(m, x[e]);
      }
      m = fminf(wave_max_f32(m), 3.4028234663852886e38f);
      const bool any_odd = any_lane(odd);
      if (lane == 0) {
        ws.high[4 * g + j] = m;
        ws.odd[4 * g + j] = any_odd ? 1.f : 0.f;
      }
    }
  }
}

// The largest value of a row and whether it is plain, for all threads.
__device__ __forceinline__ float best_of(const SampleWs& ws, int blocks, float (&lds)[2][kSmPart / 64], bool& plain) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float top = -INFINITY, odd = 0.f;
  for (int b = tid; b < blocks; b += kSmPart) {
    top = fmaxf(top, ws.high[b]);
    odd = fmaxf(odd, ws.odd[b]);
  }
  top = wave_max_f32(top);
  odd = wave_max_f32(odd);
  if (lane == 0) {
    lds[0][wave] = top;
    lds[1][wave] = odd;
  }
  __syncthreads();
  plain = fmaxf(fmaxf(lds[1][0], lds[1][1]), fmaxf(lds[1][2], lds[1][3])) == 0.f;
  return fmaxf(fmaxf(lds[0][0], lds[0][1]), fmaxf(lds[0][2], lds[0][3]));
}

// f(block, first id, words of this lane) over the blocks of this workgroup's groups
// that have a value of at least `floor`, then done(group) for each group.
template <bool PLAIN, bool BF16, typename F, typename G>
__device__ __forceinline__ void part_of_row(const Row<BF16>& words, const SampleWs& ws, int groups, float floor, F f, G done) {
  for (int g = 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); g < groups; g += 4 * gridDim.x) {
    const float4 high = reinterpret_cast<const float4*>(ws.high)[g];
    const bool in[4] = {high.x >= floor, high.y >= floor, high.z >= floor, high.w >= floor};
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (in[j]) raw[j] = words.load(4 * g + j);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!in[j]) continue;
      float x[Row<BF16>::kPer];
      words.template words<PLAIN>(raw[j], x);
      f(words.first(4 * g + j), x);
    }
    done(g);
  }
}

template <bool BF16>
__global__ __launch_bounds__(kSmPart) void sample_bins_kernel(SampleArgs a) {
  constexpr int kPer = BF16 ? 8 : 4;
  __shared__ uint64_t hist[kSmBins];
  __shared__ float best[2][kSmPart / 64];
  const int64_t row = blockIdx.y;
  const int tid = threadIdx.x;
  const Settings set(a, row);
  if (!set.shared(a.vocab) || !(set.p < 1.f)) return;
  const int groups = (a.vocab + 256 * kPer - 1) / (256 * kPer);
  SampleWs& ws = reinterpret_cast<SampleWs*>(a.ws)[row];
  for (int i = tid; i < kSmBins; i += kSmPart) hist[i] = 0;
  bool plain;
  const float top = best_of(ws, 4 * groups, best, plain);
  if (top == -INFINITY) return;
  const Row<BF16> words{static_cast<const uint16_t*>(a.x) + row * a.ld, static_cast<const float*>(a.x) + row * a.ld,
                        a.vocab, a.wide};
  const double c = 1.4426950408889634074 / static_cast<double>(set.T);
  const Scale sc = scale_of(top, c);
  auto add = [&](int, const float(&x)[kPer]) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = sc.bin(x[e]);
      if (b < kSmBins) atomicAdd(reinterpret_cast<unsigned long long*>(&hist[b]), sc.weight(x[e]));
    }
  };
  if (plain) part_of_row<true>(words, ws, groups, reach_of(top, c), add, [](int) {});
  else part_of_row<false>(words, ws, groups, reach_of(top, c), add, [](int) {});
  __syncthreads();
  for (int i = tid; i < kSmBins; i += kSmPart)
    if (hist[i] != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&ws.hist[i]), hist[i]);
}

template <bool BF16>
__global__ __launch_bounds__(kSmPart) void sample_groups_kernel(SampleArgs a) {
  constexpr int kPer = BF16 ? 8 : 4, kOwn = kSmBins / kSmPart;
  __shared__ float best[2][kSmPart / 64];
  __shared__ uint64_t waves[kSmPart / 64];
  __shared__ int reached;
  const int64_t row = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Settings set(a, row);
  if (!set.shared(a.vocab)) return;
  const int groups = (a.vocab + 256 * kPer - 1) / (256 * kPer);
  SampleWs& ws = reinterpret_cast<SampleWs*>(a.ws)[row];
  bool plain;
  const float top = best_of(ws, 4 * groups, best, plain);
  if (top == -INFINITY) return;
  int border = kSmBins;
  if (set.p < 1.f) {  // the bin that sample_kernel's find_bin finds
    uint64_t v[kOwn], sum = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      v[j] = ws.hist[kOwn * tid + j];
      sum += v[j];
    }
    const uint64_t upto = wave_upto64(sum);
    if (lane == 63) waves[wave] = upto;
    if (tid == 0) reached = kSmBins;
    __syncthreads();
    uint64_t before = upto - sum, total = 0;
#pragma unroll
    for (int w = 0; w < kSmPart / 64; ++w) {
      if (w < wave) before += waves[w];
      total += waves[w];
    }
    const double share = static_cast<double>(set.p) * static_cast<double>(total);
    if (static_cast<double>(before) < share && static_cast<double>(before + sum) >= share) {
      int at = kSmBins;
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        before += v[j];
        if (at == kSmBins && static_cast<double>(before) >= share) at = kOwn * tid + j;
      }
      reached = at;
    }
    __syncthreads();
    border = reached;
  }
  const Row<BF16> words{static_cast<const uint16_t*>(a.x) + row * a.ld, static_cast<const float*>(a.x) + row * a.ld,
                        a.vocab, a.wide};
  const double c = 1.4426950408889634074 / static_cast<double>(set.T), least = set.least();
  const Scale sc = scale_of(top, c);
  const float reach = reach_of(top, c), need = need_of(top, c, reach, least);
  const bool part = border < kSmBins;
  double sum = 0.0;
  auto add = [&](int i, const float(&x)[kPer]) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (part) {
        const int bin = sc.bin(x[e]);
        if (bin > border) continue;
        const double w = sc.weight_f64(x[e]);
        sum += bin < border && w >= least ? w : 0.0;
        if (bin == border) {
          const int at = atomicAdd(&ws.n, 1);
          if (at < kSmList) {
            ws.x[at] = x[e];
            ws.id[at] = i + e;
            ws.w[at] = units(w);
          }
        }
      } else if (x[e] >= need) {
        const double w = sc.weight_f64(x[e]);
        sum += w >= least ? w : 0.0;
      }
    }
  };
  auto done = [&](int group) {
    const uint64_t all = wave_sum64(units(sum));
    if (lane == 0) ws.sums[group] = all;
    sum = 0.0;
  };
  const float floor = part ? floor_of_bin(top, c, reach, border) : need;
  if (plain) part_of_row<true>(words, ws, groups, floor, add, done);
  else part_of_row<false>(words, ws, groups, floor, add, done);
}

// One workgroup a row.  SPLIT: after the three kernels before.
template <bool BF16, bool SPLIT>
__global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleArgs a) {
  constexpr int kPer = BF16 ? 8 : 4;
  __shared__ SampleLds s;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (a.vocab + 64 * kPer - 1) / (64 * kPer);
  const Row<BF16> words{static_cast<const uint16_t*>(a.x) + row * a.ld, static_cast<const float*>(a.x) + row * a.ld,
                        a.vocab, a.wide};
  const Settings set(a, row);
  const float T = set.T, p = set.p, u = a.u[row];
  const int k = set.k;
  const SampleWs* const ws = SPLIT ? reinterpret_cast<const SampleWs*>(a.ws) + row : nullptr;
  const bool shared = SPLIT && set.shared(a.vocab);
  int turn = 0;
  auto before64 = [&](uint64_t v, uint64_t& total) { return block_before64(v, s.wave, turn, total); };

  // the best of each of the wave's blocks, lane l: block_of(l, wave), and of the row
  const int own = 4 * (blocks / (4 * kSmWaves)) + min(max(blocks % (4 * kSmWaves) - 4 * wave, 0), 4);
  float high = -INFINITY;
  bool odd = false;
  if constexpr (SPLIT) {
    if (lane < own) {
      high = ws->high[block_of(lane, wave)];
      odd = ws->odd[block_of(lane, wave)] != 0.f;
    }
  } else {
    words.template each<true>(own >= 64 ? ~0ull : (1ull << own) - 1, wave, [&](int, int, const float(&x)[kPer], int bit) {
      float m = -INFINITY;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        odd |= !(x[e] < INFINITY);
        m = fmaxf(m, x[e]);
      }
      m = fminf(wave_max_f32(m), 3.4028234663852886e38f);
      high = lane == bit ? m : high;
    });
  }
  float top = wave_max_f32(high);
  const bool any_odd = any_lane(odd);
  if (lane == 0) s.odd[wave] = any_odd ? 1.f : 0.f;
  if (lane == 0) s.best[wave] = top;
  if (tid == 0) s.first = a.vocab;
  for (int i = tid; i < kSmBins; i += kSmThreads) s.hist[i] = 0;
  if (tid == 0) s.n = 0;
  __syncthreads();
  top = wave_max_f32(lane < kSmWaves ? s.best[lane] : -INFINITY);
  const bool plain = wave_max_f32(lane < kSmWaves ? s.odd[lane] : 0.f) == 0.f;  // no NaN, no infinity
  if (top == -INFINITY) {  // nothing to draw
    if (tid == 0) a.out[row] = -1;
    return;
  }
  // f over the words of blocks with a value of at least `floor`
  auto pass = [&](float floor, auto f) { words.each(__ballot(high >= floor), wave, f); };
  auto plain_pass = [&](float floor, auto f, auto done) {  // two forms of the code: for the passes that compute much
    if (plain) words.template each<true>(__ballot(high >= floor), wave, f, done);
    else words.each(__ballot(high >= floor), wave, f, done);
  };
  if (set.best_alone()) {  // its lowest id
    int at = a.vocab;
    pass(top, [&](int, int i, const float(&x)[kPer], int) {
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
  const Scale sc = scale_of(top, c);
  const float reach = reach_of(top, c);
  const double least = set.least();
  float cut_x = -INFINITY, floor = reach;
  int cut_id = a.vocab;
  auto kept = [&](float x, int id) { return x > cut_x || (x == cut_x && id <= cut_id); };
  uint32_t* const count = reinterpret_cast<uint32_t*>(s.hist);

  // The bin where a rule's amount is reached (BY false: `wanted` words; true:
  // `share` of the kept weight, made a weight here): s.bin, s.above = what lies in
  // the bins before it, s.held = in it.  False if the rule keeps all with weight.
  // fill() counts into the cleared histogram, which is left clear.
  auto reached = [](auto by, uint64_t t, uint32_t wanted, double share) {
    return decltype(by)::value ? static_cast<double>(t) >= share : t >= wanted;
  };
  auto find_bin = [&](auto by, uint32_t wanted, double& share, auto fill) -> bool {
    constexpr bool BY = decltype(by)::value;
    fill();
    __syncthreads();
    uint64_t v[4], sum = 0, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = BY ? s.hist[4 * tid + j] : count[4 * tid + j];
      sum += v[j];
      if (BY) s.hist[4 * tid + j] = 0;
      else count[4 * tid + j] = 0;
    }
    uint64_t before = before64(sum, total);
    if (BY) share *= static_cast<double>(total);
    if (!reached(by, total, wanted, share) || (!BY && total == wanted)) return false;
    if (!reached(by, before, wanted, share) && reached(by, before + sum, wanted, share)) {
      int j = 0;
      while (!reached(by, before + v[j], wanted, share)) before += v[j++];
      s.bin = 4 * tid + j;
      s.above = before;
      s.held = v[j];
    }
    __syncthreads();
    return true;
  };
  auto count_words = [&] {
    pass(floor, [&](int, int, const float(&x)[kPer], int) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int b = sc.bin(x[e]);
        if (b < kSmBins) atomicAdd(&count[b], 1u);
      }
    });
  };
  auto add_weights_of = [&](auto all) {
    plain_pass(floor, [&](int, int i, const float(&x)[kPer], int) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int b = sc.bin(x[e]);
        if (b < kSmBins && (decltype(all)::value || kept(x[e], i + e)))
          atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[b]), sc.weight(x[e]));
      }
    }, [](int) {});
  };
  auto add_weights = [&] {
    if (cut_x == -INFINITY) add_weights_of(std::true_type());
    else add_weights_of(std::false_type());
  };
  auto bin_floor = [&](int bin) { return floor_of_bin(top, c, reach, bin); };

  // The last word that a rule keeps: the one whose amount before it is the last
  // below the rule's.  After find_bin.
  // listed: the words of the bin are in the list already, if there is room.
  auto cut = [&](auto by, uint32_t wanted, double share, int bin, uint64_t above, bool listed) {
    constexpr bool BY = decltype(by)::value;
    auto full = [&](uint64_t t) { return BY ? static_cast<double>(t) >= share : t >= wanted; };
    const float low = bin_floor(bin), up = static_cast<float>(static_cast<double>(top) - (bin - 1) / (c * kSmBinsPerOctave));
    if (!listed) pass(low, [&](int, int i, const float(&x)[kPer], int) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (!any_lane(x[e] >= low && x[e] <= up)) continue;
        if (sc.bin(x[e]) != bin || !kept(x[e], i + e)) continue;
        const int at = atomicAdd(&s.n, 1);
        if (at < kSmList) {
          s.x[at] = x[e];
          s.id[at] = i + e;
          s.w[at] = BY ? sc.weight(x[e]) : 1;
        }
      }
    });
    __syncthreads();
    const int n = s.n;
    uint64_t total;
    if (n <= kSmList) {
      // 2^g threads for each word, its own share of the others each
      const int g = n <= 16 ? 6 : 10 - (32 - __clz(n - 1)), e = tid >> g;
      uint64_t b = 0;
      if (e < n) {
        const float x = s.x[e];
        const int id = s.id[e];
        for (int o = tid & ((1 << g) - 1); o < n; o += 1 << g)
          if (s.x[o] > x || (s.x[o] == x && s.id[o] < id)) b += s.w[o];
      }
      for (int o = 1; o < (1 << g); o <<= 1) b += shfl_xor64(b, o);
      if (e < n && (tid & ((1 << g) - 1)) == 0 && !full(above + b) && full(above + b + s.w[e])) {
        s.cut_x = s.x[e];
        s.cut_id = s.id[e];
      }
    } else {
      // the order key of the word where the amount is reached, a digit at a time
      uint32_t prefix = 0;
      uint64_t past = above;
      for (int shift = 24; shift >= 0; shift -= 8) {
        const uint32_t mask = shift == 24 ? 0 : ~0u << (shift + 8);
        pass(low, [&](int, int i, const float(&x)[kPer], int) {
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const uint32_t key = key_of(x[e]);
            if (sc.bin(x[e]) != bin || (key & mask) != prefix || !kept(x[e], i + e)) continue;
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[(key >> shift) & 255]), BY ? sc.weight(x[e]) : 1ull);
          }
        });
        __syncthreads();
        // thread t: digit 255 - t
        const uint64_t mine = tid < 256 ? s.hist[255 - tid] : 0;
        if (tid < 256) s.hist[255 - tid] = 0;
        const uint64_t ahead = past + before64(mine, total);
        if (!full(ahead) && full(ahead + mine)) {
          s.bin = 255 - tid;
          s.above = ahead;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(s.bin) << shift;
        past = s.above;
        __syncthreads();
      }
      // of the equal words, the one where it is reached: its group of blocks, its
      // block, its lane
      if (tid < kSmBlocks / 4) s.sums[tid] = 0;
      __syncthreads();
      const float value = of_key(prefix);
      auto mine_of = [&](int i, const float(&x)[kPer]) {
        uint64_t m = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (x[e] == value && kept(value, i + e)) m += BY ? sc.weight(x[e]) : 1;
        return m;
      };
      uint64_t of_group = 0;
      words.each(__ballot(high >= low), wave, [&](int, int i, const float(&x)[kPer], int) { of_group += mine_of(i, x); },
                 [&](int group) {
                   const uint64_t m = wave_sum64(of_group);
                   if (lane == 0) s.sums[group] = m;
                   of_group = 0;
                 });
      __syncthreads();
      const uint64_t m = tid < kSmBlocks / 4 ? s.sums[tid] : 0;
      const uint64_t ahead = past + before64(m, total);
      if (!full(ahead) && full(ahead + m)) {
        s.bin = tid;
        s.above = ahead;
      }
      __syncthreads();
      if (wave == 0) {
        uint64_t from = s.above;
        for (int b = 4 * s.bin; b < 4 * s.bin + 4; ++b) {
          float x[kPer];
          words.words(words.load(b), x);
          const int i = words.first(b);
          const uint64_t of_lane = mine_of(i, x), upto = wave_upto64(of_lane);
          uint64_t at = from + upto - of_lane;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            if (x[e] != value || !kept(value, i + e)) continue;
            const uint64_t w = BY ? sc.weight(x[e]) : 1;
            if (!full(at) && full(at + w)) {
              s.cut_x = value;
              s.cut_id = i + e;
            }
            at += w;
          }
          from += lane_u64(upto, 63);
        }
      }
    }
    __syncthreads();
    cut_x = s.cut_x;
    cut_id = s.cut_id;
    floor = low;
    if (tid == 0) s.n = 0;
  };

  // Draws from the words of the bins up to s.bin, which hold the first k of the
  // row, as a list.  False if they are too many for one.
  double share = static_cast<double>(p);
  auto draw_from_list = [&]() -> bool {
    const int bin = s.bin;
    const float low = bin_floor(bin);
    pass(low, [&](int, int i, const float(&x)[kPer], int) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if (!any_lane(x[e] >= low)) continue;
        if (sc.bin(x[e]) > bin) continue;
        const int at = atomicAdd(&s.n, 1);
        if (at < kSmList) {
          s.x[at] = x[e];
          s.id[at] = i + e;
          s.w[at] = sc.weight(x[e]);
        }
      }
    });
    __syncthreads();
    const int n = s.n;
    if (n > kSmList) {
      __syncthreads();
      if (tid == 0) s.n = 0;
      return false;
    }
    // 2^g threads a word
    const int g = n <= 16 ? 6 : 10 - (32 - __clz(n - 1)), e = tid >> g, sub = tid & ((1 << g) - 1);
    const bool mine = e < n && sub == 0;
    const float x = e < n ? s.x[e] : 0.f;
    const int id = e < n ? s.id[e] : 0;
    uint64_t w = e < n ? s.w[e] : 0, total, b = 0;
    int rank = 0;
    for (int o = sub; o < n && e < n; o += 1 << g)
      if (s.x[o] > x || (s.x[o] == x && s.id[o] < id)) {
        b += s.w[o];
        ++rank;
      }
    for (int o = 1; o < (1 << g); o <<= 1) {
      b += shfl_xor64(b, o);
      rank += __shfl_xor(rank, o);
    }
    if (rank >= k) w = 0;
    if (p < 1.f) {
      before64(mine ? w : 0, total);
      if (!(static_cast<double>(b) < share * static_cast<double>(total))) w = 0;
    }
    if (static_cast<double>(w) < ldexp(least, 44)) w = 0;
    __syncthreads();  // the list's weights are read
    if (mine) s.w[e] = w;
    before64(mine ? w : 0, total);
    const double target = (u > 0.f ? static_cast<double>(u) : 0.0) * static_cast<double>(total);
    b = 0;
    for (int o = sub; o < n && e < n; o += 1 << g)
      if (s.id[o] < id) b += s.w[o];
    for (int o = 1; o < (1 << g); o <<= 1) b += shfl_xor64(b, o);
    if (mine && w > 0 && (target < static_cast<double>(total)
                              ? static_cast<double>(b) <= target && static_cast<double>(b + w) > target
                              : b + w == total))
      a.out[row] = id;
    return true;
  };
  if (k > 0 && k < a.vocab) {
    const uint32_t wanted = static_cast<uint32_t>(k);
    const std::false_type by_words;
    if (k <= kSmFew && k < blocks && find_bin(by_words, wanted, share, [&] {
          const int b = sc.bin(high);
          if (lane < own && b < kSmBins) atomicAdd(&count[b], 1u);
        }) && draw_from_list())
      return;
    __syncthreads();
    if (find_bin(by_words, wanted, share, count_words)) {
      if (k <= kSmFew && s.above + s.held <= kSmList) {
        draw_from_list();
        return;
      }
      cut(by_words, wanted, share, s.bin, s.above, false);
      __syncthreads();
    }
  }
  const bool by_share = p < 1.f && find_bin(std::true_type(), 0, share, [&] {
    if (!shared) return add_weights();
    for (int i = tid; i < kSmBins; i += kSmThreads) s.hist[i] = ws->hist[i];
  });
  const int border = by_share ? s.bin : kSmBins;
  const uint64_t above = by_share ? s.above : 0;
  if (tid < kSmBlocks / 4) s.sums[tid] = 0;
  __syncthreads();

  // kept weight of each group of blocks, those of top-p's bin in the list for now
  float need = need_of(top, c, floor, least);
  auto by_groups = [&](auto part, auto simple) {  // simple: no top-k, no min-p
    constexpr bool SIMPLE = decltype(simple)::value;
    double sum = 0.0;
    plain_pass(decltype(part)::value ? fmaxf(floor, bin_floor(border)) : need, [&](int, int i, const float(&x)[kPer], int) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        if constexpr (decltype(part)::value) {
          const int bin = sc.bin(x[e]);
          if (bin <= border && (SIMPLE || kept(x[e], i + e))) {
            const double w = sc.weight_f64(x[e]);
            sum += bin < border && (SIMPLE || w >= least) ? w : 0.0;
            if (bin == border) {
              const int at = atomicAdd(&s.n, 1);
              if (at < kSmList) {
                s.x[at] = x[e];
                s.id[at] = i + e;
                s.w[at] = units(w);
              }
            }
          }
        } else if (x[e] >= need && (SIMPLE || kept(x[e], i + e))) {
          const double w = sc.weight_f64(x[e]);
          sum += SIMPLE || w >= least ? w : 0.0;
        }
      }
    }, [&](int group) {
      const uint64_t all = wave_sum64(units(sum));
      if (lane == 0) s.sums[group] = all;
      sum = 0.0;
    });
  };
  const bool simple = cut_x == -INFINITY && least == 0.0;
  if (shared) {
    if (tid < (blocks + 3) / 4) s.sums[tid] = ws->sums[tid];
    if (by_share && tid < min(ws->n, kSmList)) {
      s.x[tid] = ws->x[tid];
      s.id[tid] = ws->id[tid];
      s.w[tid] = ws->w[tid];
    }
    if (by_share && tid == 0) s.n = ws->n;
  }
  if (by_share) {
    if (shared) {
    } else if (simple) by_groups(std::true_type(), std::true_type());
    else by_groups(std::true_type(), std::false_type());
    __syncthreads();
    const int n = s.n;
    cut(std::true_type(), 0, share, border, above, true);
    if (n <= kSmList) {
      if (tid < n && kept(s.x[tid], s.id[tid]) && static_cast<double>(s.w[tid]) >= ldexp(least, 44)) {
        const int b = s.id[tid] / (64 * kPer);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.sums[b / 4]), s.w[tid]);
      }
    } else {  // the cut took the table; and it is known now
      __syncthreads();
      if (tid < kSmBlocks / 4) s.sums[tid] = 0;
      __syncthreads();
      need = fmaxf(need, floor);
      by_groups(std::false_type(), std::false_type());
    }
  } else if (shared) {
  } else if (simple) {
    by_groups(std::false_type(), std::true_type());
  } else {
    by_groups(std::false_type(), std::false_type());
  }
  __syncthreads();
  const uint64_t mine = tid < kSmBlocks / 4 ? s.sums[tid] : 0;
  uint64_t total;
  const uint64_t before = before64(mine, total);
  const double target = (u > 0.f ? static_cast<double>(u) : 0.0) * static_cast<double>(total);
  const bool inside = target < static_cast<double>(total);  // else the last word with weight
  if (mine > 0 && (inside ? static_cast<double>(before) <= target && static_cast<double>(before + mine) > target
                          : before + mine == total)) {
    s.bin = tid;
    s.above = before;
  }
  __syncthreads();
  // a wave for each block of the group
  uint64_t w[kPer], sum = 0, upto = 0;
  int i = 0;
  if (wave < 4) {
    float x[kPer];
    words.words(words.load(4 * s.bin + wave), x);
    i = words.first(4 * s.bin + wave);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      w[e] = 0;
      if (x[e] >= floor && kept(x[e], i + e)) {
        const double v = sc.weight_f64(x[e]);
        w[e] = v >= least ? units(v) : 0;
      }
      sum += w[e];
    }
    upto = wave_upto64(sum);
    if (lane == 63) s.hist[wave] = upto;
  }
  __syncthreads();
  if (wave >= 4) return;
  uint64_t at = s.above + upto - sum;
  for (int j = 0; j < wave; ++j) at += s.hist[j];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    if (w[e] > 0 && (inside ? static_cast<double>(at) <= target && static_cast<double>(at + w[e]) > target
                            : at + w[e] == total))
      a.out[row] = i + e;
    at += w[e];
  }
}

}  // namespace
}  // namespace moc

using namespace moc;

namespace {
// Three launches more pay where a pass of one workgroup takes longer and CUs are idle.
// f32 rows with top-p 0.95, us split and by one workgroup a row: 1 x 32000 28, 27; 1 x
// 50257 27, 36; 1 x 128256 30, 78; 16 x 128256 42, 81; 64 x 128256 66, 88; 128 x 128256
// 92, 93; 256 x 128256 138, 99.  With top-k 50, 1 x 32000 17, 14; 1 x 128256 18, 22.
constexpr int64_t kSmSplitVocab = 49152;

bool sample_splits(int64_t rows, int64_t vocab) { return vocab >= kSmSplitVocab && rows <= cu_count() / 4; }

template <bool BF16>
int launch_sample(const SampleArgs& a, int64_t rows, hipStream_t st) {
  if (a.ws == nullptr) {
    sample_kernel<BF16, false><<<static_cast<unsigned>(rows), kSmThreads, 0, st>>>(a);
    return check_launch("sample_kernel");
  }
  // four workgroups a CU, each wave at least one group
  const int64_t per = BF16 ? 8 : 4, groups = (a.vocab + 256 * per - 1) / (256 * per);
  const int64_t parts = std::max<int64_t>(1, std::min((groups + 3) / 4, (4 * cu_count() + rows - 1) / rows));
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(rows));
  sample_high_kernel<BF16><<<grid, kSmPart, 0, st>>>(a);
  int rc = check_launch("sample_high_kernel");
  if (rc != MOC_OK) return rc;
  sample_bins_kernel<BF16><<<grid, kSmPart, 0, st>>>(a);
  rc = check_launch("sample_bins_kernel");
  if (rc != MOC_OK) return rc;
  sample_groups_kernel<BF16><<<grid, kSmPart, 0, st>>>(a);
  rc = check_launch("sample_groups_kernel");
  if (rc != MOC_OK) return rc;
  sample_kernel<BF16, true><<<static_cast<unsigned>(rows), kSmThreads, 0, st>>>(a);
  return check_launch("sample_kernel");
}
}  // namespace

extern "C" int64_t moc_sample_tokens_workspace_size(int64_t rows, int64_t vocab) {
  return rows > 0 && vocab > 0 && vocab <= kSmMaxVocab && sample_splits(rows, vocab)
             ? rows * static_cast<int64_t>(sizeof(SampleWs)) : 0;
}

extern "C" int moc_sample_tokens_ws(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t ld, const float* u,
                                    const float* temperature, float temperature1, const int32_t* top_k, int top_k1,
                                    const float* top_p, float top_p1, const float* min_p, float min_p1, int64_t* out,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  MOC_REQUIRE(dtype == MOC_BF16 || dtype == MOC_F32, "moc_sample_tokens: logits must be bf16 or f32");
  MOC_REQUIRE(rows >= 0 && vocab >= 1 && vocab <= kSmMaxVocab && ld >= 0 && rows < (1LL << 31),
              "moc_sample_tokens: 1 to %lld words a row", (long long)kSmMaxVocab);
  if (rows == 0) return MOC_OK;
  MOC_REQUIRE(logits && u && out, "moc_sample_tokens: null pointer");
  const int64_t need = moc_sample_tokens_workspace_size(rows, vocab);
  MOC_REQUIRE(workspace == nullptr || (aligned16(workspace) && workspace_bytes >= need),
              "moc_sample_tokens: workspace of %lld bytes required", (long long)need);
  const bool wide = aligned16(logits) && (rows == 1 || ld % (dtype == MOC_BF16 ? 8 : 4) == 0);
  const SampleArgs a{logits, ld, static_cast<int>(vocab), wide, u, temperature, top_p, min_p, top_k,
                     temperature1, top_p1, min_p1, top_k1, out, need > 0 ? static_cast<char*>(workspace) : nullptr};
  return dtype == MOC_BF16 ? launch_sample<true>(a, rows, as_stream(stream))
                           : launch_sample<false>(a, rows, as_stream(stream));
}

extern "C" int moc_sample_tokens(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t ld, const float* u,
                                 const float* temperature, float temperature1, const int32_t* top_k, int top_k1,
                                 const float* top_p, float top_p1, const float* min_p, float min_p1, int64_t* out,
                                 void* stream) {
  return moc_sample_tokens_ws(dtype, logits, rows, vocab, ld, u, temperature, temperature1, top_k, top_k1, top_p, top_p1,
                              min_p, min_p1, out, nullptr, 0, stream);
}
