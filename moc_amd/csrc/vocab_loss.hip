// Losses over a vocabulary (gfx950): cross entropy against labels and the
// divergence from a teacher's top logits, of logits that the caller holds or
// of hidden rows through the head's weight, with their gradients.
//
// Row r has words i with shares q_i (sum 1; a label is one word of share 1), a
// weight w_r and logits z; with the temperature T and p = softmax(z / T)
//   l_r = T^2 sum_i q_i (ln q_i - ln p_i),  loss = sum_r w_r l_r / n
//   d loss / d z_j = T w_r / n (p_j - sum_{i: word i = j} q_i)
// where n is the sum of the weights (mean) or 1 (sum).  A row of weight 0, one
// whose label is the ignored one and one without words count for nothing, what
// is in them included: their gradient is 0 and n leaves them out.
//
// Logits are kept in units of log2(e) / T behind the first load, so an
// exponential is one v_exp_f32.  Sums over rows are in 64 bits and in a fixed
// order.
#include "abi.h"
#include "common.h"

namespace moc {
namespace {

constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kMaxWords = 1024;
constexpr int32_t kNoWord = 0x7FFFFFFF;  // behind the words of a row
constexpr int32_t kUnknown = -2;         // a label outside the vocabulary

// What the losses read of the targets, in one buffer (targets_layout).
struct Targets {
  double* total;    // sum of the weights (1 for a sum of losses)
  float* factor;    // upstream gradient / total
  float* largest;   // a power of two, no weight above it; 0: no row counts
  float* alpha;     // [2] what the f16 products for dhidden and dweight are times
  float* weight;    // [rows], 0: the row counts for nothing
  float* entropy;   // [rows] sum of q ln q (teacher only)
  int32_t* ids;     // [rows][words] ascending, kNoWord behind the last
  float* share;     // [rows][words] (teacher only); a word's second entry: -1
  uint16_t* first;  // [slabs + 1][rows] (teacher only) words left of each slab
};

int64_t slabs_of(int64_t vocab) { return (vocab + kLossSlab - 1) / kLossSlab; }

int64_t align256(int64_t n) { return (n + 255) & ~255LL; }

// words = 0: labels.
int64_t targets_layout(int64_t rows, int64_t words, int64_t vocab, char* base, Targets* t) {
  int64_t at = 256;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return base + here;
  };
  char* weight = take(rows * 4);
  char* ids = take(rows * (words > 0 ? words : 1) * 4);
  char* entropy = words > 0 ? take(rows * 4) : nullptr;
  char* share = words > 0 ? take(rows * words * 4) : nullptr;
  char* first = words > 0 ? take(rows * (slabs_of(vocab) + 1) * 2) : nullptr;
  if (t != nullptr) {
    t->total = reinterpret_cast<double*>(base);
    t->factor = reinterpret_cast<float*>(base + 8);
    t->largest = reinterpret_cast<float*>(base + 12);
    t->alpha = reinterpret_cast<float*>(base + 16);
    t->weight = reinterpret_cast<float*>(weight);
    t->ids = reinterpret_cast<int32_t*>(ids);
    t->entropy = reinterpret_cast<float*>(entropy);
    t->share = reinterpret_cast<float*>(share);
    t->first = reinterpret_cast<uint16_t*>(first);
  }
  return at;
}

// Sum or maximum over a workgroup of up to 1024 threads, in wave order.
template <bool MAX>
__device__ __forceinline__ float block_reduce(float v, float* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if (MAX) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  } else {
    v = wave_sum(v);
  }
  __syncthreads();
  if (lane == 0) red[wave] = v;
  __syncthreads();
  float t = red[0];
  for (int w = 1; w < waves; ++w) t = MAX ? fmaxf(t, red[w]) : t + red[w];
  return t;
}

__device__ __forceinline__ double block_sum64(double v, double* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if (lane == 0) red[wave] = v;
  __syncthreads();
  double t = red[0];
  for (int w = 1; w < waves; ++w) t += red[w];
  return t;
}

// ------------------------------------------------------------------ targets
// Weight of a label's row.
__device__ __forceinline__ float label_weight(int64_t label, int64_t ignore, const float* row_weight, int64_t r) {
  return label == ignore ? 0.f : row_weight != nullptr ? row_weight[r] : 1.f;
}

// The least power of two, a normal number, that x >= 0 is not above.
__device__ __forceinline__ float power_above(float x) {
  const uint32_t up = (__float_as_uint(x) + 0x7FFFFFu) >> 23;
  return __uint_as_float((up < 1 ? 1u : up > 254 ? 254u : up) << 23);
}

__device__ __forceinline__ void put_total(const Targets& t, double s, float most, int mean, const float* grad) {
  if (!mean) s = 1.0;
  *t.total = s;
  *t.factor = static_cast<float>((grad != nullptr ? static_cast<double>(*grad) : 1.0) / s);
  *t.largest = most > 0.f ? power_above(most) : 0.f;
}

// Workgroup 0 sums the weights beside the others, which write the rows' targets.
__global__ __launch_bounds__(1024) void label_targets_kernel(const int64_t* __restrict__ labels, int64_t rows,
                                                            int64_t vocab, int64_t ignore,
                                                            const float* __restrict__ row_weight, int mean,
                                                            const float* __restrict__ grad, Targets t) {
  if (blockIdx.x == 0) {
    __shared__ double red[16];
    __shared__ float most[16];
    double s = 0;
    float m = 0.f;
#pragma unroll 8
    for (int64_t r = threadIdx.x; r < rows; r += 1024) {
      const float w = label_weight(labels[r], ignore, row_weight, r);
      s += w;
      m = fmaxf(m, fabsf(w));
    }
    s = block_sum64(s, red);
    m = block_reduce<true>(m, most);
    if (threadIdx.x == 0) put_total(t, s, m, mean, grad);
    return;
  }
  const int64_t r = (static_cast<int64_t>(blockIdx.x) - 1) * 1024 + threadIdx.x;
  if (r >= rows) return;
  const int64_t label = labels[r];
  t.weight[r] = label_weight(label, ignore, row_weight, r);
  t.ids[r] = label == ignore ? kNoWord : label >= 0 && label < vocab ? static_cast<int32_t>(label) : kUnknown;
}

// One wave a row of up to 64 words, a lane a word; as the kernel below.
template <typename ID, bool TOP_F32>
__global__ __launch_bounds__(256) void teacher_wave_kernel(const ID* __restrict__ ids, int64_t ids_ld,
                                                           const void* __restrict__ top, int64_t top_ld, int64_t rows,
                                                           int words, int64_t vocab, float heat,
                                                           const float* __restrict__ row_weight, Targets t) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (r >= rows) return;
  int32_t id = kNoWord;
  float x = -INFINITY;
  if (lane < words) {
    const int64_t word = static_cast<int64_t>(ids[r * ids_ld + lane]);
    x = (TOP_F32 ? static_cast<const float*>(top)[r * top_ld + lane]
                 : bf16_to_f32(static_cast<const uint16_t*>(top)[r * top_ld + lane])) / heat;
    if (word >= 0 && word < vocab && x != -INFINITY) id = static_cast<int32_t>(word);
    else x = -INFINITY;
  }
  const bool some = __any(id != kNoWord);
  float mx = x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  float q = id == kNoWord ? 0.f : exp2f((x - mx) * kLog2E);
  q = q / wave_sum(q);
  int rank = 0;
  for (int j = 0; j < words; ++j) {
    const int32_t other = __builtin_amdgcn_readlane(id, j);
    rank += other < id || (other == id && j < lane);
  }
  if (lane >= words) rank = lane;
  id = __builtin_amdgcn_ds_permute(rank * 4, id);
  q = __int_as_float(__builtin_amdgcn_ds_permute(rank * 4, __float_as_int(q)));
  // a word's first entry gets the shares of the others, which follow it
  const int32_t before = __shfl_up(id, 1);
  const bool head = id != kNoWord && (lane == 0 || before != id);
  float share = q;
  for (int o = 1; o < words; ++o) {
    const bool same = __shfl_down(id, o) == id && id != kNoWord && lane + o < 64;
    const float other = __shfl_down(q, o);
    if (!__any(same)) break;
    if (same) share += other;
  }
  const float h = wave_sum(head && (share > 0.f || share != share) ? share * logf(share) : 0.f);
  if (lane < words) {
    t.ids[r * words + lane] = id;
    t.share[r * words + lane] = head ? share : -1.f;
  }
  if (lane == 0) {
    t.weight[r] = !some ? 0.f : row_weight != nullptr ? row_weight[r] : 1.f;
    t.entropy[r] = some ? h : 0.f;
  }
}

// One workgroup a row.  Words sorted by rank (ties by place); entries of the
// same word become one with the sum of their shares.
template <typename ID, bool TOP_F32>
__global__ __launch_bounds__(256) void teacher_targets_kernel(const ID* __restrict__ ids, int64_t ids_ld,
                                                              const void* __restrict__ top, int64_t top_ld, int words,
                                                              int64_t vocab, float heat,
                                                              const float* __restrict__ row_weight, Targets t) {
  __shared__ int32_t id[kMaxWords], sorted_id[kMaxWords];
  __shared__ float q[kMaxWords], sorted_q[kMaxWords];
  __shared__ float red[4];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  float mx = -INFINITY, any = 0.f;
  bool bad = false;
  for (int k = tid; k < words; k += 256) {
    const int64_t word = static_cast<int64_t>(ids[r * ids_ld + k]);
    const float x = (TOP_F32 ? static_cast<const float*>(top)[r * top_ld + k]
                             : bf16_to_f32(static_cast<const uint16_t*>(top)[r * top_ld + k])) / heat;
    const bool there = word >= 0 && word < vocab && x != -INFINITY;
    id[k] = there ? static_cast<int32_t>(word) : kNoWord;
    q[k] = there ? x : -INFINITY;
    if (there) {
      any = 1.f;
      mx = fmaxf(mx, x);
      bad |= !(x < INFINITY);
    }
  }
  any = block_reduce<true>(any, red);
  if (any == 0.f) {  // uniform: no words
    for (int k = tid; k < words; k += 256) {
      t.ids[r * words + k] = kNoWord;
      t.share[r * words + k] = -1.f;
    }
    if (tid == 0) {
      t.weight[r] = 0.f;
      t.entropy[r] = 0.f;
    }
    return;
  }
  mx = block_reduce<true>(bad ? INFINITY : mx, red);
  float sum = 0.f;
  for (int k = tid; k < words; k += 256) {
    const float e = id[k] == kNoWord ? 0.f : exp2f((q[k] - mx) * kLog2E);
    sum += e;
    q[k] = e;
  }
  sum = block_reduce<false>(sum, red);  // its barriers publish id and q
  for (int k = tid; k < words; k += 256) {
    const int32_t mine = id[k];
    int rank = 0;
    for (int j = 0; j < words; ++j) rank += id[j] < mine || (id[j] == mine && j < k);
    sorted_id[rank] = mine;
    sorted_q[rank] = q[k] / sum;
  }
  __syncthreads();
  float h = 0.f;
  for (int k = tid; k < words; k += 256) {
    const int32_t mine = sorted_id[k];
    float share = -1.f;
    if (mine != kNoWord && (k == 0 || sorted_id[k - 1] != mine)) {
      share = sorted_q[k];
      for (int j = k + 1; j < words && sorted_id[j] == mine; ++j) share += sorted_q[j];
      h += share > 0.f || share != share ? share * logf(share) : 0.f;
    }
    t.ids[r * words + k] = mine;
    t.share[r * words + k] = share;
  }
  h = block_reduce<false>(h, red);
  if (tid == 0) {
    t.weight[r] = row_weight != nullptr ? row_weight[r] : 1.f;
    t.entropy[r] = h;
  }
}

// How many of a row's words lie left of each slab: 64 rows a workgroup, a lane a
// row, so that the table's lines are written and read whole; each of the 16 waves
// walks a sixteenth of the slabs along its rows' words, which stand in LDS up to
// kWordsLds of them (a chain of loads from memory otherwise: 8192 rows of 64 words
// 22 us, 500 slabs).
constexpr int kWordsLds = 200;

__global__ __launch_bounds__(1024) void words_left_kernel(const int32_t* __restrict__ ids, int64_t rows, int words,
                                                          int slabs, uint16_t* __restrict__ first) {
  extern __shared__ int32_t held[];  // [64][words | 1]
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * 64, r = r0 + (threadIdx.x & 63);
  const int32_t* mine = ids + r * words;
  if (words <= kWordsLds) {
    const int n = static_cast<int>(rows - r0 < 64 ? rows - r0 : 64) * words;
    for (int i = threadIdx.x; i < n; i += 1024) held[i / words * (words | 1) + i % words] = ids[r0 * words + i];
    __syncthreads();
    mine = held + (threadIdx.x & 63) * (words | 1);
  }
  if (r >= rows) return;
  const int per = (slabs + 16) / 16, n0 = threadIdx.x / 64 * per;
  int lo = 0, hi = words;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (mine[mid] < n0 * kLossSlab) lo = mid + 1;
    else hi = mid;
  }
  int id = lo < words ? mine[lo] : kNoWord;
  for (int n = n0; n < n0 + per && n <= slabs; ++n) {
    while (id < n * kLossSlab) {
      ++lo;
      id = lo < words ? mine[lo] : kNoWord;
    }
    first[n * rows + r] = static_cast<uint16_t>(lo);
  }
}

// total = sum of the weights or 1, factor = grad / total.  One workgroup.
__global__ __launch_bounds__(1024) void target_total_kernel(int64_t rows, int mean, const float* __restrict__ grad,
                                                            Targets t) {
  __shared__ double red[16];
  __shared__ float most[16];
  double s = 0;
  float m = 0.f;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    s += t.weight[r];
    m = fmaxf(m, fabsf(t.weight[r]));
  }
  s = block_sum64(s, red);
  m = block_reduce<true>(m, most);
  if (threadIdx.x == 0) put_total(t, s, m, mean, grad);
}

// loss = sum of the rows' weighted losses / total.  One workgroup.
__global__ __launch_bounds__(1024) void loss_sum_kernel(const float* __restrict__ row_loss, int64_t rows,
                                                        const double* __restrict__ total, float* __restrict__ loss) {
  __shared__ double red[16];
  double s = 0;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < rows; r += 1024) s += row_loss[r];
  s = block_sum64(s, red);
  if (threadIdx.x == 0) *loss = static_cast<float>(s / *total);
}

// ------------------------------------------------------------------- logits
template <typename T> struct Elem;
template <> struct Elem<uint16_t> {
  static constexpr int kPer = 8;  // elements of a 16-byte chunk
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    return __uint_as_float((e & 1) ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
  }
  static __device__ __forceinline__ float one(uint16_t x) { return bf16_to_f32(x); }
  static __device__ __forceinline__ uint16_t of(float f) { return bf16_rne(f); }
};
template <> struct Elem<_Float16> {
  static __device__ __forceinline__ float one(_Float16 x) { return static_cast<float>(x); }
};
template <> struct Elem<float> {
  static constexpr int kPer = 4;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    return __uint_as_float(w[e]);
  }
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ float of(float f) { return f; }
};

// 16 bytes of a row that starts at any element.
typedef uint32_t chunk_t __attribute__((ext_vector_type(4)));
typedef chunk_t loose2_t __attribute__((aligned(2)));
typedef chunk_t loose4_t __attribute__((aligned(4)));
__device__ __forceinline__ uint4 load_chunk(const uint16_t* p) {
  const chunk_t v = *reinterpret_cast<const loose2_t*>(p);
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint4 load_chunk(const float* p) {
  const chunk_t v = *reinterpret_cast<const loose4_t*>(p);
  return make_uint4(v[0], v[1], v[2], v[3]);
}
// Elements p[0 .. per of the input chunk) = c exp2(unit x - lse).
__device__ __forceinline__ void store_grad(uint16_t* p, const float (&v)[8]) {
  chunk_t o;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    o[q] = __builtin_bit_cast(uint32_t, __builtin_convertvector((cvt_f32x2_t){v[2 * q], v[2 * q + 1]}, cvt_bf16x2_t));
  *reinterpret_cast<loose2_t*>(p) = o;
}
__device__ __forceinline__ void store_grad(float* p, const float (&v)[4]) {
  chunk_t o;
#pragma unroll
  for (int q = 0; q < 4; ++q) o[q] = __float_as_uint(v[q]);
  *reinterpret_cast<loose4_t*>(p) = o;
}

// One workgroup a row: maximum, sum, loss, gradient (dx may be x).  NC > 0: the row
// stays in registers, NC chunks of 16 bytes a thread, all loads in flight before the
// first is used, and LC more in LDS; NC = 0: it is read twice, the second time from
// the caches.
template <typename T, int NC, int TH, int LC = 0>
__global__ __launch_bounds__(TH) void logits_loss_kernel(const T* x, int64_t ld, int vocab, Targets t, int words,
                                                         float heat, float* __restrict__ row_loss, T* dx, int64_t ldd) {
  constexpr int kPer = Elem<T>::kPer, kAhead = 4;
  __shared__ float red[TH / 64], at_word[kMaxWords];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const float w = t.weight[r];
  const T* row = x + r * ld;
  T* out = dx + r * ldd;
  const int full = vocab / kPer, rest = vocab % kPer;  // whole chunks, elements behind them
  if (w == 0.f) {                                      // uniform
    if (dx != nullptr) {
      const float zero[kPer] = {};
      for (int c = tid; c < full; c += TH) store_grad(out + c * kPer, zero);
      if (tid < rest) out[full * kPer + tid] = Elem<T>::of(0.f);
    }
    if (tid == 0) row_loss[r] = 0.f;
    return;
  }
  const float unit = kLog2E / heat;
  const float last = tid < rest ? Elem<T>::one(row[full * kPer + tid]) : -INFINITY;
  uint4 v[NC > 0 ? NC : 1];
  __shared__ uint4 more[LC > 0 ? LC * TH : 1];  // chunks NC .. NC + LC of each thread, read by it alone
  float mx = last, sum = 0.f;
  if constexpr (NC > 0) {
    if (full > 0) {
      // behind the end a thread reads the last chunk again, which leaves the maximum
      // and is not summed
#pragma unroll
      for (int i = 0; i < LC; ++i) v[i] = load_chunk(row + min(tid + TH * (NC + i), full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < LC; ++i) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) mx = fmaxf(mx, Elem<T>::get(v[i], e));
        more[i * TH + tid] = v[i];
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = load_chunk(row + min(tid + TH * i, full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) mx = fmaxf(mx, Elem<T>::get(v[i], e));
    }
    mx = block_reduce<true>(mx, red) * unit;
#pragma unroll
    for (int i = 0; i < LC; ++i)
      if (tid + TH * (NC + i) < full) {
        const uint4 a = more[i * TH + tid];
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += __builtin_amdgcn_exp2f(fmaf(Elem<T>::get(a, e), unit, -mx));
      }
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (tid + TH * i < full)
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += __builtin_amdgcn_exp2f(fmaf(Elem<T>::get(v[i], e), unit, -mx));
    if (tid < rest) sum += __builtin_amdgcn_exp2f(fmaf(last, unit, -mx));
    sum = block_reduce<false>(sum, red);
  } else {
    mx = tid < rest ? last * unit : -INFINITY;
    sum = tid < rest ? (last == last && mx != INFINITY ? 1.f : NAN) : 0.f;
    if (tid < rest && mx == -INFINITY) sum = 0.f;
    for (int c0 = tid; c0 < full; c0 += TH * kAhead) {
      uint4 a[kAhead];
      float m = mx;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) a[i] = load_chunk(row + min(c0 + TH * i, full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) m = fmaxf(m, Elem<T>::get(a[i], e) * unit);
      const float ref = m == -INFINITY ? 0.f : m;
      sum *= mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - ref);  // nothing summed yet, or NaN
      mx = m;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (c0 + TH * i < full)
#pragma unroll
          for (int e = 0; e < kPer; ++e) sum += __builtin_amdgcn_exp2f(fmaf(Elem<T>::get(a[i], e), unit, -ref));
    }
    const float all = block_reduce<true>(mx, red);
    sum *= mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mx - all);
    sum = block_reduce<false>(sum, red);
    mx = all;
  }
  const float lse = mx + log2f(sum);
  const int n = words > 0 ? words : 1;
  float cross = 0.f;
  for (int k = tid; k < n; k += TH) {
    const int32_t id = t.ids[r * n + k];
    if (id == kUnknown) cross = NAN;
    const float share = words > 0 ? t.share[r * n + k] : 1.f;
    if (id < 0 || id == kNoWord || share == -1.f) continue;
    const float l = fmaf(Elem<T>::one(row[id]), unit, -lse);  // log2 p
    at_word[k] = l;
    if (share != 0.f) cross -= share * l;
  }
  cross = block_reduce<false>(cross, red);
  if (tid == 0) row_loss[r] = w * (heat * heat * (cross * kLn2 + (words > 0 ? t.entropy[r] : 0.f)));
  if (dx == nullptr) return;
  const float c = cross == cross ? heat * w * *t.factor : NAN;
  auto grad = [&](const uint4& a, int at) {
    float o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = c * __builtin_amdgcn_exp2f(fmaf(Elem<T>::get(a, e), unit, -lse));
    store_grad(out + at * kPer, o);
  };
  if constexpr (NC > 0) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (tid + TH * i < full) grad(v[i], tid + TH * i);
#pragma unroll
    for (int i = 0; i < LC; ++i)
      if (tid + TH * (NC + i) < full) grad(more[i * TH + tid], tid + TH * (NC + i));
  } else {
    for (int c0 = tid; c0 < full; c0 += TH * kAhead) {
      uint4 a[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) a[i] = load_chunk(row + min(c0 + TH * i, full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (c0 + TH * i < full) grad(a[i], c0 + TH * i);
    }
  }
  if (tid < rest) out[full * kPer + tid] = Elem<T>::of(c * __builtin_amdgcn_exp2f(fmaf(last, unit, -lse)));
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // stored before the words' own
  __syncthreads();
  for (int k = tid; k < n; k += TH) {
    const int32_t id = t.ids[r * n + k];
    const float share = words > 0 ? t.share[r * n + k] : 1.f;
    if (id < 0 || id == kNoWord || share == -1.f) continue;
    out[id] = Elem<T>::of(c * (__builtin_amdgcn_exp2f(at_word[k]) - share));
  }
}

// ------------------------------------------------- logits that were not stored
// Up to 16 rows, losses alone: the weight is read once, straight into the operand
// registers of v_mfma_f32_16x16x32_bf16 (a wave 16 words, a workgroup a slab of 64),
// 16 loads ahead; the rows stand in LDS in fragment order.  Bound by the weight's
// bytes: few_us below.
constexpr int kFewRows = 16, kFewAhead = 16, kFewHidden = 4096;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(256) void few_rows_kernel(const uint16_t* __restrict__ h, int64_t ldh, int rows,
                                                       const uint16_t* __restrict__ w, int64_t ldw, int vocab,
                                                       int hidden, float unit, const int32_t* __restrict__ ids,
                                                       const uint16_t* __restrict__ first, int64_t ld_first, int words,
                                                       float* __restrict__ z, float2* __restrict__ stat, int slabs) {
  extern __shared__ uint4 frag[];  // [steps][64], then the waves' maxima and sums
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int steps = (hidden + 31) / 32;
  float2* part = reinterpret_cast<float2*>(frag + steps * 64);  // [2][4][16]
  const int row = lane & 15, quad = lane >> 4;
  const bool ragged = hidden % 32 != 0 && 32 * (steps - 1) + 8 * quad >= hidden;  // its last chunk lies behind
  auto load = [&](uint4 (&a)[kFewAhead], const uint16_t* src, int s0) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int s = min(s0 + i, steps - 1);
      a[i] = *reinterpret_cast<const uint4*>(src + 32 * (ragged && s == steps - 1 ? 0 : s));
    }
  };
  auto word_of = [&](int slab) {
    return w + static_cast<int64_t>(min(slab * kLossSlab + wave * 16 + row, vocab - 1)) * ldw + 8 * quad;
  };
  uint4 a[kFewAhead], b[kFewAhead];
  int slab = blockIdx.x;
  load(a, word_of(slab), 0);
  for (int i = tid; i < steps * 64; i += 256) {
    const int n = i & 15, k = i / 64 * 32 + 8 * (i % 64 / 16);
    frag[i] = n < rows && k < hidden ? *reinterpret_cast<const uint4*>(h + n * ldh + k) : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  for (int turn = 0; slab < slabs; slab += gridDim.x, turn ^= 1) {
    const uint16_t* src = word_of(slab);
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    auto products = [&](uint4 (&v)[kFewAhead], int s0) {
#pragma unroll
      for (int i = 0; i < kFewAhead; ++i) {
        if (s0 + i >= steps) break;
        uint4 x = v[i];
        if (ragged && s0 + i == steps - 1) x = make_uint4(0, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x),
                                                      __builtin_bit_cast(bf16x8_t, frag[(s0 + i) * 64 + lane]), acc, 0,
                                                      0, 0);
      }
    };
    for (int s0 = 0; s0 < steps; s0 += 2 * kFewAhead) {
      if (s0 + kFewAhead < steps) load(b, src, s0 + kFewAhead);
      products(a, s0);
      if (s0 + 2 * kFewAhead < steps) load(a, src, s0 + 2 * kFewAhead);
      else if (slab + static_cast<int>(gridDim.x) < slabs) load(a, word_of(slab + gridDim.x), 0);
      products(b, s0 + kFewAhead);
    }
    // lane: row, words slab * 64 + wave * 16 + 4 quad + e
    const int c0 = wave * 16 + 4 * quad;
    if (row < rows) {
      int k = first != nullptr ? first[slab * ld_first + row] : 0;
      for (; k < words; ++k) {
        const int c = ids[row * words + k] - slab * kLossSlab - c0;
        if (c >= 4) break;
        if (c >= 0 && c < 4) z[row * words + k] = c == 0 ? acc[0] : c == 1 ? acc[1] : c == 2 ? acc[2] : acc[3];
      }
    }
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[e] = slab * kLossSlab + c0 + e < vocab ? acc[e] * unit : -INFINITY;
      m = fmaxf(m, acc[e]);
    }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(acc[e] - ref);
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16) part[(turn * 4 + wave) * 16 + row] = make_float2(m, s);
    __syncthreads();
    if (tid < rows) {
      float all = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) all = fmaxf(all, part[(turn * 4 + i) * 16 + tid].x);
      const float r = all == -INFINITY ? 0.f : all;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = part[(turn * 4 + i) * 16 + tid];
        sum += v.y * __builtin_amdgcn_exp2f(v.x - r);
      }
      stat[static_cast<int64_t>(tid) * slabs + slab] = make_float2(all, sum);
    }
  }
}

int launch_few(const void* h, int64_t rows, int64_t hidden, int64_t ldh, const void* w, int64_t vocab, int64_t ldw,
               float unit, const Targets& t, int64_t ld_first, int64_t words, float* z, float2* stat, int64_t slabs,
               hipStream_t st) {
  const int steps = static_cast<int>((hidden + 31) / 32);
  const int lds = steps * 1024 + 2 * 4 * 16 * 8;
  const int64_t resident = static_cast<int64_t>(cu_count()) * (160 * 1024 / lds < 8 ? 160 * 1024 / lds : 8);
  const unsigned grid = static_cast<unsigned>(slabs < resident ? slabs : resident);
  few_rows_kernel<<<grid, 256, lds, st>>>(static_cast<const uint16_t*>(h), ldh, (int)rows,
                                          static_cast<const uint16_t*>(w), ldw, (int)vocab, (int)hidden, unit, t.ids,
                                          words > 0 ? t.first : nullptr, ld_first, (int)(words > 0 ? words : 1), z,
                                          stat, (int)slabs);
  return check_launch("few_rows_kernel");
}

// log2 of a row's sum of exponentials from its slabs' maxima and sums; 256 threads,
// a slab's loads in flight with its seven followers'.
__device__ __forceinline__ float slabs_lse(const float2* __restrict__ stat, int slabs, float* red) {
  float m = -INFINITY, s = 0.f;
  for (int i0 = threadIdx.x; i0 < slabs; i0 += 256 * 8) {
    float2 v[8];
    float n = m;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = i0 + 256 * i < slabs ? stat[i0 + 256 * i] : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) n = fmaxf(n, v[i].x);
    const float ref = n == -INFINITY ? 0.f : n;
    s *= m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - ref);  // nothing summed yet, or NaN
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i].y * __builtin_amdgcn_exp2f(v[i].x - ref);
    m = n;
  }
  const float all = block_reduce<true>(m, red);
  s *= m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - all);
  s = block_reduce<false>(s, red);
  return all + log2f(s);
}

// A row's cross entropy sum q (-log2 p) over the words this thread takes, of log2 p
// of each word, which goes to at_word (may be null); NaN for an unknown label.
__device__ __forceinline__ float cross_of(const Targets& t, int64_t r, int words, const float* __restrict__ z,
                                          float unit, float lse, float* at_word, int first, int step) {
  const int n = words > 0 ? words : 1;
  float cross = 0.f;
  for (int k = first; k < n; k += step) {
    const int32_t id = t.ids[r * n + k];
    if (id == kUnknown) cross = NAN;
    const float share = words > 0 ? t.share[r * n + k] : 1.f;
    if (id < 0 || id == kNoWord || share == -1.f) continue;
    const float l = z[r * n + k] * unit - lse;
    if (at_word != nullptr) at_word[k] = l;
    if (share != 0.f) cross -= share * l;
  }
  return cross;
}

// Losses alone: one workgroup a row.
__global__ __launch_bounds__(256) void slabs_loss_kernel(const float2* __restrict__ stat, int slabs, Targets t,
                                                         int words, float heat, const float* __restrict__ z,
                                                         float* __restrict__ row_loss) {
  __shared__ float red[4];
  const int64_t r = blockIdx.x;
  const float w = t.weight[r];
  if (w == 0.f) {  // uniform
    if (threadIdx.x == 0) row_loss[r] = 0.f;
    return;
  }
  const float lse = slabs_lse(stat + r * slabs, slabs, red);
  const float cross = block_reduce<false>(cross_of(t, r, words, z, kLog2E / heat, lse, nullptr, threadIdx.x, 256), red);
  if (threadIdx.x == 0) row_loss[r] = w * (heat * heat * (cross * kLn2 + (words > 0 ? t.entropy[r] : 0.f)));
}

// One workgroup a row: its loss, and its f16 exponentials into gradients of the
// logits, in place: e exp2(m - lse) of a slab's reference m is p.  The gradients stay
// in f16, as (w / largest) 2^14 (p - q): a bf16 rounding of them, 2^-8 of each, would
// add to the products' sums, where the words' parts cancel, more than the sums' own
// rounding (measured: up to 1.9 times the error of f32 ones); 2^-11 does not show.
// Down to 2^-28 of the largest they have all 11 bits, below 2^-39 they are 0.
__global__ __launch_bounds__(256) void slabs_grad_kernel(uint16_t* e, int64_t ld, int vocab,
                                                         const float2* __restrict__ stat, int slabs, Targets t,
                                                         int words, float heat, const float* __restrict__ z,
                                                         float* __restrict__ row_loss) {
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  __shared__ float red[4], at_word[kMaxWords];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const float w = t.weight[r];
  uint4* row = reinterpret_cast<uint4*>(e + r * ld);
  const int chunks = (vocab + 7) / 8;
  if (w == 0.f) {  // uniform
    for (int c = tid; c < chunks; c += 256) row[c] = make_uint4(0, 0, 0, 0);
    if (tid == 0) row_loss[r] = 0.f;
    return;
  }
  const float2* st = stat + r * slabs;
  const float lse = slabs_lse(st, slabs, red);
  const float cross = block_reduce<false>(cross_of(t, r, words, z, kLog2E / heat, lse, at_word, tid, 256), red);
  if (tid == 0) row_loss[r] = w * (heat * heat * (cross * kLn2 + (words > 0 ? t.entropy[r] : 0.f)));
  const float c = cross == cross ? w / *t.largest * 0x1p14f : NAN;
  constexpr int kAhead = 4;
  for (int c0 = tid; c0 < chunks; c0 += 256 * kAhead) {
    uint4 v[kAhead];
    float m[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = min(c0 + 256 * i, chunks - 1);
      v[i] = row[at];
      m[i] = st[at / (kLossSlab / 8)].x;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = c0 + 256 * i;
      if (at >= chunks) break;
      const float f = c * __builtin_amdgcn_exp2f(m[i] - lse - 15.f);
      const uint32_t in[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t out[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, in[q]);
        out[q] = __builtin_bit_cast(uint32_t,
                                    __builtin_convertvector((cvt_f32x2_t){static_cast<float>(h.x) * f,
                                                                          static_cast<float>(h.y) * f},
                                                            f16x2_t));
      }
      row[at] = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // stored before the words' own
  __syncthreads();
  const int n = words > 0 ? words : 1;
  for (int k = tid; k < n; k += 256) {
    const int32_t id = t.ids[r * n + k];
    const float share = words > 0 ? t.share[r * n + k] : 1.f;
    if (id < 0 || id == kNoWord || share == -1.f) continue;
    e[r * ld + id] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(c * (__builtin_amdgcn_exp2f(at_word[k]) - share)));
  }
}

// Rows that count, zeros for the others: what is in those reaches no product (f32).
// Rows of 16-byte chunks, whose last one is cut off at the hidden size.
__global__ __launch_bounds__(256) void counted_rows_kernel(const float* __restrict__ h, int64_t ldh, int64_t rows,
                                                           int hidden, const float* __restrict__ weight,
                                                           float* __restrict__ out, int64_t ldo) {
  const int chunks = (hidden + 3) / 4;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * chunks; i += step) {
    const int64_t r = i / chunks;
    const int k = static_cast<int>(i - r * chunks) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (weight[r] != 0.f) {
      v = *reinterpret_cast<const float4*>(h + r * ldh + k);
      if (k + 1 >= hidden) v.y = 0.f;
      if (k + 2 >= hidden) v.z = 0.f;
      if (k + 3 >= hidden) v.w = 0.f;
    }
    *reinterpret_cast<float4*>(out + r * ldo + k) = v;
  }
}

// ------------------------------------------------------- operands in f16
// Hidden rows and weight for the products with f16 gradients: bf16 values times a
// power of two, which f16 holds as they are from 2^-17 up and rounds by at most 2^-25
// below; rows that do not count become 0.  The power is a guess that suits what
// networks hold (the largest of the hidden rows in [2^-3, 2^13], of the weight in
// [2^-7, 2^9]: what is rounded is off by 2^-24 of the largest at most); the largest
// value is found on the way, and halves_again_kernel redoes a tensor that it does not
// suit.
struct Halves {
  const uint16_t* from;
  int64_t ld, rows;
  _Float16* to;  // null: not wanted
  float guess, least, most;
};

__device__ __forceinline__ float halves_scale(const Halves& h, uint32_t range) {
  const float x = __uint_as_float(range);
  if (range == 0 || !(x < INFINITY) || (x >= h.least && x <= h.most)) return h.guess;
  const int e = static_cast<int>((__float_as_uint(power_above(x)) >> 23)) - 127;  // x <= 2^e
  return ldexpf(1.f, 15 - e < 126 ? 15 - e : 126);
}

// Rows of h by hidden columns into rows of ldo (a multiple of 64, zeros behind the
// hidden size), a wave a row, four rows' loads in flight; the bits of the largest
// |value| this lane met.
__device__ __forceinline__ uint32_t halve_rows(const Halves& h, int hidden, int64_t ldo, const float* weight,
                                               float scale) {
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  constexpr int kRows = 4;
  const int lane = threadIdx.x & 63, chunks = static_cast<int>(ldo / 8);
  const int64_t waves = static_cast<int64_t>(gridDim.x) * 4;
  uint32_t most = 0;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6); r0 < h.rows; r0 += waves * kRows) {
    for (int c = lane; c < chunks; c += 64) {
      const int k = 8 * c;
      uint4 v[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t r = r0 + waves * i;
        v[i] = k < hidden && r < h.rows && (weight == nullptr || weight[r] != 0.f)
                   ? *reinterpret_cast<const uint4*>(h.from + r * h.ld + k)
                   : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t r = r0 + waves * i;
        if (r >= h.rows) break;
        const uint32_t in[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint32_t o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          // what a chunk holds behind the hidden size is another tensor's or padding
          const uint32_t w = in[q] & (k + 2 * q + 1 < hidden ? 0xFFFFFFFFu : k + 2 * q < hidden ? 0xFFFFu : 0u);
          most = max(most, max(w << 16 & 0x7FFF0000u, w & 0x7FFF0000u));
          o[q] = __builtin_bit_cast(uint32_t,
                                    __builtin_convertvector((cvt_f32x2_t){__uint_as_float(w << 16) * scale,
                                                                          __uint_as_float(w & 0xFFFF0000u) * scale},
                                                            f16x2_t));
        }
        *reinterpret_cast<uint4*>(h.to + r * ldo + k) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
  return most;
}

__device__ __forceinline__ uint32_t block_max_bits(uint32_t m, uint32_t* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  return max(max(red[0], red[1]), max(red[2], red[3]));
}

// most [2][gridDim]: the workgroups' largest values (one word for all of them would
// have thousands of atomics in a row: 30 us).
__global__ __launch_bounds__(256) void halves_kernel(Halves hidden_rows, Halves weight_rows, int hidden, int64_t ldo,
                                                     Targets t, uint32_t* __restrict__ most) {
  __shared__ uint32_t red[4];
  uint32_t m = hidden_rows.to != nullptr ? halve_rows(hidden_rows, hidden, ldo, t.weight, hidden_rows.guess) : 0;
  m = block_max_bits(m, red);
  if (threadIdx.x == 0) most[blockIdx.x] = m;
  m = weight_rows.to != nullptr ? halve_rows(weight_rows, hidden, ldo, nullptr, weight_rows.guess) : 0;
  m = block_max_bits(m, red);
  if (threadIdx.x == 0) most[gridDim.x + blockIdx.x] = m;
}

// Redoes a tensor whose largest value the guess did not suit; the products' factors.
__global__ __launch_bounds__(256) void halves_again_kernel(Halves hidden_rows, Halves weight_rows, int hidden,
                                                           int64_t ldo, float heat, Targets t,
                                                           const uint32_t* __restrict__ most, int parts) {
  __shared__ uint32_t red[4];
  uint32_t m[2] = {0, 0};
#pragma unroll 8
  for (int i = threadIdx.x; i < parts; i += 256) {
    m[0] = max(m[0], most[i]);
    m[1] = max(m[1], most[parts + i]);
  }
  const float sx = halves_scale(hidden_rows, block_max_bits(m[0], red));
  const float sw = halves_scale(weight_rows, block_max_bits(m[1], red));
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    // no row counts: gradients of 0, whatever the divisor
    const float f = *t.largest > 0.f ? heat * *t.factor * *t.largest * 0x1p-14f : 0.f;
    t.alpha[0] = f / sw;
    t.alpha[1] = f / sx;
  }
  if (hidden_rows.to != nullptr && sx != hidden_rows.guess) halve_rows(hidden_rows, hidden, ldo, t.weight, sx);
  if (weight_rows.to != nullptr && sw != weight_rows.guess) halve_rows(weight_rows, hidden, ldo, nullptr, sw);
}

// a += b over n values; out (may be null): the sum as bf16 or f32.
template <typename OUT>
__global__ __launch_bounds__(256) void add_f32_kernel(float* a, const float* __restrict__ b, int64_t n, OUT* out) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step) {
    const float s = a[i] + b[i];
    if (out != nullptr) out[i] = Elem<OUT>::of(s);
    else a[i] = s;
  }
}

// out[i][j] = *alpha a_i b_j (alpha null: 1), the product over one row or one word (the engine takes no
// operand of one element's pitch).  Columns blockIdx.x, rows blockIdx.y and on.
template <typename T, typename OUT>
__global__ __launch_bounds__(256) void outer_kernel(const T* __restrict__ a, int64_t lda, const T* __restrict__ b,
                                                    int64_t m, int64_t n, const float* __restrict__ alpha,
                                                    OUT* __restrict__ out) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (j >= n) return;
  const float bj = Elem<T>::one(b[j]) * (alpha != nullptr ? *alpha : 1.f);
  for (int64_t i = blockIdx.y; i < m; i += gridDim.y) out[i * n + j] = Elem<OUT>::of(Elem<T>::one(a[i * lda]) * bj);
}

// p *= *g in place over whole 16-byte chunks and what is behind them.
template <typename T>
__device__ __forceinline__ void scale_values(T* __restrict__ p, int64_t n, float f) {
  constexpr int kPer = Elem<T>::kPer;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256, first = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  for (int64_t i = first; i < n / kPer; i += step) {
    const uint4 v = load_chunk(p + i * kPer);
    float o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = Elem<T>::get(v, e) * f;
    store_grad(p + i * kPer, o);
  }
  if (first < n % kPer) p[n / kPer * kPer + first] = Elem<T>::of(Elem<T>::one(p[n / kPer * kPer + first]) * f);
}

// Two tensors times *g; leaves at once where *g is 1.
__global__ __launch_bounds__(256) void scale_kernel(int f32_0, void* p0, int64_t n0, int f32_1, void* p1, int64_t n1,
                                                    const float* __restrict__ g) {
  const float f = *g;
  if (f == 1.f) return;
  if (f32_0) scale_values(static_cast<float*>(p0), n0, f);
  else scale_values(static_cast<uint16_t*>(p0), n0, f);
  if (f32_1) scale_values(static_cast<float*>(p1), n1, f);
  else scale_values(static_cast<uint16_t*>(p1), n1, f);
}

constexpr int kMostBlocks = 2048;  // of a grid that strides over its work

unsigned blocks_of(int64_t n) {
  const int64_t b = (n + 255) / 256;
  return static_cast<unsigned>(b < 1 ? 1 : b > kMostBlocks ? kMostBlocks : b);
}

// ------------------------------------------------------------------- pieces
// Logits exist for a piece of the rows at a time, within about this many bytes.
constexpr int64_t kPieceBytes = 1LL << 30;

struct Pieces {
  bool fused;              // logits inside the product (launch_loss_gemm), not stored
  int64_t rows, count;     // rows of a piece, pieces
  int64_t ldz;             // row pitch of a piece's logits
  int64_t slabs;
  int64_t z, d, x, w, acc, part, stat, at_words, most, bytes;  // offsets in the workspace
  int64_t ldx;
};

Pieces pieces_of(int dtype, int64_t rows, int64_t hidden, int64_t vocab, int64_t words, bool grads) {
  Pieces p{};
  const bool f32 = dtype == MOC_F32;
  p.fused = !f32;
  p.ldz = (vocab + 63) & ~63LL;
  p.slabs = slabs_of(vocab);
  const int64_t n_words = words > 0 ? words : 1;
  const int64_t each = !p.fused ? p.ldz * 4 : grads ? p.ldz * 2 : p.slabs * 8;
  int64_t n = kPieceBytes / each / 256 * 256;
  if (n < 256) n = 256;
  if (n > rows) n = rows < 1 ? 1 : rows;
  p.rows = n;
  p.count = rows < 1 ? 0 : (rows + n - 1) / n;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  if (p.fused) {
    p.stat = take(n * p.slabs * 8);
    p.at_words = take(n * n_words * 4);
    p.d = grads ? take(n * p.ldz * 2) : 0;
  } else {
    p.z = take(n * p.ldz * 4);
    p.d = p.z;  // in place
  }
  p.ldx = (hidden + 63) & ~63LL;
  p.x = grads ? take(rows * p.ldx * (f32 ? 4 : 2)) : 0;
  p.w = grads && !f32 ? take(vocab * p.ldx * 2) : 0;
  p.most = grads && !f32 ? take(2 * 4 * kMostBlocks) : 0;
  if (grads && p.count > 1) {
    p.acc = take(vocab * hidden * 4);
    p.part = take(vocab * hidden * 4);
  }
  p.bytes = at;
  return p;
}

constexpr int moc_th(int th, int = 0) { return th; }

template <typename T>
void launch_logits(const T* x, int64_t rows, int vocab, int64_t ld, const Targets& t, int words, float heat,
                   float* row_loss, T* dx, int64_t ldd, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(rows));
  const int chunks = vocab / Elem<T>::kPer;
#define MOC_LOGITS(NC, ...) \
  logits_loss_kernel<T, NC, __VA_ARGS__><<<grid, moc_th(__VA_ARGS__), 0, st>>>(x, ld, vocab, t, words, heat, row_loss, dx, ldd)
  if (chunks <= 4 * 256) MOC_LOGITS(4, 256);
  else if (chunks <= 4 * 512) MOC_LOGITS(4, 512);
  else if (chunks <= 8 * 512) MOC_LOGITS(8, 512);
  else if (chunks <= 8 * 1024) MOC_LOGITS(8, 1024);
  else if (chunks <= 16 * 1024) MOC_LOGITS(16, 1024);
  else if (chunks <= 32 * 1024) MOC_LOGITS(24, 1024, 8);
  else MOC_LOGITS(0, 1024);
#undef MOC_LOGITS
}

int logits_rows(bool f32, const void* x, int64_t rows, int64_t vocab, int64_t ld, const Targets& t, int64_t words,
                float heat, float* row_loss, void* dx, int64_t ldd, hipStream_t st) {
  if (rows == 0) return MOC_OK;
  const int v = static_cast<int>(vocab), k = static_cast<int>(words);
  if (f32)
    launch_logits(static_cast<const float*>(x), rows, v, ld, t, k, heat, row_loss, static_cast<float*>(dx), ldd, st);
  else
    launch_logits(static_cast<const uint16_t*>(x), rows, v, ld, t, k, heat, row_loss, static_cast<uint16_t*>(dx), ldd,
                  st);
  return check_launch("logits_loss_kernel");
}

// C [M, N] = *alpha A B over K = 1, as moc_gemm_ws or gemm_half of these strides would.
int outer(bool f32, int64_t m, int64_t n, const void* a, int64_t lda, const void* b, const float* alpha, void* c,
          int c_dtype, hipStream_t st) {
  typedef _Float16 H;
  const dim3 grid(static_cast<unsigned>((n + 255) / 256), static_cast<unsigned>(m < 8192 ? m : 8192));
  if (f32)
    outer_kernel<float, float><<<grid, 256, 0, st>>>(static_cast<const float*>(a), lda, static_cast<const float*>(b), m,
                                                     n, nullptr, static_cast<float*>(c));
  else if (c_dtype == MOC_F32)
    outer_kernel<H, float><<<grid, 256, 0, st>>>(static_cast<const H*>(a), lda, static_cast<const H*>(b), m, n, alpha,
                                                 static_cast<float*>(c));
  else
    outer_kernel<H, uint16_t><<<grid, 256, 0, st>>>(static_cast<const H*>(a), lda, static_cast<const H*>(b), m, n, alpha,
                                                    static_cast<uint16_t*>(c));
  return check_launch("outer_kernel");
}

bool sizes_ok(int64_t rows, int64_t vocab, int64_t words) {
  return rows >= 0 && rows <= (1LL << 24) && vocab >= 1 && vocab <= (1LL << 21) && words >= 0 && words <= kMaxWords;
}

}  // namespace
}  // namespace moc

using namespace moc;

#define MOC_SIZES(name)                                                                                          \
  MOC_REQUIRE(sizes_ok(rows, vocab, words), "%s: up to 2^24 rows, a vocabulary of up to 2^21 words, up to %d of " \
                                            "them a row", name, kMaxWords)

extern "C" int64_t moc_loss_targets_size(int64_t rows, int64_t words, int64_t vocab) {
  if (!sizes_ok(rows, vocab, words)) return 0;
  return targets_layout(rows, words, vocab, nullptr, nullptr);
}

extern "C" int moc_label_targets(const int64_t* labels, int64_t rows, int64_t vocab, int64_t ignore_index,
                                 const float* row_weight, int mean, const float* grad, void* targets, void* stream) {
  const int64_t words = 0;
  MOC_SIZES("moc_label_targets");
  MOC_REQUIRE((labels != nullptr || rows == 0) && targets != nullptr && aligned16(targets),
              "moc_label_targets: null operand or unaligned targets");
  hipStream_t st = as_stream(stream);
  Targets t;
  targets_layout(rows, 0, vocab, static_cast<char*>(targets), &t);
  label_targets_kernel<<<static_cast<unsigned>(1 + (rows + 1023) / 1024), 1024, 0, st>>>(
      labels, rows, vocab, ignore_index, row_weight, mean, grad, t);
  return check_launch("label_targets_kernel");
}

extern "C" int moc_teacher_targets(const void* ids, int ids_dtype, int64_t ids_ld, const void* top, int top_dtype,
                                   int64_t top_ld, int64_t rows, int64_t words, int64_t vocab, float temperature,
                                   const float* row_weight, int mean, const float* grad, void* targets,
                                   void* stream) {
  MOC_SIZES("moc_teacher_targets");
  MOC_REQUIRE(words >= 1, "moc_teacher_targets: a word a row at least");
  MOC_REQUIRE((ids_dtype == MOC_I32 || ids_dtype == MOC_I64) && (top_dtype == MOC_BF16 || top_dtype == MOC_F32),
              "moc_teacher_targets: ids are int32 or int64, the teacher's logits bf16 or f32");
  MOC_REQUIRE(temperature > 0.f && temperature < INFINITY, "moc_teacher_targets: the temperature must be above 0");
  MOC_REQUIRE(rows == 0 || (ids != nullptr && top != nullptr && (rows == 1 || (ids_ld >= words && top_ld >= words))),
              "moc_teacher_targets: null operand or rows that overlap");
  MOC_REQUIRE(targets != nullptr && aligned16(targets), "moc_teacher_targets: null or unaligned targets");
  hipStream_t st = as_stream(stream);
  Targets t;
  targets_layout(rows, words, vocab, static_cast<char*>(targets), &t);
  if (rows > 0) {
    const int k = static_cast<int>(words);
#define MOC_TEACHER(ID, F)                                                                                            \
  (k <= 64 ? teacher_wave_kernel<ID, F><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, st>>>(                        \
                 static_cast<const ID*>(ids), ids_ld, top, top_ld, rows, k, vocab, temperature, row_weight, t) \
           : teacher_targets_kernel<ID, F><<<static_cast<unsigned>(rows), 256, 0, st>>>(                               \
                 static_cast<const ID*>(ids), ids_ld, top, top_ld, k, vocab, temperature, row_weight, t))
    if (ids_dtype == MOC_I32 && top_dtype == MOC_F32) MOC_TEACHER(int32_t, true);
    else if (ids_dtype == MOC_I32) MOC_TEACHER(int32_t, false);
    else if (top_dtype == MOC_F32) MOC_TEACHER(int64_t, true);
    else MOC_TEACHER(int64_t, false);
#undef MOC_TEACHER
    const int rc = check_launch("teacher_targets_kernel");
    if (rc != MOC_OK) return rc;
  }
  target_total_kernel<<<1, 1024, 0, st>>>(rows, mean, grad, t);
  return check_launch("target_total_kernel");
}

extern "C" int moc_logits_loss(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t ld, void* targets,
                               int64_t words, float temperature, float* row_loss, float* loss, void* dlogits,
                               int64_t ldd, void* stream) {
  MOC_SIZES("moc_logits_loss");
  MOC_REQUIRE(dtype == MOC_BF16 || dtype == MOC_F32, "moc_logits_loss: logits are bf16 or f32");
  MOC_REQUIRE(temperature > 0.f && temperature < INFINITY, "moc_logits_loss: the temperature must be above 0");
  MOC_REQUIRE(targets != nullptr && (rows == 0 || (logits != nullptr && row_loss != nullptr)),
              "moc_logits_loss: null operand");
  MOC_REQUIRE(rows <= 1 || (ld >= vocab && (dlogits == nullptr || ldd >= vocab)), "moc_logits_loss: rows that overlap");
  hipStream_t st = as_stream(stream);
  Targets t;
  targets_layout(rows, words, vocab, static_cast<char*>(targets), &t);
  const bool f32 = dtype == MOC_F32;
  int rc = logits_rows(f32, logits, rows, vocab, ld, t, words, temperature, row_loss, dlogits, ldd, st);
  if (rc != MOC_OK || loss == nullptr) return rc;
  loss_sum_kernel<<<1, 1024, 0, st>>>(row_loss, rows, t.total, loss);
  return check_launch("loss_sum_kernel");
}

extern "C" int64_t moc_linear_loss_workspace_size(int dtype, int64_t rows, int64_t hidden, int64_t vocab,
                                                  int64_t words, int grads) {
  if (!sizes_ok(rows, vocab, words) || hidden < 1) return 0;
  return pieces_of(dtype, rows, hidden, vocab, words, grads != 0).bytes;
}

extern "C" int64_t moc_linear_loss_gemm_workspace_size(int dtype, int64_t rows, int64_t hidden, int64_t vocab,
                                                       int grads) {
  if (!sizes_ok(rows, vocab, 0) || hidden < 1) return 0;
  const Pieces p = pieces_of(dtype, rows, hidden, vocab, 0, grads != 0);
  int64_t most = 0;
  for (int64_t i = 0; i < p.count; i += p.count > 1 ? p.count - 1 : 1) {  // the first piece and the last
    const int64_t n = i + 1 < p.count ? p.rows : rows - i * p.rows;
    int64_t b = p.fused ? 0 : moc_gemm_workspace_size(dtype, n, vocab, hidden, 0);
    if (b > most) most = b;
    if (!grads) continue;
    b = p.fused ? gemm_half_workspace(n, hidden, vocab) : moc_gemm_workspace_size(dtype, n, hidden, vocab, 0);
    if (b > most) most = b;
    b = p.fused ? gemm_half_workspace(vocab, hidden, n) : moc_gemm_workspace_size(dtype, vocab, hidden, n, 0);
    if (b > most) most = b;
  }
  return most;
}

extern "C" int moc_linear_loss(int dtype, const void* h, int64_t rows, int64_t hidden, int64_t ldh, const void* w,
                               int64_t vocab, int64_t ldw, void* targets, int64_t words, float temperature,
                               float* row_loss, float* loss, void* dh, int dh_dtype, void* dw, int dw_dtype,
                               void* workspace, int64_t workspace_bytes, void* gemm_ws, int64_t gemm_ws_bytes,
                               void* stream) {
  MOC_SIZES("moc_linear_loss");
  MOC_REQUIRE(dtype == MOC_BF16 || dtype == MOC_F32, "moc_linear_loss: operands are bf16 or f32");
  const bool f32 = dtype == MOC_F32;
  const int es = f32 ? 4 : 2;
  MOC_REQUIRE(hidden >= 1 && hidden <= (1 << 20), "moc_linear_loss: hidden size of 1 to 2^20");
  MOC_REQUIRE(temperature > 0.f && temperature < INFINITY, "moc_linear_loss: the temperature must be above 0");
  MOC_REQUIRE(targets != nullptr && w != nullptr && (rows == 0 || (h != nullptr && row_loss != nullptr)),
              "moc_linear_loss: null operand");
  MOC_REQUIRE(aligned16(h) && aligned16(w) && ldh * es % 16 == 0 && ldw * es % 16 == 0 && ldh >= hidden &&
                  ldw >= hidden,
              "moc_linear_loss: operands need 16-byte aligned rows");
  MOC_REQUIRE(f32 || vocab * ldw * 2 < (1LL << 31) - 1024, "moc_linear_loss: a bf16 weight of up to 2 GiB");
  MOC_REQUIRE((dh == nullptr || (dh_dtype == MOC_F32 || (dh_dtype == MOC_BF16 && !f32))) &&
                  (dw == nullptr || (dw_dtype == MOC_F32 || (dw_dtype == MOC_BF16 && !f32))),
              "moc_linear_loss: gradients are f32, or bf16 of bf16 operands");
  const bool grads = dh != nullptr || dw != nullptr;
  const Pieces p = pieces_of(dtype, rows, hidden, vocab, words, grads);
  MOC_REQUIRE(workspace_bytes >= p.bytes && (workspace != nullptr || p.bytes == 0) && aligned16(workspace),
              "moc_linear_loss: workspace of %lld bytes needed", (long long)p.bytes);
  MOC_REQUIRE(f32 || p.rows * p.ldx * 2 < (1LL << 31) - 1024, "moc_linear_loss: hidden rows of a piece up to 2 GiB");
  hipStream_t st = as_stream(stream);
  Targets t;
  targets_layout(rows, words, vocab, static_cast<char*>(targets), &t);
  char* ws = static_cast<char*>(workspace);
  const int64_t n_words = words > 0 ? words : 1;
  int rc;
  if (grads && rows > 0 && f32) {
    counted_rows_kernel<<<blocks_of(rows * ((hidden + 3) / 4)), 256, 0, st>>>(
        static_cast<const float*>(h), ldh, rows, (int)hidden, t.weight, reinterpret_cast<float*>(ws + p.x), p.ldx);
    if ((rc = check_launch("counted_rows_kernel")) != MOC_OK) return rc;
  } else if (grads && rows > 0) {
    const Halves hx{static_cast<const uint16_t*>(h), ldh, rows,
                    dw != nullptr ? reinterpret_cast<_Float16*>(ws + p.x) : nullptr, 0x1p2f, 0x1p-3f, 0x1p13f};
    const Halves hw{static_cast<const uint16_t*>(w), ldw, vocab,
                    dh != nullptr ? reinterpret_cast<_Float16*>(ws + p.w) : nullptr, 0x1p6f, 0x1p-7f, 0x1p9f};
    const unsigned grid = blocks_of((rows > vocab ? rows : vocab) * 16);  // four waves of four rows
    uint32_t* most = reinterpret_cast<uint32_t*>(ws + p.most);
    halves_kernel<<<grid, 256, 0, st>>>(hx, hw, (int)hidden, p.ldx, t, most);
    if ((rc = check_launch("halves_kernel")) != MOC_OK) return rc;
    halves_again_kernel<<<grid < 512 ? grid : 512, 256, 0, st>>>(hx, hw, (int)hidden, p.ldx, temperature, t, most,
                                                                 (int)grid);
    if ((rc = check_launch("halves_again_kernel")) != MOC_OK) return rc;
  }
  if (p.fused && words > 0 && rows > 0) {
    words_left_kernel<<<static_cast<unsigned>((rows + 63) / 64), 1024,
                        words <= kWordsLds ? 64 * (words | 1) * 4 : 0, st>>>(t.ids, rows, (int)words, (int)p.slabs,
                                                                             t.first);
    if ((rc = check_launch("words_left_kernel")) != MOC_OK) return rc;
  }
  // f32: the rows that count in every product; bf16: in dweight's alone, as nothing is
  // read of the others' logits
  const bool copied = grads && f32;
  const char* x = copied ? ws + p.x : static_cast<const char*>(h);
  const int64_t ldx = copied ? p.ldx : ldh;
  for (int64_t i = 0; i < p.count; ++i) {
    const int64_t r0 = i * p.rows, n = rows - r0 < p.rows ? rows - r0 : p.rows;
    const char* xi = x + r0 * ldx * es;
    Targets ti = t;
    ti.weight += r0;
    ti.ids += r0 * n_words;
    if (words > 0) {
      ti.entropy += r0;
      ti.share += r0 * words;
      ti.first += r0;
    }
    if (p.fused) {
      float2* stat = reinterpret_cast<float2*>(ws + p.stat);
      float* z = reinterpret_cast<float*>(ws + p.at_words);
      const bool few = !grads && n <= kFewRows && hidden % 8 == 0 && hidden <= kFewHidden;
      rc = few ? launch_few(xi, n, hidden, ldx, w, vocab, ldw, kLog2E / temperature, ti, rows, words, z, stat, p.slabs, st)
               : launch_loss_gemm(xi, n, hidden, ldx, w, vocab, ldw, kLog2E / temperature, ti.ids,
                            words > 0 ? ti.first : nullptr, rows, n_words, z, stat, grads ? ws + p.d : nullptr, p.ldz, st);
      MOC_REQUIRE(rc <= 0, "moc_linear_loss: operands of up to 2 GiB");
      if (rc != MOC_OK) return rc;
      if (grads)
        slabs_grad_kernel<<<static_cast<unsigned>(n), 256, 0, st>>>(
            reinterpret_cast<uint16_t*>(ws + p.d), p.ldz, (int)vocab, stat, (int)p.slabs, ti, (int)words, temperature, z,
            row_loss + r0);
      else
        slabs_loss_kernel<<<static_cast<unsigned>(n), 256, 0, st>>>(stat, (int)p.slabs, ti, (int)words, temperature, z,
                                                                    row_loss + r0);
      rc = check_launch("slabs_grad_kernel");
    } else {
      rc = moc_gemm_ws(dtype, n, vocab, hidden, xi, ldx, 1, w, 1, ldw, 0, nullptr, 0, 0, nullptr, 0, 0, ws + p.z, p.ldz,
                       MOC_F32, gemm_ws, gemm_ws_bytes, stream);
      if (rc != MOC_OK) return rc;
      rc = logits_rows(true, ws + p.z, n, vocab, p.ldz, ti, words, temperature, row_loss + r0,
                       grads ? ws + p.d : nullptr, p.ldz, st);
    }
    if (rc != MOC_OK) return rc;
    if (dh != nullptr) {
      char* to = static_cast<char*>(dh) + r0 * hidden * (dh_dtype == MOC_F32 ? 4 : 2);
      const char* b = p.fused ? ws + p.w : static_cast<const char*>(w);
      rc = vocab == 1 ? outer(f32, n, hidden, ws + p.d, p.ldz, b, t.alpha, to, dh_dtype, st)
           : p.fused  ? gemm_half(n, hidden, vocab, ws + p.d, p.ldz, 1, b, p.ldx, to, hidden, dh_dtype, t.alpha, gemm_ws,
                                  gemm_ws_bytes, stream)
                      : moc_gemm_ws(dtype, n, hidden, vocab, ws + p.d, p.ldz, 1, b, ldw, 1, 0, nullptr, 0, 0, nullptr, 0,
                                    0, to, hidden, dh_dtype, gemm_ws, gemm_ws_bytes, stream);
      if (rc != MOC_OK) return rc;
    }
    if (dw != nullptr) {
      const bool one = p.count == 1;
      char* to = one ? static_cast<char*>(dw) : ws + (i == 0 ? p.acc : p.part);
      const int to_dtype = one ? dw_dtype : MOC_F32;
      const char* b = ws + p.x + r0 * p.ldx * es;
      rc = n == 1    ? outer(f32, vocab, hidden, ws + p.d, 1, b, t.alpha + 1, to, to_dtype, st)
           : p.fused ? gemm_half(vocab, hidden, n, ws + p.d, 1, p.ldz, b, p.ldx, to, hidden, to_dtype, t.alpha + 1,
                                 gemm_ws, gemm_ws_bytes, stream)
                     : moc_gemm_ws(dtype, vocab, hidden, n, ws + p.d, 1, p.ldz, b, p.ldx, 1, 0, nullptr, 0, 0, nullptr, 0,
                                   0, to, hidden, to_dtype, gemm_ws, gemm_ws_bytes, stream);
      if (rc != MOC_OK) return rc;
      if (i > 0) {
        float* acc = reinterpret_cast<float*>(ws + p.acc);
        const float* part = reinterpret_cast<const float*>(ws + p.part);
        const int64_t size = vocab * hidden;
        void* out = i + 1 == p.count ? dw : nullptr;
        if (dw_dtype == MOC_F32)
          add_f32_kernel<float><<<blocks_of(size), 256, 0, st>>>(acc, part, size, static_cast<float*>(out));
        else
          add_f32_kernel<uint16_t><<<blocks_of(size), 256, 0, st>>>(acc, part, size, static_cast<uint16_t*>(out));
        if ((rc = check_launch("add_f32_kernel")) != MOC_OK) return rc;
      }
    }
  }
  if (rows == 0 && dw != nullptr) {
    rc = moc_fill_zero(dw, vocab * hidden * (dw_dtype == MOC_F32 ? 4 : 2), stream);
    if (rc != MOC_OK) return rc;
  }
  if (loss == nullptr) return MOC_OK;
  loss_sum_kernel<<<1, 1024, 0, st>>>(row_loss, rows, t.total, loss);
  return check_launch("loss_sum_kernel");
}

extern "C" int moc_scale_inplace(int dtype0, void* p0, int64_t n0, int dtype1, void* p1, int64_t n1,
                                 const float* factor, void* stream) {
  MOC_REQUIRE((dtype0 == MOC_BF16 || dtype0 == MOC_F32) && (dtype1 == MOC_BF16 || dtype1 == MOC_F32),
              "moc_scale_inplace: bf16 or f32");
  MOC_REQUIRE(n0 >= 0 && n1 >= 0 && (n0 == 0 || p0 != nullptr) && (n1 == 0 || p1 != nullptr) && factor != nullptr,
              "moc_scale_inplace: null operand");
  if (n0 + n1 == 0) return MOC_OK;
  scale_kernel<<<blocks_of((n0 > n1 ? n0 : n1) / 8), 256, 0, as_stream(stream)>>>(dtype0 == MOC_F32, p0, n0,
                                                                                dtype1 == MOC_F32, p1, n1, factor);
  return check_launch("scale_kernel");
}
