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
// Logits are in units of log2(e) / T where they meet an exponential, which then is
// one v_exp_f32.  Sums over rows are in 64 bits and in a fixed
// order.
//
// A linear loss in bf16, by pieces of the rows (pieces_of), a row with all its words in
// one piece: with pieces of the words the gradient would need the logits a second time.
//   1. a teacher's words sorted, shares of one word added up (teacher_wave_kernel)
//   2. hidden rows and weight in f16 (halves_kernel), where there are gradients
//   3. the logits' product, of which the maximum and the sum of exponentials of every
//      64 words are kept, the exponentials as f16 and the targets' logits
//      (launch_loss_gemm; up to 16 rows few_rows_kernel)
//   4. each row's loss, and the exponentials into gradients of the logits, in place
//      (slabs_grad_kernel; slabs_loss_kernel without)
//   5. the products for dhidden and dweight (gemm_half)
// 16384 x 2048 x 32000: 5.7 ms, the three products 1.85, 1.64 and 1.68 (1160 to 1310
// TFLOP/s; 6.44e12 FLOP take 4.75 at a large library product's rate), (4) 0.43 at 4.9
// TB/s, (2) 0.07.
#include <algorithm>

#include "abi.h"
#include "common.h"

namespace moc {
namespace {

constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kMaxWords = 1024;
constexpr int32_t kNoWord = 0x7FFFFFFF;  // behind the words of a row
constexpr int32_t kUnknown = -2;         // a label outside the vocabulary

// What the losses read of the targets.  The pointers of a row's data are those of
// all rows; kernels of a piece of the rows add its first.
struct Targets {
  // labels (null: a teacher)
  const int64_t* labels;
  int64_t ignore;
  const float* row_weight;  // null: 1
  // a teacher
  float* weight;    // [rows], 0: the row counts for nothing
  float* entropy;   // [rows] sum of q ln q
  int32_t* ids;     // [rows][words] ascending, kNoWord behind the last
  float* share;     // [rows][words]; a word's second entry: -1
  uint16_t* first;  // [slabs + 1][rows] words left of each slab
  // over all rows
  double* total;    // sum of the weights (1 for a sum of losses)
  float* factor;    // upstream gradient / total
  float* largest;   // a power of two, no finite weight above it; 0: no row counts
  float* alpha;     // [2] what the f16 products for dhidden and dweight are times
};

__device__ __forceinline__ float weight_of(const Targets& t, int64_t r) {
  if (t.labels == nullptr) return t.weight[r];
  return t.labels[r] == t.ignore ? 0.f : t.row_weight != nullptr ? t.row_weight[r] : 1.f;
}

// Word k of row r, kUnknown for a label outside the vocabulary; its share, -1 for
// what is no word of its own.
__device__ __forceinline__ int32_t word_of(const Targets& t, int64_t r, int words, int k, int vocab, float& share) {
  if (t.labels != nullptr) {
    const int64_t label = t.labels[r];
    share = 1.f;
    return label >= 0 && label < vocab ? static_cast<int32_t>(label) : kUnknown;
  }
  const int32_t id = t.ids[r * words + k];
  share = id == kNoWord ? -1.f : t.share[r * words + k];
  return id;
}

int64_t slabs_of(int64_t vocab) { return (vocab + kLossSlab - 1) / kLossSlab; }

int64_t align256(int64_t n) { return (n + 255) & ~255LL; }

// A workspace's parts, taken one after another.
struct Taken {
  char* base;
  int64_t at = 0;
  template <typename T>
  T* take(int64_t n) {
    const int64_t here = at;
    at += align256(n * static_cast<int64_t>(sizeof(T)));
    return reinterpret_cast<T*>(base + here);
  }
};

// table: with the words left of each slab (linear losses).
void take_targets(Taken& ws, int64_t rows, int64_t words, int64_t slabs, bool table, Targets& t) {
  t.total = ws.take<double>(32);
  t.factor = reinterpret_cast<float*>(t.total + 1);
  t.largest = t.factor + 1;
  t.alpha = t.factor + 2;
  if (words > 0) {
    t.weight = ws.take<float>(rows);
    t.entropy = ws.take<float>(rows);
    t.ids = ws.take<int32_t>(rows * words);
    t.share = ws.take<float>(rows * words);
    if (table) t.first = ws.take<uint16_t>(rows * (slabs + 1));
  }
}

// Arrival counters of a launch, in the zeroed bytes at the start of a GEMM workspace
// (the products' own count from the front, as many as the CUs) and left zero.
constexpr int kTeacherCounter = 1022, kLossCounter = 1023;
static_assert(kLossCounter * 4 < MOC_GEMM_WS_COUNTER_BYTES, "counters");
// Rows whose losses the last workgroup of their own launch sums up: more have a
// launch for it, since arrivals at one word take some 4 ns each.
constexpr int64_t kArriveRows = 2048;

// Values that another workgroup of the same launch reads: through to memory, past the
// L2 of this XCD.
__device__ __forceinline__ void put_far(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get_far(const float* p) {
  return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Counts the workgroup; called by its thread 0, behind its put_far, which has reached
// memory when the count does.  True for the launch's last, for which get_far has what
// all of them put.  Nothing waits for another workgroup.
__device__ __forceinline__ bool arrive(int* counter, int blocks) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const bool last =
      __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == blocks - 1;
  if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return last;
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
// The least power of two, a normal number, that x >= 0 is not above.
__device__ __forceinline__ float power_above(float x) {
  const uint32_t up = (__float_as_uint(x) + 0x7FFFFFu) >> 23;
  return __uint_as_float((up < 1 ? 1u : up > 254 ? 254u : up) << 23);
}

// Sum and largest of the weights by one workgroup: total (a sum of losses: 1),
// factor = grad / total, largest.  FAR: of weights from the same launch.
template <bool FAR>
__device__ __forceinline__ void put_total(const Targets& t, int64_t rows, int mean, const float* grad, double* red64,
                                          float* red) {
  double s = 0;
  float m = 0.f;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) {
    const float w = FAR ? get_far(t.weight + r) : weight_of(t, r);
    s += w;
    // an infinite weight makes its own row's gradient infinite, not the others' 0
    m = fmaxf(m, fabsf(w) < INFINITY ? fabsf(w) : 0x1p-126f);
  }
  s = block_sum64(s, red64);
  m = block_reduce<true>(m, red);
  if (threadIdx.x != 0) return;
  if (!mean) s = 1.0;
  *t.total = s;
  *t.factor = static_cast<float>((grad != nullptr ? static_cast<double>(*grad) : 1.0) / s);
  *t.largest = m > 0.f ? power_above(m) : 0.f;
}

// A teacher's rows of up to 64 W words, a wave a row, W words a lane: sorted by rank
// (ties by place), entries of one word made one.  Bound by words^2 comparisons: four
// rows a workgroup spread them over the CUs (807 rows of 256 words 12 us, 47 with 16
// rows a workgroup; 8192 of 64 8.3).  counter (null: not here): the last workgroup sums
// the weights.
template <typename ID, bool TOP_F32, int W>
__global__ __launch_bounds__(256) void teacher_wave_kernel(const ID* __restrict__ ids, int64_t ids_ld,
                                                            const void* __restrict__ top, int64_t top_ld, int64_t rows,
                                                            int words, int vocab, float heat,
                                                            const float* __restrict__ row_weight, int mean,
                                                            const float* __restrict__ grad, Targets t, int* counter) {
  constexpr int kWide = 64 * W;
  __shared__ __attribute__((aligned(16))) uint32_t keys[4][kWide];
  __shared__ int32_t sorted_id[4][kWide];
  __shared__ float sorted_q[4][kWide];
  __shared__ double red64[4];
  __shared__ float red[4];
  __shared__ int flag;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (r < rows) {
    int32_t id[W];
    uint32_t key[W];  // the word, then its place: no two alike
    float q[W], mx = -INFINITY;
    const float unit = kLog2E / heat;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int k = lane + 64 * i;
      id[i] = kNoWord;
      q[i] = -INFINITY;
      if (k < words) {
        const int64_t word = static_cast<int64_t>(ids[r * ids_ld + k]);
        const float x = (TOP_F32 ? static_cast<const float*>(top)[r * top_ld + k]
                                 : bf16_to_f32(static_cast<const uint16_t*>(top)[r * top_ld + k]));
        if (word >= 0 && word < vocab && x != -INFINITY) {
          id[i] = static_cast<int32_t>(word);
          q[i] = x;
        }
      }
      mx = fmaxf(mx, q[i]);
      key[i] = (id[i] == kNoWord ? 1u << 31 : static_cast<uint32_t>(id[i]) << 10) + k;
      keys[wave][k] = key[i];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    float sum = 0.f;
    bool some = false;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      some |= id[i] != kNoWord;
      q[i] = id[i] == kNoWord ? 0.f : exp2f((q[i] - mx) * unit);
      sum += q[i];
    }
    some = __any(some);
    sum = wave_sum(sum);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's own row of LDS
    __builtin_amdgcn_wave_barrier();
    int rank[W] = {};
    for (int j = 0; j < kWide; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(&keys[wave][j]);
      const uint32_t other[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < W; ++i) rank[i] += other[e] < key[i];
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      sorted_id[wave][rank[i]] = id[i];
      sorted_q[wave][rank[i]] = q[i] / sum;
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_wave_barrier();
    float h = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int k = lane + 64 * i;
      const int32_t mine = sorted_id[wave][k];
      float share = -1.f;
      if (mine != kNoWord && (k == 0 || sorted_id[wave][k - 1] != mine)) {
        share = sorted_q[wave][k];
        for (int j = k + 1; j < words && sorted_id[wave][j] == mine; ++j) share += sorted_q[wave][j];
        h += share > 0.f || share != share ? share * logf(share) : 0.f;
      }
      if (k < words) {
        t.ids[r * words + k] = mine;
        t.share[r * words + k] = share;
      }
    }
    h = wave_sum(h);
    if (lane == 0) {
      put_far(t.weight + r, !some ? 0.f : row_weight != nullptr ? row_weight[r] : 1.f);
      t.entropy[r] = some ? h : 0.f;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // there before the workgroup is counted
    }
  }
  if (counter == nullptr) return;
  __syncthreads();  // every wave's row; thread 0's count covers them (put_far by each wave's lane 0)
  if (threadIdx.x == 0) flag = arrive(counter, gridDim.x);
  __syncthreads();
  if (flag) put_total<true>(t, rows, mean, grad, red64, red);
}

// The same for more words, one workgroup a row (256 words, us, 807 / 4096 rows: 16 /
// 44, by waves 12 / 26).
template <typename ID, bool TOP_F32>
__global__ __launch_bounds__(256) void teacher_targets_kernel(const ID* __restrict__ ids, int64_t ids_ld,
                                                              const void* __restrict__ top, int64_t top_ld, int words,
                                                              int vocab, float heat,
                                                              const float* __restrict__ row_weight, Targets t,
                                                              int64_t r0) {
  __shared__ int32_t id[kMaxWords], sorted_id[kMaxWords];
  __shared__ float q[kMaxWords], sorted_q[kMaxWords];
  __shared__ float red[4];
  const int64_t r = r0 + blockIdx.x;
  const int tid = threadIdx.x;
  const float unit = kLog2E / heat;
  float mx = -INFINITY, any = 0.f;
  bool bad = false;
  for (int k = tid; k < words; k += 256) {
    const int64_t word = static_cast<int64_t>(ids[r * ids_ld + k]);
    const float x = (TOP_F32 ? static_cast<const float*>(top)[r * top_ld + k]
                             : bf16_to_f32(static_cast<const uint16_t*>(top)[r * top_ld + k]));
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
    const float e = id[k] == kNoWord ? 0.f : exp2f((q[k] - mx) * unit);
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

// How many of a row's words lie left of each slab: 16 rows a workgroup, 16 threads a
// row that walk a sixteenth of the slabs each along its words (64 rows and 4 threads
// each: 35 us of 777 rows and 500 slabs), a line's quarter written at a time; the words
// in LDS up to kWordsLds of them (a chain of loads from memory otherwise).
constexpr int kWordsLds = 256;

__device__ __forceinline__ void words_left(const int32_t* __restrict__ ids, int64_t rows, int words, int slabs,
                                           uint16_t* __restrict__ first, int block, int32_t* held) {
  const int64_t r0 = static_cast<int64_t>(block) * 16, r = r0 + (threadIdx.x & 15);
  const int32_t* mine = ids + r * words;
  if (words <= kWordsLds) {
    const int n = static_cast<int>(rows - r0 < 16 ? rows - r0 : 16) * words;
    for (int i = threadIdx.x; i < n; i += 256) held[i / words * (words | 1) + i % words] = ids[r0 * words + i];
    __syncthreads();
    mine = held + (threadIdx.x & 15) * (words | 1);
  }
  if (r >= rows) return;
  const int per = (slabs + 16) / 16, n0 = threadIdx.x / 16 * per;
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

__global__ __launch_bounds__(256) void words_left_kernel(Targets t, int64_t rows, int words, int slabs) {
  __shared__ int32_t held[16 * (kWordsLds + 1)];
  words_left(t.ids, rows, words, slabs, t.first, blockIdx.x, held);
}

// The sums over the weights where no other launch makes them.
__global__ __launch_bounds__(1024) void target_total_kernel(int64_t rows, int mean, const float* __restrict__ grad,
                                                            Targets t) {
  __shared__ double red64[16];
  __shared__ float red[16];
  put_total<false>(t, rows, mean, grad, red64, red);
}

// What a kernel of the rows' losses leaves: each row's, and from the last workgroup
// of the launch to count itself the loss of all (loss null: not here).
struct LossOut {
  float* row_loss;  // [rows of all]
  float* loss;
  int64_t rows;    // of all
  int mean, known;  // known: total holds the divisor
  int* counter;
};

// loss = sum of the rows' weighted losses / sum of their weights (mean) or 1, by one
// workgroup.  FAR: of rows from the same launch.
template <bool FAR>
__device__ __forceinline__ void put_loss(const Targets& t, const LossOut& o, double* red64) {
  double s = 0, w = 0;
  const bool weights = o.mean && !o.known;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < o.rows; r += blockDim.x) {
    s += FAR ? get_far(o.row_loss + r) : o.row_loss[r];
    if (weights) w += weight_of(t, r);
  }
  s = block_sum64(s, red64);
  if (weights) w = block_sum64(w, red64);
  if (threadIdx.x == 0) *o.loss = static_cast<float>(!o.mean ? s : s / (o.known ? *t.total : w));
}

__global__ __launch_bounds__(1024) void loss_sum_kernel(Targets t, LossOut o) {
  __shared__ double red64[16];
  put_loss<false>(t, o, red64);
}

// A row's loss, by thread 0 of its workgroup; true where put_loss is this one's.
__device__ __forceinline__ bool put_row(const LossOut& o, int64_t r, float loss, int blocks) {
  put_far(o.row_loss + r, loss);
  return o.loss != nullptr && arrive(o.counter, blocks);
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
// A chunk's elements as T, to any element's address.
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
template <typename T, int NC, int TH, int LC>
__device__ __forceinline__ void logits_row(const T* x, int64_t ld, int vocab, const Targets& t, int64_t r0, int words,
                                           float heat, const LossOut& o, int& flag, T* dx, int64_t ldd) {
  constexpr int kPer = Elem<T>::kPer, kAhead = 4;
  __shared__ float red[TH / 64], at_word[kMaxWords];
  const int64_t r = r0 + blockIdx.x;
  const int tid = threadIdx.x;
  const float w = weight_of(t, r);
  const T* row = x + blockIdx.x * ld;
  T* out = dx + blockIdx.x * ldd;
  // whole chunks, from the first 16-byte boundary on, and the `loose` elements before and
  // behind them, a thread each
  const int head = min(vocab, static_cast<int>(-(reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (kPer - 1)));
  const int full = (vocab - head) / kPer, loose = vocab - full * kPer;
  const int lone = tid < head ? tid : full * kPer + tid;  // this thread's, tid < loose
  const T* chunks = row + head;
  T* out_chunks = out + head;
  if (w == 0.f) {                                      // uniform
    if (dx != nullptr) {
      const float zero[kPer] = {};
      for (int c = tid; c < full; c += TH) store_grad(out_chunks + c * kPer, zero);
      if (tid < loose) out[lone] = Elem<T>::of(0.f);
    }
    if (tid == 0) flag = put_row(o, r, 0.f, gridDim.x);
    return;
  }
  const float unit = kLog2E / heat;
  const float last = tid < loose ? Elem<T>::one(row[lone]) : -INFINITY;
  uint4 v[NC > 0 ? NC : 1];
  __shared__ uint4 more[LC > 0 ? LC * TH : 1];  // chunks NC .. NC + LC of each thread, read by it alone
  float mx = last, sum = 0.f;
  if constexpr (NC > 0) {
    if (full > 0) {
      // behind the end a thread reads the last chunk again, which leaves the maximum
      // and is not summed
#pragma unroll
      for (int i = 0; i < LC; ++i) v[i] = load_chunk(chunks + min(tid + TH * (NC + i), full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < LC; ++i) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) mx = fmaxf(mx, Elem<T>::get(v[i], e));
        more[i * TH + tid] = v[i];
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = load_chunk(chunks + min(tid + TH * i, full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) mx = fmaxf(mx, Elem<T>::get(v[i], e));
    }
    mx = block_reduce<true>(mx, red);
#pragma unroll
    for (int i = 0; i < LC; ++i)
      if (tid + TH * (NC + i) < full) {
        const uint4 a = more[i * TH + tid];
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += __builtin_amdgcn_exp2f((Elem<T>::get(a, e) - mx) * unit);
      }
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (tid + TH * i < full)
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += __builtin_amdgcn_exp2f((Elem<T>::get(v[i], e) - mx) * unit);
    if (tid < loose) sum += __builtin_amdgcn_exp2f((last - mx) * unit);
    sum = block_reduce<false>(sum, red);
  } else {
    mx = last;
    sum = tid < loose ? (last == last && mx != INFINITY ? 1.f : NAN) : 0.f;
    if (tid < loose && mx == -INFINITY) sum = 0.f;
    for (int c0 = tid; c0 < full; c0 += TH * kAhead) {
      uint4 a[kAhead];
      float m = mx;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) a[i] = load_chunk(chunks + min(c0 + TH * i, full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int e = 0; e < kPer; ++e) m = fmaxf(m, Elem<T>::get(a[i], e));
      const float ref = m == -INFINITY ? 0.f : m;
      sum *= mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mx - ref) * unit);  // nothing summed yet, or NaN
      mx = m;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (c0 + TH * i < full)
#pragma unroll
          for (int e = 0; e < kPer; ++e) sum += __builtin_amdgcn_exp2f((Elem<T>::get(a[i], e) - ref) * unit);
    }
    const float all = block_reduce<true>(mx, red);
    sum *= mx == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mx - all) * unit);
    sum = block_reduce<false>(sum, red);
    mx = all;
  }
  // log2 p = (z - mx) unit - lsum: the difference first, as z unit of a mask of the
  // type's lowest value is beyond f32
  const float lsum = log2f(sum);
  const int n = words > 0 ? words : 1;
  float cross = 0.f;
  for (int k = tid; k < n; k += TH) {
    float share;
    const int32_t id = word_of(t, r, words, k, vocab, share);
    if (id == kUnknown) cross = NAN;
    if (id == kUnknown || share == -1.f) continue;
    const float z = Elem<T>::one(row[id]) - mx;
    at_word[k] = fmaf(z, unit, -lsum);
    if (share != 0.f) cross += share * (heat * (lsum * kLn2) - z);  // -T ln p
  }
  cross = block_reduce<false>(cross, red);
  // counted before the gradient is written, which its wait then overlaps
  if (tid == 0)
    flag = put_row(o, r, w * (heat * (cross + (words > 0 ? heat * t.entropy[r] : 0.f))), gridDim.x);
  if (dx == nullptr) return;
  const float c = cross == cross ? heat * w * *t.factor : NAN;
  auto grad = [&](const uint4& a, int at) {
    float o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = c * __builtin_amdgcn_exp2f(fmaf(Elem<T>::get(a, e) - mx, unit, -lsum));
    store_grad(out_chunks + at * kPer, o);
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
      for (int i = 0; i < kAhead; ++i) a[i] = load_chunk(chunks + min(c0 + TH * i, full - 1) * kPer);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (c0 + TH * i < full) grad(a[i], c0 + TH * i);
    }
  }
  if (tid < loose) out[lone] = Elem<T>::of(c * __builtin_amdgcn_exp2f(fmaf(last - mx, unit, -lsum)));
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // stored before the words' own
  __syncthreads();
  for (int k = tid; k < n; k += TH) {
    float share;
    const int32_t id = word_of(t, r, words, k, vocab, share);
    if (id == kUnknown || share == -1.f) continue;
    out[id] = Elem<T>::of(c * (__builtin_amdgcn_exp2f(at_word[k]) - share));
  }
}

template <typename T, int NC, int TH, int LC = 0>
__global__ __launch_bounds__(TH) void logits_loss_kernel(const T* x, int64_t ld, int vocab, Targets t, int64_t r0,
                                                         int words, float heat, LossOut o, T* dx, int64_t ldd) {
  __shared__ double red64[TH / 64];
  __shared__ int flag;
  logits_row<T, NC, TH, LC>(x, ld, vocab, t, r0, words, heat, o, flag, dx, ldd);
  __syncthreads();
  if (flag) put_loss<true>(t, o, red64);
}

// ------------------------------------------------- logits that were not stored
// Up to 16 rows: the weight is read once, straight into the operand
// registers of v_mfma_f32_16x16x32_bf16 (a wave 16 words, a workgroup a slab of 64),
// 16 loads ahead; the rows stand in LDS in fragment order.  Bound by the weight's
// bytes: 32000 x 2048, 1 row 25.2 us, 5.2 TB/s, 16 rows 26.1; 128256 x 1024, 16 rows
// 45.1, 5.8 TB/s; 128256 x 4096, 4 rows 202, 5.2 TB/s.  Sums in four chains have half the
// error of the tiled product's one (2048 x 32000: losses off by 5e-7 on average, 9e-7).
constexpr int kFewRows = 16, kFewAhead = 16, kFewHidden = 4096, kFewSums = 4;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// The column of the chunk of 8 that a quarter of the lanes loads in the last step: the
// row's first where its own lies behind the hidden size, since a row may hold no more
// than the hidden size up to a multiple of 8.
constexpr int few_last_column(int hidden, int quad) {
  const int k = (hidden - 1) / 32 * 32 + 8 * quad;
  return k < hidden ? k : 0;
}

constexpr bool few_columns_in_rows() {
  for (int hidden = 1; hidden <= kFewHidden; ++hidden)
    for (int quad = 0; quad < 4; ++quad)
      if (few_last_column(hidden, quad) + 8 > (hidden + 7) / 8 * 8) return false;
  return true;
}
static_assert(few_columns_in_rows(), "a load behind its row");

// RAGGED: a hidden size that is no multiple of 32 (its masks cost 1.5 us of 28).  KEEP:
// with exponentials as launch_loss_gemm keeps them.
template <bool RAGGED, bool KEEP>
__global__ __launch_bounds__(256) void few_rows_kernel(const uint16_t* __restrict__ h, int64_t ldh, int rows,
                                                       const uint16_t* __restrict__ w, int64_t ldw, int vocab,
                                                       int hidden, float unit, const int32_t* __restrict__ ids,
                                                       int64_t ld_ids, const uint16_t* __restrict__ first,
                                                       int64_t ld_first, int words,
                                                       float* __restrict__ z, float2* __restrict__ stat, int slabs,
                                                       _Float16* __restrict__ kept, int64_t ld_kept) {
  extern __shared__ uint4 frag[];  // [steps][64], then the waves' maxima and sums
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int steps = (hidden + 31) / 32;
  float2* part = reinterpret_cast<float2*>(frag + steps * 64);  // [2][4][16]
  const int row = lane & 15, quad = lane >> 4;
  const int last = few_last_column(hidden, quad) - 8 * quad;
  // what a chunk of 8 at column k holds of the hidden size (behind it is another tensor's
  // or padding)
  auto held = [&](uint4 v, int k) {
    const int n = hidden - k;
    auto word = [&](uint32_t x, int at) { return at + 1 < n ? x : at < n ? x & 0xFFFFu : 0u; };
    return make_uint4(word(v.x, 0), word(v.y, 2), word(v.z, 4), word(v.w, 6));
  };
  const uint4 end = held(make_uint4(~0u, ~0u, ~0u, ~0u), 32 * (steps - 1) + 8 * quad);
  auto load = [&](uint4 (&a)[kFewAhead], const uint16_t* src, int s0) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int s = min(s0 + i, steps - 1);
      a[i] = *reinterpret_cast<const uint4*>(src + (RAGGED && s == steps - 1 ? last : 32 * s));
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
    frag[i] = n < rows && (!RAGGED || k < hidden) ? *reinterpret_cast<const uint4*>(h + n * ldh + k)
                                                  : make_uint4(0, 0, 0, 0);
    if constexpr (RAGGED) frag[i] = held(frag[i], k);
  }
  __syncthreads();
  for (int turn = 0; slab < slabs; slab += gridDim.x, turn ^= 1) {
    const uint16_t* src = word_of(slab);
    f32x4_t sums[kFewSums] = {};  // chains of a quarter of the steps: fewer roundings in a row
    auto products = [&](uint4 (&v)[kFewAhead], int s0) {
#pragma unroll
      for (int i = 0; i < kFewAhead; ++i) {
        if (s0 + i >= steps) break;
        uint4 x = v[i];
        if (RAGGED && s0 + i == steps - 1) x = make_uint4(x.x & end.x, x.y & end.y, x.z & end.z, x.w & end.w);
        f32x4_t& to = sums[i % kFewSums];
        to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x),
                                                     __builtin_bit_cast(bf16x8_t, frag[(s0 + i) * 64 + lane]), to, 0, 0,
                                                     0);
      }
    };
    for (int s0 = 0; s0 < steps; s0 += 2 * kFewAhead) {
      if (s0 + kFewAhead < steps) load(b, src, s0 + kFewAhead);
      products(a, s0);
      if (s0 + 2 * kFewAhead < steps) load(a, src, s0 + 2 * kFewAhead);
      else if (slab + static_cast<int>(gridDim.x) < slabs) load(a, word_of(slab + gridDim.x), 0);
      products(b, s0 + kFewAhead);
    }
    f32x4_t acc = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    // lane: row, words slab * 64 + wave * 16 + 4 quad + e
    const int c0 = wave * 16 + 4 * quad;
    if (row < rows) {
      int k = first != nullptr ? first[slab * ld_first + row] : 0;
      for (; k < words; ++k) {
        const int c = ids[row * ld_ids + k] - slab * kLossSlab - c0;
        if (c >= 4) break;
        if (c >= 0 && c < 4) z[row * words + k] = c == 0 ? acc[0] : c == 1 ? acc[1] : c == 2 ? acc[2] : acc[3];
      }
    }
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[e] = slab * kLossSlab + c0 + e < vocab ? acc[e] : -INFINITY;
      m = fmaxf(m, acc[e]);
    }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = ceilf(fmaxf(m, __shfl_xor(m, 32)) * unit);  // as in launch_loss_gemm's statistics
    const float ref = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(fmaf(acc[e], unit, -ref));
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane < 16) part[(turn * 4 + wave) * 16 + row] = make_float2(m, s);
    __syncthreads();
    if (KEEP && row < rows) {
      typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
      float all = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) all = fmaxf(all, part[(turn * 4 + i) * 16 + row].x);
      const float from = all == -INFINITY ? 0.f : all - 15.f;
      f16x4_t e;
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = static_cast<_Float16>(__builtin_amdgcn_exp2f(fmaf(acc[i], unit, -from)));
      *reinterpret_cast<f16x4_t*>(kept + row * ld_kept + slab * kLossSlab + c0) = e;  // rows of whole slabs
    }
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

// A row's sum of exponentials from its slabs' references and sums: the largest
// reference, and log2 of the sum against it (one number would be rounded at the
// reference's size, and a small loss with it); 256 threads, a slab's loads in flight
// with its seven followers'.
struct Lse {
  float ref, log2_sum;
};

__device__ __forceinline__ Lse slabs_lse(const float2* __restrict__ stat, int slabs, float* red) {
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
  return {all, log2f(s)};
}

// A row's cross entropy sum q (-log2 p) over the words this thread takes, log2 p of
// each into at_word (may be null); NaN for an unknown label.  z: its words' logits.
__device__ __forceinline__ float cross_of(const Targets& t, int64_t r, int words, int vocab,
                                          const float* __restrict__ z, float unit, const Lse& lse, float* at_word) {
  float cross = 0.f;
  for (int k = threadIdx.x; k < (words > 0 ? words : 1); k += 256) {
    float share;
    const int32_t id = word_of(t, r, words, k, vocab, share);
    if (id == kUnknown) cross = NAN;
    if (id == kUnknown || share == -1.f) continue;
    const float l = fmaf(z[k], unit, -lse.ref) - lse.log2_sum;
    if (at_word != nullptr) at_word[k] = l;
    if (share != 0.f) cross -= share * l;
  }
  return cross;
}

// What a row's logits left (launch_loss_gemm): statistics of its slabs and its words'
// logits, rows of the piece; r0: the piece's first row.
struct Slabs {
  const float2* stat;
  const float* z;
  int count, vocab, words;
  int64_t r0;
  float heat;
};

// Losses alone: one workgroup a row, bound by latency (4099 rows of 782 slabs, 26 MB:
// 11 us).
__global__ __launch_bounds__(256) void slabs_loss_kernel(Slabs s, Targets t, LossOut o) {
  __shared__ float red[4];
  __shared__ double red64[4];
  __shared__ int flag;
  const int64_t r = s.r0 + blockIdx.x;
  const float w = weight_of(t, r);
  float loss = 0.f;
  if (w != 0.f) {  // uniform
    const Lse lse = slabs_lse(s.stat + static_cast<int64_t>(blockIdx.x) * s.count, s.count, red);
    const float* z = s.z + static_cast<int64_t>(blockIdx.x) * (s.words > 0 ? s.words : 1);
    const float cross = block_reduce<false>(cross_of(t, r, s.words, s.vocab, z, kLog2E / s.heat, lse, nullptr), red);
    loss = w * (s.heat * s.heat * (cross * kLn2 + (s.words > 0 ? t.entropy[r] : 0.f)));
  }
  if (threadIdx.x == 0) flag = put_row(o, r, loss, gridDim.x);
  __syncthreads();
  if (flag) put_loss<true>(t, o, red64);
}

// ------------------------------------------------------- operands in f16
// Hidden rows and weight for the products with f16 gradients: bf16 values times a
// power of two, which f16 holds as they are from 2^-17 up and rounds by at most 2^-25
// below; rows that do not count become 0.  The power is a guess that suits what
// networks hold (the largest of the hidden rows in [2^-3, 2^13], of the weight in
// [2^-7, 2^9]: what is rounded is off by 2^-24 of the largest at most); the largest
// value is found on the way, and slabs_grad_kernel redoes a tensor that it does not
// suit.  Bound by its bytes: 32000 x 2048 and 16384 rows 69 us, 5.8 TB/s;
// 128256 x 2048 and 4096 rows 203, 5.3.
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
__device__ __forceinline__ uint32_t halve_rows(const Halves& h, int hidden, int64_t ldo, const Targets* counts,
                                               float scale, int block, int blocks) {
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  constexpr int kRows = 4;
  const int lane = threadIdx.x & 63, chunks = static_cast<int>(ldo / 8);
  const int64_t waves = static_cast<int64_t>(blocks) * 4;
  uint32_t most = 0;
  for (int64_t r0 = static_cast<int64_t>(block) * 4 + (threadIdx.x >> 6); r0 < h.rows; r0 += waves * kRows) {
    for (int c = lane; c < chunks; c += 64) {
      const int k = 8 * c;
      uint4 v[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t r = r0 + waves * i;
        v[i] = k < hidden && r < h.rows && (counts == nullptr || weight_of(*counts, r) != 0.f)
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

// most [2][blocks]: the workgroups' largest values (one word for all of them would
// have as many atomics in a row).  Workgroup 0 sums the rows' weights meanwhile, and
// those behind it look up a teacher's words, so that neither is a launch of its own.
__global__ __launch_bounds__(256) void halves_kernel(Halves hidden_rows, Halves weight_rows, int hidden, int64_t ldo,
                                                     Targets t, int64_t rows, int mean,
                                                     const float* __restrict__ grad, int words, int slabs,
                                                     uint32_t* __restrict__ most, int blocks, int* counters) {
  __shared__ int32_t held[16 * (kWordsLds + 1)];
  __shared__ uint32_t red[4];
  __shared__ float redf[4];
  __shared__ double red64[4];
  const int extra = static_cast<int>(gridDim.x) - blocks, block = static_cast<int>(blockIdx.x) - extra;
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < MOC_GEMM_WS_COUNTER_BYTES / 4; i += 256) counters[i] = 0;  // of the products and losses
    put_total<false>(t, rows, mean, grad, red64, redf);
  } else if (block < 0) {
    words_left(t.ids, rows, words, slabs, t.first, blockIdx.x - 1, held);
  } else {
    uint32_t m = hidden_rows.to != nullptr ? halve_rows(hidden_rows, hidden, ldo, &t, hidden_rows.guess, block, blocks) : 0;
    m = block_max_bits(m, red);
    if (threadIdx.x == 0) most[block] = m;
    m = weight_rows.to != nullptr ? halve_rows(weight_rows, hidden, ldo, nullptr, weight_rows.guess, block, blocks) : 0;
    m = block_max_bits(m, red);
    if (threadIdx.x == 0) most[blocks + block] = m;
  }
}

// One workgroup a row: its loss, and its f16 exponentials into gradients of the
// logits, in place: e exp2(m - lse) of a slab's reference m is p.  The gradients stay
// in f16, as (w / largest) 2^14 (p - q): a bf16 rounding of them, 2^-8 of each, would
// add to the products' sums, where the words' parts cancel, more than the sums' own
// rounding (measured: up to 1.9 times the error of f32 ones); 2^-11 does not show.
// Down to 2^-28 of the largest they have all 11 bits, below 2^-39 they are 0, so rows
// whose weights lie further below the largest get gradients of fewer bits, or none.
// Bound by its bytes: 16384 x 32000 427 us, 4.9 TB/s; 8192 165, 6.3 with what the caches
// still hold.
//
// TWO (few rows): as two bf16 parts too, rows [0, rows) and [rows, 2 rows) of two, for
// a product with the weight as it is.
template <bool TWO>
__device__ __forceinline__ void slabs_grad_row(uint16_t* e, int64_t ld, const Slabs& s, const Targets& t,
                                               const LossOut& o, int& flag, int64_t at, int rows, int part, int parts,
                                               uint16_t* two) {
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  __shared__ float red[4], at_word[kMaxWords];
  const int64_t r = s.r0 + at;
  const int tid = threadIdx.x;
  const float w = weight_of(t, r);
  uint16_t* out = e + at * ld;
  uint4* row = reinterpret_cast<uint4*>(out);
  uint16_t* pair[2] = {two + at * ld, two + (rows + at) * ld};
  // this workgroup's part of the row
  const int all = (s.vocab + 7) / 8, each = (all + parts - 1) / parts, begin = part * each,
            chunks = all < begin + each ? all : begin + each;
  if (w == 0.f) {  // uniform
    for (int c = begin + tid; c < chunks; c += 256) {
      row[c] = make_uint4(0, 0, 0, 0);
      if constexpr (TWO)
        for (uint16_t* p : pair) reinterpret_cast<uint4*>(p)[c] = make_uint4(0, 0, 0, 0);
    }
    if (tid == 0) flag = part == 0 && put_row(o, r, 0.f, rows);
    return;
  }
  const float2* st = s.stat + at * s.count;
  constexpr int kAhead = 4;
  uint4 v[kAhead];
  float m[kAhead];
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int c = min(c0 + 256 * i, chunks - 1);
      v[i] = row[c];
      m[i] = st[c / (kLossSlab / 8)].x;
    }
  };
  load(begin + tid);  // on their way during the statistics
  const Lse lse = slabs_lse(st, s.count, red);
  const float* z = s.z + at * (s.words > 0 ? s.words : 1);
  const float cross = block_reduce<false>(cross_of(t, r, s.words, s.vocab, z, kLog2E / s.heat, lse, at_word), red);
  // counted before the gradient is written, which its wait then overlaps
  if (tid == 0)
    flag = part == 0 &&
           put_row(o, r, w * (s.heat * s.heat * (cross * kLn2 + (s.words > 0 ? t.entropy[r] : 0.f))), rows);
  const float c = cross == cross ? w / *t.largest * 0x1p14f : NAN;
  for (int c0 = begin + tid; c0 < chunks; c0 += 256 * kAhead) {
    if (c0 != begin + tid) load(c0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = c0 + 256 * i;
      if (at >= chunks) break;
      const float f = c * __builtin_amdgcn_exp2f(m[i] - lse.ref - lse.log2_sum - 15.f);
      const uint32_t in[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t out[4], high[4], low[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, in[q]);
        const cvt_f32x2_t g = {static_cast<float>(h.x) * f, static_cast<float>(h.y) * f};
        out[q] = __builtin_bit_cast(uint32_t, __builtin_convertvector(g, f16x2_t));
        if constexpr (TWO) {
          high[q] = __builtin_bit_cast(uint32_t, __builtin_convertvector(g, cvt_bf16x2_t));
          const cvt_f32x2_t rest = {g.x - __uint_as_float(high[q] << 16), g.y - __uint_as_float(high[q] & 0xFFFF0000u)};
          low[q] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, cvt_bf16x2_t));
        }
      }
      row[at] = make_uint4(out[0], out[1], out[2], out[3]);
      if constexpr (TWO) {
        reinterpret_cast<uint4*>(pair[0])[at] = make_uint4(high[0], high[1], high[2], high[3]);
        reinterpret_cast<uint4*>(pair[1])[at] = make_uint4(low[0], low[1], low[2], low[3]);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // stored before the words' own
  __syncthreads();
  for (int k = tid; k < (s.words > 0 ? s.words : 1); k += 256) {
    float share;
    const int32_t id = word_of(t, r, s.words, k, s.vocab, share);
    if (id == kUnknown || share == -1.f || id < 8 * begin || id >= 8 * chunks) continue;
    const float g = c * (__builtin_amdgcn_exp2f(at_word[k]) - share);
    out[id] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(g));
    if constexpr (TWO) {
      pair[0][id] = bf16_rne(g);
      pair[1][id] = bf16_rne(g - bf16_to_f32(pair[0][id]));
    }
  }
}

// The first piece has kAgainBlocks workgroups more, which look at the f16 operands:
// those that the guess did not suit are done again, and the products' factors written.
constexpr int kAgainBlocks = 64;

template <bool TWO>
__global__ __launch_bounds__(256) void slabs_grad_kernel(uint16_t* e, int64_t ld, Slabs s, Targets t, LossOut o,
                                                         Halves hidden_rows, Halves weight_rows, int hidden,
                                                         int64_t ldo, const uint32_t* __restrict__ most, int blocks,
                                                         int parts, uint16_t* two) {
  __shared__ double red64[4];
  __shared__ uint32_t red[4];
  __shared__ int flag;
  const int again = s.r0 == 0 ? kAgainBlocks : 0;
  if (static_cast<int>(blockIdx.x) < again) {
    uint32_t m[2] = {0, 0};
#pragma unroll 4
    for (int i = threadIdx.x; i < blocks; i += 256) {
      m[0] = max(m[0], most[i]);
      m[1] = max(m[1], most[blocks + i]);
    }
    const float sx = halves_scale(hidden_rows, block_max_bits(m[0], red));
    const float sw = halves_scale(weight_rows, block_max_bits(m[1], red));
    if (sx != hidden_rows.guess) halve_rows(hidden_rows, hidden, ldo, &t, sx, blockIdx.x, again);
    if (sw != weight_rows.guess) halve_rows(weight_rows, hidden, ldo, nullptr, sw, blockIdx.x, again);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      // no row counts: gradients of 0, whatever the divisor
      const float f = *t.largest > 0.f ? s.heat * *t.factor * *t.largest * 0x1p-14f : 0.f;
      t.alpha[0] = f / sw;
      t.alpha[1] = f / sx;
    }
    return;
  }
  const int i = static_cast<int>(blockIdx.x) - again, rows = (static_cast<int>(gridDim.x) - again) / parts;
  slabs_grad_row<TWO>(e, ld, s, t, o, flag, i / parts, rows, i % parts, parts, two);
  __syncthreads();
  if (flag) put_loss<true>(t, o, red64);
}

// Rows that count, zeros for the others: what is in those reaches no product (f32).
// Rows of 16-byte chunks, whose last one is cut off at the hidden size.
__global__ __launch_bounds__(256) void counted_rows_kernel(const float* __restrict__ h, int64_t ldh, int64_t rows,
                                                           int hidden, Targets t, float* __restrict__ out,
                                                           int64_t ldo) {
  const int chunks = (hidden + 3) / 4;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * chunks; i += step) {
    const int64_t r = i / chunks;
    const int k = static_cast<int>(i - r * chunks) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (weight_of(t, r) != 0.f) {
      v = *reinterpret_cast<const float4*>(h + r * ldh + k);
      if (k + 1 >= hidden) v.y = 0.f;
      if (k + 2 >= hidden) v.z = 0.f;
      if (k + 3 >= hidden) v.w = 0.f;
    }
    *reinterpret_cast<float4*>(out + r * ldo + k) = v;
  }
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

// The rows of a product with gradients in two parts, where no K split's sum adds them up
// (gemm_pair_rows): out = *alpha (a[r] + a[rows + r]).
template <typename OUT>
__global__ __launch_bounds__(256) void two_parts_kernel(const float* __restrict__ a, int64_t n,
                                                        const float* __restrict__ alpha, OUT* __restrict__ out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) out[i] = Elem<OUT>::of(*alpha * (a[i] + a[n + i]));
}

// out[i][j] = *alpha a_i b_j (alpha null: 1), the product over one row or one word (the
// engine takes no operand of one element's pitch).  Columns blockIdx.x, rows blockIdx.y
// and on.
template <typename T, typename OUT>
__global__ __launch_bounds__(256) void outer_kernel(const T* __restrict__ a, int64_t lda, const T* __restrict__ b,
                                                    int64_t m, int64_t n, const float* __restrict__ alpha,
                                                    OUT* __restrict__ out) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (j >= n) return;
  const float bj = Elem<T>::one(b[j]) * (alpha != nullptr ? *alpha : 1.f);
  for (int64_t i = blockIdx.y; i < m; i += gridDim.y) out[i * n + j] = Elem<OUT>::of(Elem<T>::one(a[i * lda]) * bj);
}

// The words behind the last whole four of f32 gradients of logits (the tiled f32
// products take extents in fours): the sum of d[r][j] w[j], j below rest, is added
// to dh[r] (add) or stored there.
__global__ __launch_bounds__(256) void rest_words_kernel(const float* __restrict__ d, int64_t ldd,
                                                         const float* __restrict__ w, int64_t ldw, int add, int rest,
                                                         int64_t rows, int hidden, float* __restrict__ dh) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * hidden; i += step) {
    const int64_t r = i / hidden;
    const int k = static_cast<int>(i - r * hidden);
    float s = add ? dh[i] : 0.f;
    for (int j = 0; j < rest; ++j) s = fmaf(d[r * ldd + j], w[j * ldw + k], s);
    dh[i] = s;
  }
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

// --------------------------------------------------------------------- host
// Logits, or what is kept of them, exist for a piece of the rows at a time: within a GiB,
// f16 gradients within what a product's operand may have, since each piece adds its part
// of dweight in f32 (16384 x 512 x 128256 8.8 ms by 1 GiB, 8.6 by 2; 8192 x 2048 x 128256
// 12.3, 11.6).
constexpr int64_t kPieceBytes = 1LL << 30, kGradPieceBytes = (1LL << 31) - 4096;
constexpr int64_t kWidest = 4;
constexpr int64_t kF32Weight = 48LL << 20;
// Bytes of an f32 product's K split: with more of them the parts' own traffic costs more
// than the split saves, and up to 16 times the result would be held.  us, split / whole:
//   dweight  4000 x 128 x 4000 rows     4 MB   56 /   94    10000 x 300 x 3000    144 MB   243 /  229
//           50048 x 768 x 2048       2460 MB 2596 / 1416   128256 x 256 x  500   1051 MB   870 /  354
//   dhidden  2048 x 768 x 50256 words  13 MB 1411 / 1838     3000 x 300 x 10000    54 MB   203 /  216
constexpr int64_t kF32Parts = 64LL << 20;
// Few rows: dhidden comes from gradients in two bf16 parts, twice the rows, with the
// weight as it is (TWO), else from f16 ones and a copy of the weight.  The copy moves 4
// bytes of each of the weight's values, the parts cost as many products and 16 bytes of
// each logit again.  GPU time of a step, us, copy / two parts:
//   32000 words, hidden  256:   64 rows  68 /  69   128  71 /  74   256  79 /  89
//   32000               1024:   64       99 /  96   128 111 / 111   256 134 / 136
//   32000               2048:   64      180 / 139   256 251 / 226   384 289 / 288
//   32000               4096:   64      354 / 280   256 425 / 405   384 497 / 503
//   100000              1024:   64      296 / 233   192 342 / 320   384 464 / 509
//   100000              2048:   64      542 / 410   256 657 / 593   512 890 / 923
bool in_two_parts(int64_t rows, int64_t hidden, int64_t vocab) {
  return rows * (hidden + 960) <= 420 * hidden && vocab > 1;
}

// Workgroups of slabs_grad_kernel a row, each a part of its gradient (and the
// statistics, again): few rows leave the CUs idle otherwise.  us, 1 / these: 4 x 32000
// words 10.3 / 7.1, 64 x 128256 23.9 / 15.3, 100 x 32000 12.4 / 10.5; 400 x 128256 and
// 512 x 32000 take as long in two parts as in one, 2000 x 32000 56 in four, 52 in one.
int grad_parts(int64_t rows) { return rows > 256 ? 1 : rows < 64 ? 8 : static_cast<int>(512 / rows); }

constexpr int kHalvesBlocks = 1024;  // workgroups of halves_kernel that write f16 rows

// A linear loss's pieces and the parts of its workspace.
struct Pieces {
  bool fused;           // bf16: logits inside the product (launch_loss_gemm), not stored
  int64_t rows, count;  // rows of a piece, pieces
  int64_t ldz, ldx;     // row pitches: a piece's logits, the copies of hidden rows and weight
  int64_t slabs;
  Targets t;
  float* row_loss;
  char *d, *x, *w;  // logits, then their gradients; copies of hidden rows and weight
  float *acc, *part, *z;
  char* two;    // few rows (in_two_parts): gradients in two parts,
  float* both;  // their product
  float* rest;  // f32: rows of dweight behind the whole fours; parts of dhidden
  uint32_t* most;
  float2* stat;
  int64_t bytes;
};

Pieces pieces_of(int dtype, int64_t rows, int64_t hidden, int64_t vocab, int64_t words, bool grads, void* base) {
  Pieces p{};
  const bool f32 = dtype == MOC_F32;
  const int64_t es = f32 ? 4 : 2;
  p.fused = !f32;
  p.ldz = (vocab + 63) & ~63LL;
  p.ldx = (hidden + 63) & ~63LL;
  p.slabs = slabs_of(vocab);
  const int64_t each = f32 ? p.ldz * 4 : grads ? p.ldz * 2 : p.slabs * 8;
  int64_t n = (p.fused && grads ? kGradPieceBytes : kPieceBytes) / each / 256 * 256;
  // its hidden rows within 32-bit offsets, at up to kWidest times their own pitch
  const int64_t most = ((1LL << 31) - 4096) / (es * kWidest * p.ldx) / 256 * 256;
  if (n > most) n = most;
  if (n < 256) n = 256;
  if (n > rows) n = rows < 1 ? 1 : rows;
  p.rows = n;
  p.count = rows < 1 ? 0 : (rows + n - 1) / n;
  Taken ws{static_cast<char*>(base)};
  take_targets(ws, rows, words, p.slabs, p.fused, p.t);
  p.row_loss = ws.take<float>(rows);
  if (p.fused) {
    p.stat = ws.take<float2>(n * p.slabs);
    p.z = ws.take<float>(n * (words > 0 ? words : 1));
  }
  if (f32 || grads) p.d = ws.take<char>(n * p.ldz * es);
  if (grads) p.x = ws.take<char>(rows * p.ldx * es);
  if (grads && f32) p.rest = ws.take<float>((n > 4 ? n : 4) * hidden);
  if (grads && p.fused) {
    if (in_two_parts(rows, hidden, vocab)) {
      p.two = ws.take<char>(2 * rows * p.ldz * 2);
      p.both = ws.take<float>(2 * rows * hidden);
    } else {
      p.w = ws.take<char>(vocab * p.ldx * 2);
    }
    p.most = ws.take<uint32_t>(2 * kHalvesBlocks);
  }
  if (grads && p.count > 1) {
    p.acc = ws.take<float>(vocab * hidden);
    p.part = ws.take<float>(vocab * hidden);
  }
  p.bytes = ws.at;
  return p;
}

// Rows of a launch with a workgroup a row: a grid has less than 2^32 threads, and one of
// 1024 a row for the widest rows.
constexpr int64_t kLaunchRows = 1 << 20;

// Workspace of an f32 product over K (0: it does not split K).
int64_t f32_room(int64_t M, int64_t N, int64_t K) {
  const int64_t b = moc_gemm_workspace_size(MOC_F32, M, N, K, 0);
  return b <= MOC_GEMM_WS_COUNTER_BYTES + kF32Parts ? b : 0;
}

// Words whose f32 logits are one product: those whose weights the last-level cache holds
// beside the logits, since every 64 rows read them again: 1024 x 768 x 50257 795 us, in
// one product 1557.
int64_t f32_columns(int64_t ldw) {
  const int64_t fit = kF32Weight / (ldw * 4) / 64 * 64;
  return fit < 1024 ? 1024 : fit;
}

// A teacher as its caller has it.
struct Teacher {
  const void* ids;
  int ids_dtype;
  int64_t ids_ld;
  const void* top;
  int top_dtype;
  int64_t top_ld;
  float heat;
};

template <typename ID, bool TOP_F32>
void launch_teacher(const Teacher& a, int64_t rows, int words, int vocab, const float* row_weight, int mean,
                    const float* grad, const Targets& t, int* counter, hipStream_t st) {
  const ID* ids = static_cast<const ID*>(a.ids);
#define MOC_WAVES(W)                                                                                                \
  teacher_wave_kernel<ID, TOP_F32, W><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, st>>>(                         \
      ids, a.ids_ld, a.top, a.top_ld, rows, words, vocab, a.heat, row_weight, mean, grad, t, counter)
  if (words <= 64) MOC_WAVES(1);
  else if (words <= 128) MOC_WAVES(2);
  else if (words <= 256) MOC_WAVES(4);
  else
    for (int64_t r0 = 0; r0 < rows; r0 += kLaunchRows)
      teacher_targets_kernel<ID, TOP_F32><<<static_cast<unsigned>(std::min(rows - r0, kLaunchRows)), 256, 0, st>>>(
          ids, a.ids_ld, a.top, a.top_ld, words, vocab, a.heat, row_weight, t, r0);
#undef MOC_WAVES
}

// Words, shares and weights; total: the weights' sums too.
int run_teacher(const Teacher& a, int64_t rows, int64_t words, int64_t vocab, const float* row_weight, int mean,
                const float* grad, const Targets& t, bool total, int* counters, hipStream_t st) {
  if (rows == 0) return MOC_OK;
  const int k = static_cast<int>(words), v = static_cast<int>(vocab);
  const bool arrive = words <= 256 && rows <= 2 * kArriveRows;  // four rows a workgroup
  int* counter = total && arrive ? counters + kTeacherCounter : nullptr;
#define MOC_TEACHER(ID, F) launch_teacher<ID, F>(a, rows, k, v, row_weight, mean, grad, t, counter, st)
  if (a.ids_dtype == MOC_I32 && a.top_dtype == MOC_F32) MOC_TEACHER(int32_t, true);
  else if (a.ids_dtype == MOC_I32) MOC_TEACHER(int32_t, false);
  else if (a.top_dtype == MOC_F32) MOC_TEACHER(int64_t, true);
  else MOC_TEACHER(int64_t, false);
#undef MOC_TEACHER
  const int rc = check_launch("teacher_wave_kernel");
  if (rc != MOC_OK || !total || arrive) return rc;
  target_total_kernel<<<1, 1024, 0, st>>>(rows, mean, grad, t);
  return check_launch("target_total_kernel");
}

constexpr int moc_th(int th, int = 0) { return th; }

// The smallest of these that holds a row, so that few of its loads repeat the last
// chunk, and two workgroups or more on a CU (up to 128 registers, 80 KB of LDS), since
// one alone leaves the memory idle while it computes.  us, one / the next:
//   bf16    8000 words x 8192 rows  (4, 256)      55 / (4, 512)        85
//          16000       x 8192       (8, 256)     109 / (4, 512)       121
//          32000       x 8192       (8, 512)     205 / (16, 256)      211, (8, 1024) 334, read twice 317
//          40000       x 4096       (12, 512)    135 / (8, 512, 8)    148, (8, 1024) 193
//          50021       x 4096       (8, 512, 8)  176 / (16, 512)      180, (8, 1024) 228
//          80000       x 2048       (16, 512, 8) 143 / (24, 512, 8)   148, (16, 1024) 181
//         128256       x 2048       (24, 512, 8) 214 / (16, 1024)     253
//   f32   128256       x 2048       (24, 1024, 8) 415 / read twice    507
//         262144       x 1024       read twice by 1024 threads 579 / by 512 625
// (32000 x 8192 in bf16: 5.1 TB/s, 128256 x 2048 in f32: 5.1).
template <typename T>
void launch_logits(const T* x, int64_t rows, int vocab, int64_t ld, const Targets& t, int64_t r0, int words, float heat,
                   const LossOut& o, T* dx, int64_t ldd, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(rows));
  const int chunks = vocab / Elem<T>::kPer;
#define MOC_LOGITS(NC, ...)                                                                                        \
  logits_loss_kernel<T, NC, __VA_ARGS__><<<grid, moc_th(__VA_ARGS__), 0, st>>>(x, ld, vocab, t, r0, words, heat, o, dx, \
                                                                               ldd)
  if (chunks <= 4 * 256) MOC_LOGITS(4, 256);
  else if (chunks <= 8 * 256) MOC_LOGITS(8, 256);
  else if (chunks <= 8 * 512) MOC_LOGITS(8, 512);
  else if (chunks <= 12 * 512) MOC_LOGITS(12, 512);
  else if (chunks <= 16 * 512) MOC_LOGITS(8, 512, 8);
  else if (chunks <= 24 * 512) MOC_LOGITS(16, 512, 8);
  else if (chunks <= 32 * 512) MOC_LOGITS(24, 512, 8);
  else if (chunks <= 32 * 1024) MOC_LOGITS(24, 1024, 8);
  else MOC_LOGITS(0, 1024);
#undef MOC_LOGITS
}

int logits_rows(bool f32, const void* x, int64_t rows, int64_t vocab, int64_t ld, const Targets& t, int64_t r0,
                int64_t words, float heat, const LossOut& o, void* dx, int64_t ldd, hipStream_t st) {
  const int v = static_cast<int>(vocab), k = static_cast<int>(words);
  for (int64_t i = 0; i < rows; i += kLaunchRows) {
    const int64_t n = std::min(rows - i, kLaunchRows);
    auto launch = [&](auto* to) {  // null: no gradients
      auto* from = static_cast<decltype(to)>(const_cast<void*>(x));
      launch_logits(from + i * ld, n, v, ld, t, r0 + i, k, heat, o, to == nullptr ? to : to + i * ldd, ldd, st);
    };
    if (f32) launch(static_cast<float*>(dx));
    else launch(static_cast<uint16_t*>(dx));
  }
  return check_launch("logits_loss_kernel");
}

// The loss where the rows' own launch does not sum it up.
int sum_loss(const Targets& t, LossOut o, float* loss, hipStream_t st) {
  o.loss = loss;
  loss_sum_kernel<<<1, 1024, 0, st>>>(t, o);
  return check_launch("loss_sum_kernel");
}

int few_lds(int64_t hidden) { return static_cast<int>((hidden + 31) / 32) * 1024 + 2 * 4 * 16 * 8; }

// Whether few_rows_kernel takes a piece of the rows.  Not where its workgroups, two
// a CU, have two slabs or more while the tiles of the product are all on a CU at once.
// us, it / the product, of 4 rows and 32000, 50021, 65536 and 128256 words:
//   hidden  512    8.6 / 12.1   13.8 / 13.1    15.3 / 14.9    25.6 / 25.7
//          1024   15.2 / 18.1   22.5 / 19.2    26.2 / 23.0    44.3 / 41.7
//          2048   25.4 / 30.6   41.7 / 31.8    46.3 / 40.9   102.7 / 123.0
//          4096   57.3 / 56.3   94.2 / 94.7   113.9 / 122.9  199.4 / 172 to 209 (one a CU)
bool by_few(int64_t rows, int64_t hidden, int64_t vocab) {
  if (rows > kFewRows || hidden > kFewHidden) return false;
  const int64_t cus = cu_count();
  return 2 * few_lds(hidden) > 160 * 1024 || slabs_of(vocab) <= 2 * cus || (vocab + 255) / 256 > cus;
}

// Logits of up to kFewRows rows.
int launch_few(const void* h, int64_t rows, int64_t hidden, int64_t ldh, const void* w, int64_t vocab, int64_t ldw,
               float unit, const int32_t* ids, int64_t ld_ids, const uint16_t* first, int64_t ld_first, int64_t words,
               float* z, float2* stat, int64_t slabs, void* kept, int64_t ld_kept, hipStream_t st) {
  const int lds = few_lds(hidden);
  // what registers and LDS let a CU have, each as many slabs: 128256 x 4096 203 us, 221
  // with two a CU in turn; 50021 x 768 20.5, 22.8 with a workgroup a slab
  const int64_t resident = static_cast<int64_t>(cu_count()) * (2 * lds > 160 * 1024 ? 1 : 2);
  const int64_t rounds = (slabs + resident - 1) / resident;
  const unsigned grid = static_cast<unsigned>((slabs + rounds - 1) / rounds);
  const bool ragged = hidden % 32 != 0;
  auto kernel = kept != nullptr ? (ragged ? few_rows_kernel<true, true> : few_rows_kernel<false, true>)
                                : (ragged ? few_rows_kernel<true, false> : few_rows_kernel<false, false>);
  kernel<<<grid, 256, lds, st>>>(static_cast<const uint16_t*>(h), ldh, (int)rows, static_cast<const uint16_t*>(w), ldw,
                                 (int)vocab, (int)hidden, unit, ids, ld_ids, first, ld_first, (int)words, z, stat,
                                 (int)slabs, static_cast<_Float16*>(kept), ld_kept);
  return check_launch("few_rows_kernel");
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

bool temperature_ok(float t) { return t > 0.f && t < INFINITY; }

int teacher_ok(const char* name, const Teacher& a, int64_t rows, int64_t words) {
  MOC_REQUIRE((a.ids_dtype == MOC_I32 || a.ids_dtype == MOC_I64) && (a.top_dtype == MOC_BF16 || a.top_dtype == MOC_F32),
              "%s: ids are int32 or int64, the teacher's logits bf16 or f32", name);
  MOC_REQUIRE(rows == 0 || (a.ids != nullptr && a.top != nullptr && (rows == 1 || (a.ids_ld >= words && a.top_ld >= words))),
              "%s: a teacher's operand is null or its rows overlap", name);
  return MOC_OK;
}

}  // namespace
}  // namespace moc

using namespace moc;

#define MOC_SIZES(name)                                                                                          \
  MOC_REQUIRE(sizes_ok(rows, vocab, words), "%s: up to 2^24 rows, a vocabulary of up to 2^21 words, up to %d of " \
                                            "them a row", name, kMaxWords);                                       \
  MOC_REQUIRE(temperature_ok(temperature), "%s: the temperature must be above 0", name)

extern "C" int64_t moc_logits_loss_workspace_size(int64_t rows, int64_t words) {
  if (!sizes_ok(rows, 1, words)) return 0;
  Taken ws{nullptr};
  Targets t{};
  take_targets(ws, rows, words, 0, false, t);
  ws.take<float>(rows);
  return ws.at;
}

extern "C" int moc_logits_loss(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t ld, const void* ids,
                               int ids_dtype, int64_t ids_ld, const void* top, int top_dtype, int64_t top_ld,
                               int64_t words, float temperature, const float* row_weight, int mean, const float* grad,
                               float* row_loss, float* loss, void* dlogits, int64_t ldd, void* workspace,
                               int64_t workspace_bytes, void* counters, void* stream) {
  MOC_SIZES("moc_logits_loss");
  MOC_REQUIRE(dtype == MOC_BF16 || dtype == MOC_F32, "moc_logits_loss: logits are bf16 or f32");
  MOC_REQUIRE(words >= 1, "moc_logits_loss: a word a row at least");
  const Teacher a{ids, ids_dtype, ids_ld, top, top_dtype, top_ld, temperature};
  int rc = teacher_ok("moc_logits_loss", a, rows, words);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(rows == 0 || logits != nullptr, "moc_logits_loss: null logits");
  MOC_REQUIRE(rows <= 1 || (ld >= vocab && (dlogits == nullptr || ldd >= vocab)), "moc_logits_loss: rows that overlap");
  Taken ws{static_cast<char*>(workspace)};
  Targets t{};
  take_targets(ws, rows, words, 0, false, t);
  float* each = ws.take<float>(rows);
  MOC_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= ws.at && counters != nullptr &&
                  aligned16(counters),
              "moc_logits_loss: counters and a workspace of %lld bytes needed", (long long)ws.at);
  if (row_loss == nullptr) row_loss = each;
  hipStream_t st = as_stream(stream);
  int* count = static_cast<int*>(counters);
  const bool total = dlogits != nullptr && rows > 0;
  rc = run_teacher(a, rows, words, vocab, row_weight, mean, grad, t, total, count, st);
  if (rc != MOC_OK) return rc;
  const bool arrive = rows > 0 && rows <= kArriveRows;
  const LossOut o{row_loss, arrive ? loss : nullptr, rows, mean, total, count + kLossCounter};
  if (rows > 0) {
    rc = logits_rows(dtype == MOC_F32, logits, rows, vocab, ld, t, 0, words, temperature, o, dlogits, ldd, st);
    if (rc != MOC_OK) return rc;
  }
  return loss == nullptr || arrive ? MOC_OK : sum_loss(t, o, loss, st);
}

extern "C" int64_t moc_linear_loss_workspace_size(int dtype, int64_t rows, int64_t hidden, int64_t vocab,
                                                  int64_t words, int grads) {
  if (!sizes_ok(rows, vocab, words) || hidden < 1) return 0;
  return pieces_of(dtype, rows, hidden, vocab, words, grads != 0, nullptr).bytes;
}

extern "C" int64_t moc_linear_loss_gemm_workspace_size(int dtype, int64_t rows, int64_t hidden, int64_t vocab,
                                                       int grads) {
  int64_t most = MOC_GEMM_WS_COUNTER_BYTES;
  if (!sizes_ok(rows, vocab, 0) || hidden < 1) return most;
  const Pieces p = pieces_of(dtype, rows, hidden, vocab, 0, grads != 0, nullptr);
  auto need = [&](int64_t b) { most = b > most ? b : most; };
  const int64_t four = p.fused ? vocab : vocab & ~3LL;
  for (int64_t i = 0; i < p.count; i += p.count > 1 ? p.count - 1 : 1) {  // the first piece and the last
    const int64_t n = i + 1 < p.count ? p.rows : rows - i * p.rows;
    if (!p.fused) {
      const int64_t cols = f32_columns((hidden + 3) & ~3LL);
      need(f32_room(n, vocab < cols ? vocab : cols, hidden));
      need(f32_room(n, vocab % cols, hidden));
    }
    if (!grads) continue;
    if (four < vocab) need(f32_room(4, hidden, n));
    need(p.fused ? gemm_half_workspace(in_two_parts(rows, hidden, vocab) ? 2 * n : n, hidden, vocab)
                 : f32_room(n, hidden, four));
    need(p.fused ? gemm_half_workspace(vocab, hidden, n) : f32_room(four, hidden, n));
  }
  return most;
}

extern "C" int moc_linear_loss(int dtype, const void* h, int64_t rows, int64_t hidden, int64_t ldh, const void* w,
                               int64_t vocab, int64_t ldw, const int64_t* labels, int64_t ignore_index, const void* ids,
                               int ids_dtype, int64_t ids_ld, const void* top, int top_dtype, int64_t top_ld,
                               int64_t words, float temperature, const float* row_weight, int mean, const float* grad,
                               float* row_loss, float* loss, void* dh, int dh_dtype, void* dw, int dw_dtype,
                               void* workspace, int64_t workspace_bytes, void* gemm_ws, int64_t gemm_ws_bytes,
                               void* stream) {
  MOC_SIZES("moc_linear_loss");
  MOC_REQUIRE(dtype == MOC_BF16 || dtype == MOC_F32, "moc_linear_loss: operands are bf16 or f32");
  const bool f32 = dtype == MOC_F32;
  const int es = f32 ? 4 : 2;
  MOC_REQUIRE(hidden >= 1 && hidden <= (1 << 20), "moc_linear_loss: hidden size of 1 to 2^20");
  MOC_REQUIRE(w != nullptr && (rows == 0 || h != nullptr), "moc_linear_loss: null operand");
  const Teacher a{ids, ids_dtype, ids_ld, top, top_dtype, top_ld, temperature};
  int rc = MOC_OK;
  if (words > 0) rc = teacher_ok("moc_linear_loss", a, rows, words);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(words > 0 || labels != nullptr || rows == 0, "moc_linear_loss: null labels");
  MOC_REQUIRE(words > 0 || temperature == 1.f, "moc_linear_loss: labels have the temperature 1");
  MOC_REQUIRE(aligned16(h) && aligned16(w) && ldh * es % 16 == 0 && ldw * es % 16 == 0 && ldh >= hidden &&
                  ldw >= hidden,
              "moc_linear_loss: operands need 16-byte aligned rows");
  MOC_REQUIRE(f32 || vocab * ldw * 2 < (1LL << 31) - 1024, "moc_linear_loss: a bf16 weight of up to 2 GiB");
  MOC_REQUIRE((dh == nullptr || (dh_dtype == MOC_F32 || (dh_dtype == MOC_BF16 && !f32))) &&
                  (dw == nullptr || (dw_dtype == MOC_F32 || (dw_dtype == MOC_BF16 && !f32))),
              "moc_linear_loss: gradients are f32, or bf16 of bf16 operands");
  const bool grads = dh != nullptr || dw != nullptr;
  Pieces p = pieces_of(dtype, rows, hidden, vocab, words, grads, workspace);
  MOC_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= p.bytes && gemm_ws != nullptr &&
                  gemm_ws_bytes >= MOC_GEMM_WS_COUNTER_BYTES && aligned16(gemm_ws),
              "moc_linear_loss: workspaces of %lld and at least %d bytes needed", (long long)p.bytes,
              MOC_GEMM_WS_COUNTER_BYTES);
  const int64_t ld_most = ldh > p.ldx ? ldh : p.ldx, ldv_most = ldw > p.ldx ? ldw : p.ldx;
  MOC_REQUIRE(f32 || (p.rows * ld_most * 2 < (1LL << 31) - 1024 && vocab * ldv_most * 2 < (1LL << 31) - 1024),
              "moc_linear_loss: operands of up to 2 GiB a piece");
  hipStream_t st = as_stream(stream);
  int* count = static_cast<int*>(gemm_ws);
  auto room = [&](int64_t M, int64_t N, int64_t K) { return std::min(gemm_ws_bytes, f32_room(M, N, K)); };
  Targets& t = p.t;
  if (words == 0) {
    t.labels = labels;
    t.ignore = ignore_index;
    t.row_weight = row_weight;
  }
  if (row_loss == nullptr) row_loss = p.row_loss;
  const int64_t n_words = words > 0 ? words : 1;
  if (f32 && (rc = moc_fill_zero(count, MOC_GEMM_WS_COUNTER_BYTES, stream)) != MOC_OK) return rc;
  if (words > 0) {
    rc = run_teacher(a, rows, words, vocab, row_weight, mean, grad, t, grads && f32, count, st);
    if (rc != MOC_OK) return rc;
  }
  const bool table = p.fused && words > 0 && rows > 0;
  const unsigned table_blocks = table ? static_cast<unsigned>((rows + 15) / 16) : 0;
  if (table && !grads) {
    words_left_kernel<<<table_blocks, 256, 0, st>>>(t, rows, (int)words, (int)p.slabs);
    if ((rc = check_launch("words_left_kernel")) != MOC_OK) return rc;
  }
  const Halves hx{static_cast<const uint16_t*>(h), ldh, rows, dw != nullptr ? reinterpret_cast<_Float16*>(p.x) : nullptr,
                  0x1p2f, 0x1p-3f, 0x1p13f};
  const bool two = grads && p.fused && in_two_parts(rows, hidden, vocab);
  const bool copy_w = dh != nullptr && !two;
  const Halves hw{static_cast<const uint16_t*>(w), ldw, vocab, copy_w ? reinterpret_cast<_Float16*>(p.w) : nullptr,
                  copy_w ? 0x1p6f : 1.f, 0x1p-7f, 0x1p9f};
  int halves = 0;
  if (grads && rows > 0 && f32) {
    if (words == 0) {
      target_total_kernel<<<1, 1024, 0, st>>>(rows, mean, grad, t);
      if ((rc = check_launch("target_total_kernel")) != MOC_OK) return rc;
    }
    counted_rows_kernel<<<blocks_of(rows * ((hidden + 3) / 4)), 256, 0, st>>>(
        static_cast<const float*>(h), ldh, rows, (int)hidden, t, reinterpret_cast<float*>(p.x), p.ldx);
    if ((rc = check_launch("counted_rows_kernel")) != MOC_OK) return rc;
  } else if (grads && rows > 0) {
    const int64_t most_rows = copy_w && vocab > rows ? vocab : rows, want = (most_rows + 15) / 16;  // four waves of four rows
    halves = static_cast<int>(want < kHalvesBlocks ? want : kHalvesBlocks);
    halves_kernel<<<1 + table_blocks + halves, 256, 0, st>>>(hx, hw, (int)hidden, p.ldx, t, rows, mean, grad, (int)words,
                                                             (int)p.slabs, p.most, halves, count);
    if ((rc = check_launch("halves_kernel")) != MOC_OK) return rc;
  }
  // f32: the rows that count in every product; bf16: in dweight's alone, as nothing is
  // read of the others' logits
  const bool copied = grads && f32;
  const char* x = copied ? p.x : static_cast<const char*>(h);
  const int64_t ldx = copied ? p.ldx : ldh;
  // a label is one word, the low half of its int64
  const int32_t* word_ids = words > 0 ? t.ids : reinterpret_cast<const int32_t*>(labels);
  const int64_t ld_ids = words > 0 ? words : 2;
  const int64_t four = vocab & ~3LL;  // f32 products: rest_words_kernel
  const bool arrive = p.count == 1 && rows <= kArriveRows;
  const LossOut o{row_loss, arrive ? loss : nullptr, rows, mean, grads && rows > 0, count + kLossCounter};
  for (int64_t i = 0; i < p.count; ++i) {
    const int64_t r0 = i * p.rows, n = rows - r0 < p.rows ? rows - r0 : p.rows;
    const char* xi = x + r0 * ldx * es;
    if (p.fused) {
      const uint16_t* first = words > 0 ? t.first + r0 : nullptr;
      const float unit = kLog2E / temperature;
      if (by_few(n, hidden, vocab))
        rc = launch_few(xi, n, hidden, ldx, w, vocab, ldw, unit, word_ids + r0 * ld_ids, ld_ids, first, rows, n_words, p.z,
                        p.stat, p.slabs, grads ? p.d : nullptr, p.ldz, st);
      else
        rc = launch_loss_gemm(xi, n, hidden, ldx, w, vocab, ldw, unit, word_ids + r0 * ld_ids, ld_ids, first, rows, n_words,
                              p.z, p.stat, grads ? p.d : nullptr, p.ldz, st);
      MOC_REQUIRE(rc <= 0, "moc_linear_loss: operands of up to 2 GiB");
      if (rc != MOC_OK) return rc;
      const Slabs s{p.stat, p.z, (int)p.slabs, (int)vocab, (int)words, r0, temperature};
      const int parts = grad_parts(n);
      const unsigned blocks = static_cast<unsigned>(n) * parts + (i == 0 ? kAgainBlocks : 0);
      uint16_t* d = reinterpret_cast<uint16_t*>(p.d);
      if (two && dh != nullptr)
        slabs_grad_kernel<true><<<blocks, 256, 0, st>>>(d, p.ldz, s, t, o, hx, hw, (int)hidden, p.ldx, p.most, halves,
                                                        parts, reinterpret_cast<uint16_t*>(p.two));
      else if (grads)
        slabs_grad_kernel<false><<<blocks, 256, 0, st>>>(d, p.ldz, s, t, o, hx, hw, (int)hidden, p.ldx, p.most, halves,
                                                         parts, nullptr);
      else
        slabs_loss_kernel<<<static_cast<unsigned>(n), 256, 0, st>>>(s, t, o);
      rc = check_launch("slabs_grad_kernel");
    } else {
      const int64_t cols = f32_columns(ldw);
      for (int64_t c = 0; c < vocab && rc == MOC_OK; c += cols) {
        const int64_t m = vocab - c < cols ? vocab - c : cols;
        rc = moc_gemm_ws(dtype, n, m, hidden, xi, ldx, 1, static_cast<const float*>(w) + c * ldw, 1, ldw, 0, nullptr, 0, 0,
                         nullptr, 0, 0, reinterpret_cast<float*>(p.d) + c, p.ldz, MOC_F32, gemm_ws, room(n, m, hidden),
                         stream);
      }
      if (rc != MOC_OK) return rc;
      rc = logits_rows(true, p.d, n, vocab, p.ldz, t, r0, words, temperature, o, grads ? p.d : nullptr, p.ldz, st);
    }
    if (rc != MOC_OK) return rc;
    if (dh != nullptr && two) {
      void* to = static_cast<char*>(dh) + r0 * hidden * (dh_dtype == MOC_F32 ? 4 : 2);
      HalfPair sum{to, dh_dtype, t.alpha, false};
      rc = gemm_pair_rows(n, hidden, vocab, p.two, p.ldz, w, ldw, p.both, sum, gemm_ws, gemm_ws_bytes, stream);
      if (rc != MOC_OK) return rc;
      const int64_t size = n * hidden;
      const unsigned blocks = static_cast<unsigned>((size + 255) / 256);
      if (!sum.done && dh_dtype == MOC_F32)
        two_parts_kernel<float><<<blocks, 256, 0, st>>>(p.both, size, t.alpha, static_cast<float*>(to));
      else if (!sum.done)
        two_parts_kernel<uint16_t><<<blocks, 256, 0, st>>>(p.both, size, t.alpha, static_cast<uint16_t*>(to));
      if ((rc = check_launch("two_parts_kernel")) != MOC_OK) return rc;
    } else if (dh != nullptr && f32) {
      float* to = static_cast<float*>(dh) + r0 * hidden;
      const float *d = reinterpret_cast<const float*>(p.d), *wf = static_cast<const float*>(w);
      // words whose weights the tiled products reach with 32-bit offsets at a time
      const int64_t reach = ((1LL << 31) - 64) / (ldw * 4) / 4 * 4, step = reach < 4 ? 4 : reach;
      for (int64_t c = 0; c < four; c += step) {
        const int64_t k = four - c < step ? four - c : step;
        rc = moc_gemm_ws(dtype, n, hidden, k, d + c, p.ldz, 1, wf + c * ldw, ldw, 1, 0, nullptr, 0, 0, nullptr, 0, 0,
                         c == 0 ? to : p.rest, hidden, MOC_F32, gemm_ws, room(n, hidden, k), stream);
        if (rc != MOC_OK) return rc;
        if (c == 0) continue;
        add_f32_kernel<float><<<blocks_of(n * hidden), 256, 0, st>>>(to, p.rest, n * hidden, nullptr);
        if ((rc = check_launch("add_f32_kernel")) != MOC_OK) return rc;
      }
      if (four < vocab) {
        rest_words_kernel<<<blocks_of(n * hidden), 256, 0, st>>>(d + four, p.ldz, wf + four * ldw, ldw, four > 0,
                                                                 (int)(vocab - four), n, (int)hidden, to);
        if ((rc = check_launch("rest_words_kernel")) != MOC_OK) return rc;
      }
    } else if (dh != nullptr) {
      char* to = static_cast<char*>(dh) + r0 * hidden * (dh_dtype == MOC_F32 ? 4 : 2);
      rc = vocab == 1 ? outer(false, n, hidden, p.d, p.ldz, p.w, t.alpha, to, dh_dtype, st)
                      : gemm_half(n, hidden, vocab, p.d, p.ldz, 1, p.w, p.ldx, to, hidden, dh_dtype, t.alpha, gemm_ws,
                                  gemm_ws_bytes, stream);
      if (rc != MOC_OK) return rc;
    }
    if (dw != nullptr) {
      const bool one = p.count == 1;
      char* to = one ? static_cast<char*>(dw) : reinterpret_cast<char*>(i == 0 ? p.acc : p.part);
      const int to_dtype = one ? dw_dtype : MOC_F32;
      const char* b = p.x + r0 * p.ldx * es;
      // f32: the whole fours, and the words behind them as four of which the first count
      // (columns of p.d up to a multiple of 64 are there; what they hold stays in its rows)
      const int64_t cut = f32 && n > 1 ? four : vocab;
      if (cut < vocab) {
        rc = moc_gemm_ws(dtype, 4, hidden, n, reinterpret_cast<const float*>(p.d) + cut, 1, p.ldz, b, p.ldx, 1, 0, nullptr, 0,
                         0, nullptr, 0, 0, p.rest, hidden, MOC_F32, gemm_ws, room(4, hidden, n), stream);
        if (rc != MOC_OK) return rc;
        const int64_t size = (vocab - cut) * hidden;
        rc = moc_copy_pad_2d(MOC_F32, p.rest, 1, size, size, reinterpret_cast<float*>(to) + cut * hidden, size, size, stream);
        if (rc != MOC_OK) return rc;
      }
      rc = n == 1    ? outer(f32, vocab, hidden, p.d, 1, b, t.alpha + 1, to, to_dtype, st)
           : p.fused ? gemm_half(vocab, hidden, n, p.d, 1, p.ldz, b, p.ldx, to, hidden, to_dtype, t.alpha + 1, gemm_ws,
                                 gemm_ws_bytes, stream)
                     : moc_gemm_ws(dtype, cut, hidden, n, p.d, 1, p.ldz, b, p.ldx, 1, 0, nullptr, 0, 0, nullptr, 0, 0, to,
                                   hidden, to_dtype, gemm_ws, room(cut, hidden, n), stream);
      if (rc != MOC_OK) return rc;
      if (i > 0) {
        const int64_t size = vocab * hidden;
        void* out = i + 1 == p.count ? dw : nullptr;
        if (dw_dtype == MOC_F32)
          add_f32_kernel<float><<<blocks_of(size), 256, 0, st>>>(p.acc, p.part, size, static_cast<float*>(out));
        else
          add_f32_kernel<uint16_t><<<blocks_of(size), 256, 0, st>>>(p.acc, p.part, size, static_cast<uint16_t*>(out));
        if ((rc = check_launch("add_f32_kernel")) != MOC_OK) return rc;
      }
    }
  }
  if (rows == 0 && dw != nullptr) {
    rc = moc_fill_zero(dw, vocab * hidden * (dw_dtype == MOC_F32 ? 4 : 2), stream);
    if (rc != MOC_OK) return rc;
  }
  return loss == nullptr || (rows > 0 && arrive) ? MOC_OK : sum_loss(t, o, loss, st);
}

extern "C" int64_t moc_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(as_stream(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusNone ? 0 : static_cast<int64_t>(id) + 1;
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
