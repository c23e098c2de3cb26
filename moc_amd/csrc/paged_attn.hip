// Causal attention of new tokens over a paged 8-bit cache (gfx950):
//   o = sum_j p_j v_j,  p = softmax_j(scale q k_j) over the positions j that the
//   token sees, k_j and v_j a code times the scale of its page and head.
//
// A row tile holds 16 rows, one column of the MFMA each: the heads of a group
// (those that share a key head) of one token after the other.  Orientation:
// S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_16x16x32_bf16, so a lane has one
// row (l & 15), its softmax factors are per-lane values, and the four positions
// that a 16-position tile of S^T leaves in a lane (4 (l >> 4) + r) are, two
// tiles together, the eight k of the second product's operand: P never moves
// between lanes.  P is rounded to bf16 for that product, V's type there: an error of
// at most 2^-8 of each probability, of either sign, where the output's own rounding
// to bf16 is 2^-8 of the result (together 0.0023 of the output's size against 64
// bits, 0.0017 with P in f32).  P in two bf16 parts would double that product's
// instructions.  The sum below the fraction is of P before the rounding.  V's operand needs the same positions for one dimension: a
// lane reads D / 16 neighbouring dimensions of each of its eight positions and
// transposes them in registers (v_perm).  Codes become bf16 exactly; the page's
// scales go onto the scores and the probabilities in f32, V's before P is rounded.
//
// The cache is read once for a tile, straight into registers; one workgroup
// takes a chunk of the positions, a wave 64 at a time, and the waves join
// through LDS.  Chunks of one row join in a second launch.  Bound: HBM bytes of
// the codes: 64 sequences of up to 8192, 8 key heads of 128, 712 MB in 138 us (5.2
// TB/s; reads alone reach 5.9), 16 of up to 4096, 16 heads, 169 MB in 38 us.
#include <algorithm>

#include "abi.h"
#include "paged.h"

namespace moc {
namespace {

constexpr int kPaWaves = 4;
constexpr int kPaThreads = 64 * kPaWaves;
constexpr int kPaTile = 64;  // positions per wave and step
constexpr int64_t kPaMaxSplits = 1024;
// Rows of a sequence and key head up to which paged_attn_kernel takes it, reading the
// cache once for 16 of them (the tiles of a head run side by side, L2 serves the rest),
// where paged_wide_kernel's four waves read it once for 128 of which most are missing:
// 48 sequences of 8192, 8 key heads of 128: 32 rows 183, 263 us; 48 255, 275; 64 285,
// 277; of 16384, 4 of 64: 153, 228 and 163, 228; of 32768, one of 256: 399, 522 and
// 479, 421.
constexpr int kPaFew = 48;
constexpr int kPaAll = 256;  // rows of a ragged batch up to which it takes all: 2.5 us for a launch without work

struct PagedAttnArgs {
  PagedSeqs s;
  const uint16_t* q;
  int64_t q_ld, q_lh;
  uint16_t* o;
  int64_t o_ld, o_lh;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  int pages, log_page, heads, kv_heads, group;
  float c2;      // scale log2(e)
  int few;       // rows of a sequence for paged_attn_kernel, more for paged_wide_kernel
  int chunk, splits;
  float* part_o;    // [tiles][kv_heads][16 rows][splits][D]
  float2* part_ml;  // [tiles][kv_heads][16 rows][splits]: largest score, sum
  uint32_t wide_chunk;  // paged_wide_kernel's
  int wide_splits;
  float* wide_o;                // [units][kv_heads][128 rows][splits][D]
  float2* wide_ml;
};

// Two codes (bytes 2 H, 2 H + 1 of w) as bf16.
template <bool INT8, bool H>
__device__ __forceinline__ uint32_t two_bf16(uint32_t w) {
  if constexpr (INT8) {
    const float a = static_cast<float>(static_cast<int8_t>(w >> (H ? 16 : 0)));
    const float b = static_cast<float>(static_cast<int8_t>(w >> (H ? 24 : 8)));
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  } else {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, H));
  }
}

template <bool INT8>
__device__ __forceinline__ bf16x8_t eight_bf16(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(bf16x8_t, make_uint4(two_bf16<INT8, false>(lo), two_bf16<INT8, true>(lo),
                                                 two_bf16<INT8, false>(hi), two_bf16<INT8, true>(hi)));
}

__device__ __forceinline__ SeqSpan uniform(SeqSpan s) {
  s.seq = __builtin_amdgcn_readfirstlane(s.seq);
  s.row0 = __builtin_amdgcn_readfirstlane(s.row0);
  s.n = __builtin_amdgcn_readfirstlane(s.n);
  s.unit = __builtin_amdgcn_readfirstlane(s.unit);
  s.len = __builtin_amdgcn_readfirstlane(static_cast<int>(s.len));
  return s;
}

// Where 16-position groups of a head lie and their scales, one group a lane, so
// that the loops look nothing up in memory: the next 64 pages' numbers are on their
// way from when the last 64 were taken.
struct Groups {
  uint32_t lo, hi;  // byte offset of the group's first code
  float ks, vs;     // K's scale times the scores' factor, V's
  int page;         // of the 64 groups after these

  // Position p of this lane's group, or -1.
  __device__ __forceinline__ void ask(const PagedAttnArgs& a, const int32_t* table, int64_t p) {
    page = p >= 0 ? table[p >> a.log_page] : 0;
  }
  __device__ __forceinline__ void take(const PagedAttnArgs& a, int64_t p, int head, int dim) {
    const bool ok = p >= 0 && page >= 0 && page < a.pages;
    const int64_t block = static_cast<int64_t>(ok ? page : 0) * a.kv_heads + head;
    const int64_t byte = ((block << a.log_page) + (p >= 0 ? p & ((1 << a.log_page) - 1) : 0)) * dim;
    lo = static_cast<uint32_t>(byte);
    hi = static_cast<uint32_t>(byte >> 32);
    ks = vs = 1.f;
    if (ok) {
      ks = a.ks[block] * a.c2;
      vs = a.vs[block];
    } else if (p >= 0) {
      ks = __uint_as_float(0x7FC00000u);  // a page out of range: NaN for who sees it
    }
  }
  __device__ __forceinline__ int64_t byte_of(int l) const {
    return static_cast<int64_t>(wave_read_lane(lo, l) | (static_cast<uint64_t>(wave_read_lane(hi, l)) << 32));
  }
  __device__ __forceinline__ float ks_of(int l) const { return __uint_as_float(wave_read_lane(__float_as_uint(ks), l)); }
  __device__ __forceinline__ float vs_of(int l) const { return __uint_as_float(wave_read_lane(__float_as_uint(vs), l)); }
};

// Any of four e4m3 codes NaN.
__device__ __forceinline__ bool has_nan_code(uint32_t w) {
  return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
}

template <int D, bool INT8>
__global__ __launch_bounds__(kPaThreads, D == 64 ? 3 : D == 128 ? 2 : 1) void paged_attn_kernel(PagedAttnArgs a) {
  constexpr int kLoads = D / 64;     // 16-byte loads of a K row per lane
  constexpr int kVDims = D / 16;     // dimensions of V per lane
  constexpr int kVWords = kVDims / 4;
  __shared__ float part[kPaWaves][16][D + 4];
  __shared__ float2 ml[kPaWaves][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, h = lane >> 4;
  const int lp = a.log_page, page = 1 << lp;
  // Workgroups go round the 8 XCDs: a tile's heads and chunks are neighbours, so that
  // all read one long sequence (16 sequences of 16 heads, one of 65536 and the others
  // of 2048 positions: with tiles as neighbours 384 us, so 87), and a short one's only
  // chunk is a different neighbour in each tile
  const uint32_t splits = a.splits, around = blockIdx.x / a.kv_heads, tile = around / splits;
  const int head = blockIdx.x - around * a.kv_heads;
  const uint32_t chunk = (around - tile * splits + tile) % splits;
  // the row tile: rows [unit 16, unit 16 + 16) of a sequence's n group
  SeqSpan sp;
  const int group = a.group;
  if (a.s.cu == nullptr) {
    const int each = (group + 15) / 16;
    sp.seq = sp.row0 = tile / each;
    sp.unit = tile - sp.seq * each;
    sp.n = 1;
    sp.len = a.s.lens[sp.seq];
  } else {
    sp = find_unit(a.s, tile, [group, few = a.few](int n, int64_t) {
      return n * group <= few ? (n * group + 15) / 16 : 0;
    });
    if (sp.seq < 0) return;
  }
  sp = uniform(sp);
  const int r = sp.unit * 16 + col, token = r / group, sub = r - token * group;
  const bool live = token < sp.n;
  const int64_t room = static_cast<int64_t>(a.s.width) << lp;
  // positions that this lane's row sees, and that any row of the tile does
  const int64_t sees = live ? sp.len - sp.n + 1 + token : 0;
  const int last = min(sp.unit * 16 + 15, sp.n * group - 1) / group;
  const int64_t most = min(max(sp.len - sp.n + 1 + last, int64_t(0)), room);
  const bool lost = sees > room;  // positions without a page: NaN
  const int64_t lim = sees;
  const int64_t from = static_cast<int64_t>(chunk) * a.chunk, to = min(most, from + a.chunk);

  bf16x8_t qf[kLoads][2];
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint4 t = make_uint4(0, 0, 0, 0);
      if (live)
        t = *reinterpret_cast<const uint4*>(a.q + (sp.row0 + token) * a.q_ld + (head * group + sub) * a.q_lh + i * 64 +
                                            h * 16 + j * 8);
      qf[i][j] = __builtin_bit_cast(bf16x8_t, t);
    }

  float m = -INFINITY, l = 0.f;
  f32x4_t acc[kVDims];
#pragma unroll
  for (int j = 0; j < kVDims; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int32_t* table = a.s.table + sp.seq * a.s.ld_table;
  const uint32_t k_off = col * D + h * 16, v_off = 4 * h * D + col * kVDims;

  // lane l: group l & 3 of the wave's tile l >> 2
  constexpr int64_t kStep = kPaTile * kPaWaves;
  Groups pg;
  auto group_at = [&](int64_t t0) {
    const int64_t p = t0 + kStep * (lane >> 2) + 16 * (lane & 3);
    return p < to ? p : int64_t(-1);
  };
  // K's registers are loaded again as soon as the scores are computed from them,
  // V's after the products, so that a wave always has one of them on its way
  uint4 kr[4][kLoads];
  uint32_t vr[4][4][kVWords];
  int64_t byte[4];
  auto load_k = [&](int j) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      byte[g] = pg.byte_of(4 * j + g);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) kr[g][i] = *reinterpret_cast<const uint4*>(a.kc + byte[g] + k_off + 64 * i);
    }
  };
  auto load_v = [&] {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* p = a.vc + byte[g] + v_off + i * D;
        if constexpr (kVWords == 1) {
          vr[g][i][0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (kVWords == 2) {
          const uint2 t = *reinterpret_cast<const uint2*>(p);
          vr[g][i][0] = t.x; vr[g][i][1] = t.y;
        } else {
          const uint4 t = *reinterpret_cast<const uint4*>(p);
          vr[g][i][0] = t.x; vr[g][i][1] = t.y; vr[g][i][2] = t.z; vr[g][i][3] = t.w;
        }
      }
  };
  float ksc[4], vsc[4];
  auto scales = [&](int j) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      ksc[g] = pg.ks_of(4 * j + g);
      vsc[g] = pg.vs_of(4 * j + g);
    }
  };
  const int64_t start = from + wave * kPaTile;
  if (start < to) {
    pg.ask(a, table, group_at(start));
    pg.take(a, group_at(start), head, D);
    pg.ask(a, table, group_at(start + 16 * kStep));
    // K before V, as in the loop: its scores wait for K's loads alone
    __builtin_amdgcn_sched_barrier(0);
    load_k(0);
    __builtin_amdgcn_sched_barrier(0);
    load_v();
    __builtin_amdgcn_sched_barrier(0);
    scales(0);
  }
  int j = 0;  // the tile's lanes are 4 j ..
  for (int64_t t0 = start; t0 < to; t0 += kStep) {
    const bool more = t0 + kStep < to;
    float s[4][4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<INT8>(kr[g][i].x, kr[g][i].y), qf[i][0], x, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<INT8>(kr[g][i].z, kr[g][i].w), qf[i][1], x, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[g][i] = x[i] * ksc[g];
    }
    if (more) {
      if (++j == 16) {
        j = 0;
        pg.take(a, group_at(t0 + kStep), head, D);
        pg.ask(a, table, group_at(t0 + 17 * kStep));
      }
      load_k(j);
    }
    const int64_t whole = min(sp.len - sp.n + 1 + sp.unit * 16 / group, to);  // every row sees up to here
    const bool edge = t0 + kPaTile > whole;
    if (edge) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t p = t0 + 16 * g + 4 * h + i;
          // places that a row does not see may hold anything: 0 times a NaN code is
          // NaN.  Such a position's V counts as 0, and its score as NaN
          bool nan = false;
          if constexpr (!INT8) {
#pragma unroll
            for (int w = 0; w < kVWords; ++w) nan |= has_nan_code(vr[g][i][w]);
            nan = (__ballot(nan) >> (16 * h)) & 0xFFFFu;  // in any lane's dimensions
          }
          if (nan) s[g][i] = __uint_as_float(0x7FC00000u);
          if (p >= lim || p >= to) s[g][i] = -INFINITY;
          if (nan || p >= to) {
#pragma unroll
            for (int w = 0; w < kVWords; ++w) vr[g][i][w] = 0;
          }
        }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) mt = fmaxf(mt, s[g][i]);
    mt = fmaxf(mt, __shfl_xor(mt, 16));
    mt = fmaxf(mt, __shfl_xor(mt, 32));
    // m may lag the largest score by 2^8: the sums have the range
    if (__builtin_amdgcn_ballot_w64(mt > m + 8.f) != 0) {
      const float mn = fmaxf(m, mt);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int j = 0; j < kVDims; ++j) acc[j] *= f;
      m = mn;
    }
    const float base = m == -INFINITY ? 0.f : m;
    uint32_t pb[4][2];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = __builtin_amdgcn_exp2f(s[g][i] - base);
        l += p[i];
        p[i] = p[i] == 0.f ? 0.f : p[i] * vsc[g];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pb[g][i] = __builtin_bit_cast(
            uint32_t, __builtin_convertvector((cvt_f32x2_t){p[2 * i], p[2 * i + 1]}, cvt_bf16x2_t));
    }
#pragma unroll
    for (int gg = 0; gg < 2; ++gg) {
      const bf16x8_t pf = __builtin_bit_cast(
          bf16x8_t, make_uint4(pb[2 * gg][0], pb[2 * gg][1], pb[2 * gg + 1][0], pb[2 * gg + 1][1]));
#pragma unroll
      for (int w = 0; w < kVWords; ++w) {
        // [position][two dimensions] -> [dimension][two positions]
        uint32_t x[2][4][2];
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[g][i][0] = two_bf16<INT8, false>(vr[2 * gg + g][i][w]);
            x[g][i][1] = two_bf16<INT8, true>(vr[2 * gg + g][i][w]);
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
          uint32_t v[4];
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              v[2 * g + i] = __builtin_amdgcn_perm(x[g][2 * i + 1][j >> 1], x[g][2 * i][j >> 1], sel);
          const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, make_uint4(v[0], v[1], v[2], v[3]));
          acc[4 * w + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf, acc[4 * w + j], 0, 0, 0);
        }
      }
    }
    if (more) {
      load_v();
      scales(j);
    }
  }
  // join the waves: a lane holds dimensions h D / 4 .. of its row
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (lost) l = __uint_as_float(0x7FC00000u);
  if (h == 0) ml[wave][col] = make_float2(m, l);
#pragma unroll
  for (int j = 0; j < kVDims; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][col][(4 * h + i) * kVDims + j] = acc[j][i];
  __syncthreads();
  constexpr int kPer = D * 16 / kPaThreads;  // values per thread: D / 16
  const int row = tid / 16, d0 = (tid & 15) * kPer;
  const int rr = sp.unit * 16 + row, tk = rr / group, sb = rr - tk * group;
  if (tk >= sp.n) return;
  float mm = -INFINITY, ll = 0.f;
#pragma unroll
  for (int w = 0; w < kPaWaves; ++w) mm = fmaxf(mm, ml[w][row].x);
  const float base = mm == -INFINITY ? 0.f : mm;
  float out[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kPaWaves; ++w) {
    const float f = __builtin_amdgcn_exp2f(ml[w][row].x - base);
    ll += ml[w][row].y * f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[i] += part[w][row][d0 + i] * f;
  }
  const int64_t token_row = sp.row0 + tk;
  if (a.splits == 1) {
    const float inv = ll == 0.f ? 0.f : 1.0f / ll;
    uint16_t* o = a.o + token_row * a.o_ld + (head * group + sb) * a.o_lh + d0;
#pragma unroll
    for (int i = 0; i < kPer; i += 2)
      *reinterpret_cast<uint32_t*>(o + i) =
          __builtin_bit_cast(uint32_t, __builtin_convertvector((cvt_f32x2_t){out[i] * inv, out[i + 1] * inv}, cvt_bf16x2_t));
    return;
  }
  const int64_t slot = ((static_cast<int64_t>(tile) * a.kv_heads + head) * 16 + row) * a.splits + chunk;
  if ((tid & 15) == 0) a.part_ml[slot] = make_float2(mm, ll);
  if (mm == -INFINITY) return;  // nothing in this chunk
  float* po = a.part_o + slot * D + d0;
#pragma unroll
  for (int i = 0; i < kPer; i += 4)
    *reinterpret_cast<float4*>(po + i) = make_float4(out[i], out[i + 1], out[i + 2], out[i + 3]);
}

// o from the chunks of a row: one workgroup a row, 16 bytes of a chunk a thread.
template <int D>
__global__ __launch_bounds__(kPaThreads) void paged_join_kernel(PagedAttnArgs a) {
  constexpr int kLanes = D / 4, kSlots = kPaThreads / kLanes;  // chunks at a time
  __shared__ float weight[kPaMaxSplits];
  __shared__ float red[2][kPaWaves];
  __shared__ float4 sums[kSlots][kLanes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = a.group, row = blockIdx.z;
  SeqSpan sp;
  if (a.s.cu == nullptr) {
    const int tiles = (group + 15) / 16;
    sp.seq = sp.row0 = blockIdx.x / tiles;
    sp.unit = blockIdx.x - sp.seq * tiles;
    sp.n = 1;
  } else {
    sp = find_unit(a.s, blockIdx.x, [group, few = a.few](int n, int64_t) {
      return n * group <= few ? (n * group + 15) / 16 : 0;
    });
    if (sp.seq < 0) return;
  }
  const int r = sp.unit * 16 + row, token = r / group, sub = r - token * group;
  if (token >= sp.n) return;
  const int64_t slot = ((static_cast<int64_t>(blockIdx.x) * a.kv_heads + blockIdx.y) * 16 + row) * a.splits;
  float m = -INFINITY;
  for (int i = tid; i < a.splits; i += kPaThreads) m = fmaxf(m, a.part_ml[slot + i].x);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPaWaves; ++w) m = fmaxf(m, red[0][w]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int i = tid; i < a.splits; i += kPaThreads) {
    const float2 t = a.part_ml[slot + i];
    weight[i] = __builtin_amdgcn_exp2f(t.x - base);
    l += t.x == -INFINITY ? t.y : t.y * weight[i];  // an empty chunk: 0, or NaN where it lies outside the cache
  }
  l = wave_sum(l);
  if (lane == 0) red[1][wave] = l;
  __syncthreads();
  const int c = tid % kLanes, at = tid / kLanes;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = at; i < a.splits; i += kSlots) {
    const float f = weight[i];
    if (f == 0.f) continue;  // also: nothing was written there
    const float4 t = reinterpret_cast<const float4*>(a.part_o + (slot + i) * D)[c];
    v.x += f * t.x;
    v.y += f * t.y;
    v.z += f * t.z;
    v.w += f * t.w;
  }
  sums[at][c] = v;
  __syncthreads();
  if (at > 0) return;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kPaWaves; ++w) l += red[1][w];
#pragma unroll
  for (int i = 1; i < kSlots; ++i) {
    const float4 t = sums[i][c];
    v.x += t.x;
    v.y += t.y;
    v.z += t.z;
    v.w += t.w;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint16_t* o = a.o + static_cast<int64_t>(sp.row0 + token) * a.o_ld + (blockIdx.y * group + sub) * a.o_lh + 4 * c;
  const cvt_bf16x2_t lo = __builtin_convertvector((cvt_f32x2_t){v.x * inv, v.y * inv}, cvt_bf16x2_t);
  const cvt_bf16x2_t hi = __builtin_convertvector((cvt_f32x2_t){v.z * inv, v.w * inv}, cvt_bf16x2_t);
  *reinterpret_cast<uint2*>(o) = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// ------------------------------------------------------------- many rows
// Sequences with more than 48 rows a key head (prompts, chunks of them, groups of
// many drafted tokens): v_mfma_f32_32x32x16_bf16 in the same orientation, 32
// rows a wave, 128 a workgroup over the same tiles of 64 positions, P in bf16 for the
// same reason.  Every thread
// takes its part of the next tile's codes into registers while this one is worked
// on, and stores them to LDS as bf16: a conversion for all waves, where each wave
// converting for itself took 128 instructions a tile and as many permutations to
// transpose V (4 x 1024 new rows over 4096, 16 heads of 128: 279 us, now 236).  V
// is read transposed (ds_read_b64_tr_b16) under the order of positions that the
// scores leave in a lane (attn.hip).  16-byte chunk c of a row of 64 tile positions
// lies in slot c ^ row_swz(row).  Bound by VALU work and LDS reads beside the
// MFMAs: per 64 positions and 32 rows 32 MFMAs of 32 clocks, 32 KB of LDS, 32
// exponentials and about 170 instructions: 722 TFLOP/s for 16 x 1024 rows.  585 for 4
// sequences of different lengths (171 us for 100 GFLOP): their 480 workgroups are one
// round of 25 to 80 tiles each, since chunks go by the table's width and not by a
// unit's own length, and the CUs work 72 % of the time.  The wave
// in its products goes first, the other's softmax fills the gaps (381 us for 4 x 4096
// rows, 409 with equal priorities).
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

// The transposing reads meet four rows in a row at four neighbouring chunks, K's
// reads eight rows at one chunk: both fall on different banks.
template <int D>
__device__ __forceinline__ int row_swz(int r) {
  return D == 64 ? 4 * ((r >> 1) & 1) + ((r >> 2) & 3) : 4 * (r & 3) + ((r >> 2) & 3);
}

constexpr int kPaWide = 32 * kPaWaves;  // rows a workgroup

__device__ __forceinline__ SeqSpan find_wide(const PagedAttnArgs& a, int unit) {
  return uniform(find_unit(a.s, unit, [group = a.group, few = a.few](int n, int64_t) {
    return n * group > few ? (n * group + kPaWide - 1) / kPaWide : 0;
  }));
}

template <int D, bool INT8>
__global__ __launch_bounds__(kPaThreads, D == 256 ? 1 : 2) void paged_wide_kernel(PagedAttnArgs a) {
  constexpr int kLd = D / 64;                 // 16-byte loads per lane of 16 positions
  constexpr int kQ = D / 16, kV = D / 32;     // k steps of the scores, blocks of 32 dimensions
  constexpr int kBytes = kPaTile * D * 2;
  constexpr int kBufs = D <= 128 ? 2 : 1;     // two tiles of LDS: one barrier a tile
  __shared__ __attribute__((aligned(1024))) char lds[kBufs][2][kBytes];
  __shared__ uint32_t nan_at[kBufs][2];  // positions whose V holds a NaN code
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int head = blockIdx.x % a.kv_heads, lp = a.log_page, group = a.group;
  const SeqSpan sp = find_wide(a, blockIdx.x / a.kv_heads);
  if (sp.seq < 0) return;
  // the last rows, which see most, first
  const int unit = (sp.n * group + kPaWide - 1) / kPaWide - 1 - sp.unit;
  const int r0 = unit * kPaWide + wave * 32, r = r0 + col, token = r / group, sub = r - token * group;
  const bool live = token < sp.n;
  const int64_t room = static_cast<int64_t>(a.s.width) << lp, before = sp.len - sp.n;
  const bool lost = live && before + 1 + token > room;
  // a position, of less than 2^31, plus a tile's or a page group's offset: 32 bits
  auto seen = [&](int row) {
    return static_cast<uint32_t>(min(max(before + 1 + min(row, sp.n * group - 1) / group, int64_t(0)), room));
  };
  const uint32_t lim = live ? seen(r) : 0;
  const uint32_t from = blockIdx.y * a.wide_chunk;  // a multiple of a tile
  const uint32_t most = min(seen(unit * kPaWide + kPaWide - 1), from + a.wide_chunk);  // by any row of the workgroup
  const uint32_t mine = r0 < sp.n * group ? seen(r0 + 31) : 0;  // of the wave
  const uint32_t whole = r0 < sp.n * group ? seen(r0) : 0;      // by each row of the wave
  const uint32_t first = seen(unit * kPaWide);                   // by each row of the workgroup

  bf16x8_t qf[kQ];
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    uint4 t = make_uint4(0, 0, 0, 0);
    if (live)
      t = *reinterpret_cast<const uint4*>(a.q + (sp.row0 + token) * a.q_ld + (head * group + sub) * a.q_lh + 16 * i + 8 * h);
    qf[i] = __builtin_bit_cast(bf16x8_t, t);
  }
  float m = -INFINITY, l = 0.f, v_unit = 0.f, unit_inv = 0.f;
  f32x16_t acc[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) acc[j] = f32x16_t{};
  const int32_t* table = a.s.table + sp.seq * a.s.ld_table;

  // wave w stages positions 16 w .. of a tile: 16 D bytes in a row of the cache, load
  // j of lane l is chunk 16 l % D / 16 of row (1024 j + 16 l) / D of them
  Groups pg;  // lane l: positions 16 l .. of 1024 that begin at from or a multiple later
  auto group_at = [&](uint32_t t0) { return t0 + 16 * lane < most ? int64_t(t0 + 16 * lane) : int64_t(-1); };
  uint4 kr[kLd], vr[kLd];
  auto load_tile = [&](uint32_t t0) {
    if (t0 + 16 * wave >= most) return;  // nobody sees what the registers hold
    const int64_t byte = pg.byte_of(static_cast<int>((t0 - from) % 1024) / 16 + wave);
#pragma unroll
    for (int j = 0; j < kLd; ++j) {
      kr[j] = *reinterpret_cast<const uint4*>(a.kc + byte + 1024 * j + 16 * lane);
      vr[j] = *reinterpret_cast<const uint4*>(a.vc + byte + 1024 * j + 16 * lane);
    }
  };
#pragma unroll
  for (int j = 0; j < kLd; ++j) kr[j] = vr[j] = make_uint4(0, 0, 0, 0);
  if (from < most) {
    pg.ask(a, table, group_at(from));
    pg.take(a, group_at(from), head, D);
    pg.ask(a, table, group_at(from + 1024));
    load_tile(from);
  }
  // LDS bytes that this lane reads: of K the row col (+ 32), k step i at k_at ^ 32 i;
  // of V by transposing reads the rows vrow and vrow + 8 (+ 16 g), block j of 32
  // dimensions at v_lo, v_hi ^ 64 j
  const uint32_t k_at = col * (D * 2) + 16 * (h ^ row_swz<D>(col));
  const int vi = lane & 15, vrow = 4 * (lane >> 5) + (vi >> 2), vch = 2 * ((lane >> 4) & 1) + ((vi >> 1) & 1);
  const uint32_t v_lo = vrow * (D * 2) + 16 * (vch ^ row_swz<D>(vrow)) + 8 * (vi & 1);
  const uint32_t v_hi = (vrow + 8) * (D * 2) + 16 * (vch ^ row_swz<D>(vrow + 8)) + 8 * (vi & 1);

  int buf = 0;
  for (uint32_t t0 = from; t0 < most; t0 += kPaTile, buf ^= kBufs - 1) {
    const bool edge_step = !INT8 && t0 + kPaTile > first;  // some row does not see all of it
    float ksc[4], vsc[4];
    {
      const int g0 = static_cast<int>((t0 - from) % 1024) / 16;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        ksc[g] = pg.ks_of(g0 + g);
        vsc[g] = pg.vs_of(g0 + g);
      }
    }
    if (kBufs == 1) __syncthreads();  // the tile before is read
    if (edge_step) {
      if (tid < 2) nan_at[buf][tid] = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kLd; ++j)
        // 0 times a NaN code would reach rows that do not see it
        if (has_nan_code(vr[j].x) || has_nan_code(vr[j].y) || has_nan_code(vr[j].z) || has_nan_code(vr[j].w)) {
          const int row = 16 * wave + (1024 * j + 16 * lane) / D;
          if (t0 + row < most) atomicOr(&nan_at[buf][row >> 5], 1u << (row & 31));
          vr[j] = make_uint4(0, 0, 0, 0);
        }
    }
    char* kt = lds[buf][0];
    char* vt = lds[buf][1];
#pragma unroll
    for (int j = 0; j < kLd; ++j) {
      const int row = 16 * wave + (1024 * j + 16 * lane) / D, c = 2 * (16 * lane % D / 16);
      const uint4 k = kr[j], v = vr[j];
      const int lo = row * (D * 2) + 16 * (c ^ row_swz<D>(row)), hi = row * (D * 2) + 16 * ((c + 1) ^ row_swz<D>(row));
      *reinterpret_cast<bf16x8_t*>(kt + lo) = eight_bf16<INT8>(k.x, k.y);
      *reinterpret_cast<bf16x8_t*>(kt + hi) = eight_bf16<INT8>(k.z, k.w);
      *reinterpret_cast<bf16x8_t*>(vt + lo) = eight_bf16<INT8>(v.x, v.y);
      *reinterpret_cast<bf16x8_t*>(vt + hi) = eight_bf16<INT8>(v.z, v.w);
    }
    if (t0 + kPaTile < most) {
      if ((t0 + kPaTile - from) % 1024 == 0) {
        pg.take(a, group_at(t0 + kPaTile), head, D);
        pg.ask(a, table, group_at(t0 + kPaTile + 1024));
      }
      load_tile(t0 + kPaTile);
    }
    __syncthreads();
    if (t0 >= mine) continue;
    __builtin_amdgcn_s_setprio(1);
    f32x16_t s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) s[b] = f32x16_t{};
#pragma unroll
    for (int i = 0; i < kQ; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const bf16x8_t k = *reinterpret_cast<const bf16x8_t*>(kt + (k_at ^ (32u * i)) + b * (32 * D * 2));
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, qf[i], s[b], 0, 0, 0);
      }
    __builtin_amdgcn_s_setprio(0);
    // x[i]: position 32 (i >> 4) + 8 ((i >> 2) & 3) + 4 h + (i & 3), group i >> 3
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = s[i >> 4][i & 15];
    bool usual = true;  // scales above 0: the largest score is the largest product
#pragma unroll
    for (int g = 0; g < 4; ++g) usual = usual && ksc[g] > 0.f;
    if (!usual) {
      asm volatile("");  // a branch, not 32 selects in every tile
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float sign = ksc[g] < 0.f ? -1.f : 1.f;
        ksc[g] = ksc[g] == 0.f ? 1e-30f : fabsf(ksc[g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[8 * g + i] *= sign;
      }
    }
    if (t0 + kPaTile > whole) {
      uint32_t nans[2] = {edge_step ? nan_at[buf][0] : 0u, edge_step ? nan_at[buf][1] : 0u};
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (!(fabsf(vsc[g]) <= 3.4028234e38f) || !(ksc[g] <= 3.4028234e38f)) {
          nans[g >> 1] |= 0xFFFFu << (16 * (g & 1));
          ksc[g] = vsc[g] = 1.f;
        }
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int at = 8 * ((i >> 2) & 3) + 4 * h + (i & 3);
        if ((nans[i >> 4] >> at) & 1) x[i] = __uint_as_float(0x7FC00000u);
        if (t0 + 32 * (i >> 4) + at >= lim) x[i] = -INFINITY;
      }
    } else if (edge_step) {
      if (nan_at[buf][0] | nan_at[buf][1]) l = __uint_as_float(0x7FC00000u);  // every row of the wave sees it
    }
    float mt = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float y = x[8 * g];
#pragma unroll
      for (int i = 1; i < 8; ++i) y = fmaxf(y, x[8 * g + i]);
      mt = fmaxf(mt, y * ksc[g]);
    }
    mt = fmaxf(mt, __shfl_xor(mt, 32));
    // m may lag the largest score by 2^8: of 32 rows some find a larger one in most
    // tiles, and the sums have the range
    if (__builtin_amdgcn_ballot_w64(mt > m + 8.f) != 0) {
      const float mn = fmaxf(m, mt);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] *= f;
      m = mn;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[8 * g + i] = __builtin_amdgcn_exp2f(fmaf(x[8 * g + i], ksc[g], -base));
        l += x[8 * g + i];
      }
    // V's scale goes onto the probabilities, relative to the first one: pages of
    // one size of values share theirs
    if (v_unit == 0.f) {
      v_unit = vsc[0] >= 1e-30f && vsc[0] <= 1e30f ? vsc[0] : 1.f;
      unit_inv = 1.0f / v_unit;
    }
    if (vsc[0] != v_unit || vsc[1] != v_unit || vsc[2] != v_unit || vsc[3] != v_unit) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float f = vsc[g] * unit_inv;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[8 * g + i] *= f;
      }
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      uint32_t pb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        pb[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(
                                                 (cvt_f32x2_t){x[8 * g + 2 * i], x[8 * g + 2 * i + 1]}, cvt_bf16x2_t));
      const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, make_uint4(pb[0], pb[1], pb[2], pb[3]));
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const char* const lo = vt + (v_lo ^ (64u * j)) + 16 * g * (D * 2);
        const char* const hi = vt + (v_hi ^ (64u * j)) + 16 * g * (D * 2);
        const i16x4_t v[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)lo),
                              __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)hi)};
        acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v), pf, acc[j], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
  l += __shfl_xor(l, 32);
  if (lost) l = __uint_as_float(0x7FC00000u);
  if (!live) return;
  if (a.wide_splits > 1) {
    const int64_t slot = (static_cast<int64_t>(blockIdx.x) * kPaWide + wave * 32 + col) * a.wide_splits + blockIdx.y;
    if (h == 0) a.wide_ml[slot] = make_float2(m, l);
    if (m == -INFINITY) return;  // nothing here
    float* o = a.wide_o + slot * D;
#pragma unroll
    for (int j = 0; j < kV; ++j)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(o + 32 * j + 2 * i + 4 * h) = make_float4(
            acc[j][i] * v_unit, acc[j][i + 1] * v_unit, acc[j][i + 2] * v_unit, acc[j][i + 3] * v_unit);
    return;
  }
  const float inv = l == 0.f ? 0.f : v_unit / l;
  uint16_t* o = a.o + (sp.row0 + token) * a.o_ld + (head * group + sub) * a.o_lh;
#pragma unroll
  for (int j = 0; j < kV; ++j)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const cvt_bf16x2_t lo = __builtin_convertvector((cvt_f32x2_t){acc[j][i] * inv, acc[j][i + 1] * inv}, cvt_bf16x2_t);
      const cvt_bf16x2_t hi = __builtin_convertvector((cvt_f32x2_t){acc[j][i + 2] * inv, acc[j][i + 3] * inv}, cvt_bf16x2_t);
      *reinterpret_cast<uint2*>(o + 32 * j + 2 * i + 4 * h) =
          make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
    }
}

// o of paged_wide_kernel's rows from their chunks: 8 dimensions of a row a thread.
template <int D>
__global__ __launch_bounds__(kPaThreads) void paged_wide_join_kernel(PagedAttnArgs a) {
  constexpr int kLanes = D / 8, kAtOnce = kPaThreads / kLanes;
  const int group = a.group, c = threadIdx.x % kLanes;
  const int unit = blockIdx.x / a.kv_heads, head = blockIdx.x - unit * a.kv_heads;
  const SeqSpan sp = find_wide(a, unit);
  if (sp.seq < 0) return;
  const int row = blockIdx.y * kAtOnce + threadIdx.x / kLanes;
  const int r = ((sp.n * group + kPaWide - 1) / kPaWide - 1 - sp.unit) * kPaWide + row;
  const int token = r / group, sub = r - token * group;
  if (token >= sp.n) return;
  const int64_t slot = (static_cast<int64_t>(blockIdx.x) * kPaWide + row) * a.wide_splits;
  float m = -INFINITY;
  for (int i = 0; i < a.wide_splits; ++i) m = fmaxf(m, a.wide_ml[slot + i].x);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float v[8] = {};
  for (int i = 0; i < a.wide_splits; ++i) {
    const float2 t = a.wide_ml[slot + i];
    if (t.x == -INFINITY) {
      l += t.y;  // 0, or NaN where a chunk lies outside the cache
      continue;
    }
    const float f = __builtin_amdgcn_exp2f(t.x - base);
    l += t.y * f;
    const float4* p = reinterpret_cast<const float4*>(a.wide_o + (slot + i) * D + 8 * c);
    const float4 x = p[0], y = p[1];
    v[0] += x.x * f; v[1] += x.y * f; v[2] += x.z * f; v[3] += x.w * f;
    v[4] += y.x * f; v[5] += y.y * f; v[6] += y.z * f; v[7] += y.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((cvt_f32x2_t){v[2 * i] * inv, v[2 * i + 1] * inv}, cvt_bf16x2_t));
  uint16_t* o = a.o + (sp.row0 + token) * a.o_ld + (head * group + sub) * a.o_lh + 8 * c;
  *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace
}  // namespace moc

using namespace moc;

namespace {
// The positions' chunks of both kernels.
constexpr int64_t kPaLongest = 8192;  // positions
constexpr int64_t kWidePlaces = 2, kWideLeast = 512;  // workgroups a CU, positions
constexpr int64_t kPaRoom = 1LL << 30;                 // positions of a table: 32-bit arithmetic
struct Plan {
  int64_t tiles, chunk, splits, few;
  int64_t units, wide_chunk, wide_splits;
  int64_t few_floats, wide_floats;  // of partial sums
};
Plan plan_of(int64_t tokens, int64_t seqs, bool ragged, int64_t group, int64_t kv_heads, int64_t dim, int64_t room) {
  Plan p;
  const int64_t rows = tokens * group, with_rows = std::min(seqs, tokens);
  p.few = !ragged ? group : rows <= kPaAll ? kPaAll : kPaFew;
  p.tiles = !ragged ? seqs * ((group + 15) / 16)
            : p.few == kPaAll ? rows / 16 + with_rows
            : group <= kPaFew ? std::min(rows / 16 + with_rows, with_rows * (kPaFew / 16)) : 0;
  // paged_attn_kernel, whole steps: one workgroup a CU keeps more loads in flight than
  // several that begin and join, and without chunks there is no second launch.  Row
  // tiles x key heads, 32 heads of 128 over 4096 positions, us with a workgroup a CU
  // and with four: 64 19.7, 20.2; 160 27.9, 35.5; 256 43.4, 46.8; past that, where the
  // second round of CUs is nearly empty, 272 66.4, 54.8; 384 82.9, 78.9; and where two
  // a CU are nearly full, 448 87.2, 94.6.  Tables of less than 4096 positions stay whole
  // there (want is 0): 272 tiles of 1024 positions 20.3 us, with four a CU 21.9, of 512
  // 13.2, 16.3, and of heads of 64 up to 4032 35.7, 36.3; of 128 from 2048 on the split
  // would gain, 40.5, 36.1, and 384 tiles 44.1, 44.3.  A sequence far longer than the others is the
  // end of the call, so chunks are of about 8192 positions at most (one of 65536 among
  // 16: whole 383 us, 16384 126, 8192 87, 4096 85; 64 of 8192: 191, with 4096 203).
  // The tiles are counted as if the rows were spread evenly: the grid's bound is more
  // than most calls have.
  const int64_t step = kPaTile * kPaWaves, cus = cu_count();
  const int64_t tiles =
      kv_heads * (ragged ? std::min(p.tiles, with_rows * ((rows + 16 * with_rows - 1) / (16 * with_rows))) : p.tiles);
  const int64_t steps = std::max<int64_t>(1, (room + step - 1) / step);
  int64_t want = std::max<int64_t>(tiles > 0 ? cus / tiles : 1, (room + kPaLongest / 2) / kPaLongest);
  if (tiles * want > cus && 4 * tiles * want < 7 * cus) want = 4 * cus / tiles;
  want = std::min(std::max<int64_t>(want, 1), kPaMaxSplits);
  const int64_t per = (steps + want - 1) / want;
  p.chunk = per * step;
  p.splits = (steps + per - 1) / per;
  p.few_floats = p.splits > 1 ? p.tiles * kv_heads * 16 * p.splits * dim : 0;
  // paged_wide_kernel: two workgroups a CU, counted as if the rows were spread evenly;
  // more are more to join.  With 1, 2, 4 of them a CU at most: 352, 211, 222 us (512
  // rows over 32768, 16 heads), 203, 189, 193 (2900 rows of 4 sequences of up to 5120),
  // 92 and 103 with 2 and 4 (16 sequences of 8192, 64 rows of 8 heads).
  p.units = ragged && p.few == kPaFew ? rows / kPaWide + with_rows : 0;
  const int64_t units = kv_heads * with_rows * ((rows + kPaWide * with_rows - 1) / (kPaWide * with_rows));
  const int64_t places = std::max<int64_t>(1, kWidePlaces * cus / units);
  const int64_t wide_per = (room / places + kPaTile - 1) / kPaTile * kPaTile;
  p.wide_chunk = std::max<int64_t>(kWideLeast, wide_per);
  p.wide_splits = std::max<int64_t>(1, (room + p.wide_chunk - 1) / p.wide_chunk);
  p.wide_floats = p.units > 0 && p.wide_splits > 1 ? p.units * kv_heads * kPaWide * p.wide_splits * dim : 0;
  return p;
}
}  // namespace

extern "C" int64_t moc_paged_attention_workspace_size(int64_t tokens, int64_t seqs, int ragged, int64_t q_heads,
                                                      int64_t kv_heads, int64_t head_dim, int64_t page, int64_t width) {
  if (tokens <= 0 || seqs <= 0 || kv_heads <= 0 || q_heads <= 0 || head_dim <= 0) return 0;
  if (page <= 0 || width < 0 || width > kPaRoom / page) return 0;  // refused
  const Plan p = plan_of(tokens, seqs, ragged != 0, q_heads / kv_heads, kv_heads, head_dim, page * width);
  return (p.few_floats + p.wide_floats) / head_dim * (head_dim * 4 + 8);
}

extern "C" int moc_paged_attention_bf16(const void* q, int64_t q_ld, int64_t q_lh, int64_t tokens, int64_t q_heads,
                                        int64_t kv_heads, int64_t head_dim, int code, const void* k_codes,
                                        const void* v_codes, const float* k_scale, const float* v_scale, int64_t pages,
                                        int64_t page, const int32_t* table, int64_t ld_table, int64_t width,
                                        const int32_t* lens, const int32_t* cu, int64_t seqs, float scale, void* out,
                                        int64_t o_ld, int64_t o_lh, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
  MOC_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256,
              "moc_paged_attention_bf16: head_dim must be 64, 128 or 256");
  MOC_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0,
              "moc_paged_attention_bf16: page must be a power of two from 16 to 256");
  MOC_REQUIRE(code == MOC_E4M3 || code == MOC_I8, "moc_paged_attention_bf16: codes must be e4m3 or int8");
  MOC_REQUIRE(tokens >= 0 && seqs >= 0 && kv_heads >= 1 && q_heads >= 1 && q_heads % kv_heads == 0 && width >= 0 &&
                  pages >= 0 && tokens < (1 << 24) && seqs < (1 << 24) && kv_heads <= 65535 && q_heads <= 65536 &&
                  pages < (1LL << 31) && width < (1LL << 31) && tokens * (q_heads / kv_heads) < (1LL << 31),
              "moc_paged_attention_bf16: bad shape");
  MOC_REQUIRE(page * width <= kPaRoom, "moc_paged_attention_bf16: tables of at most 2^30 positions");
  MOC_REQUIRE(cu != nullptr || tokens == seqs, "moc_paged_attention_bf16: one token a sequence without cu");
  if (tokens == 0 || seqs == 0) return MOC_OK;
  MOC_REQUIRE(pages >= 1, "moc_paged_attention_bf16: the cache has no pages");
  MOC_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && (table || width == 0) && lens && out,
              "moc_paged_attention_bf16: null pointer");
  MOC_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_codes) && aligned16(v_codes) &&
                  (q_ld | q_lh | o_ld | o_lh) % 8 == 0,
              "moc_paged_attention_bf16: rows must be 16-byte aligned");
  const int64_t group = q_heads / kv_heads;
  const Plan p = plan_of(tokens, seqs, cu != nullptr, group, kv_heads, head_dim, page * width);
  const int64_t need = moc_paged_attention_workspace_size(tokens, seqs, cu != nullptr, q_heads, kv_heads, head_dim, page,
                                                          width);
  MOC_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
              "moc_paged_attention_bf16: workspace of %lld bytes required", (long long)need);
  PagedAttnArgs a;
  a.s = PagedSeqs{cu, lens, table, ld_table, static_cast<int>(seqs), static_cast<int>(tokens), static_cast<int>(width)};
  a.q = static_cast<const uint16_t*>(q);
  a.q_ld = q_ld; a.q_lh = q_lh;
  a.o = static_cast<uint16_t*>(out);
  a.o_ld = o_ld; a.o_lh = o_lh;
  a.kc = static_cast<const uint8_t*>(k_codes);
  a.vc = static_cast<const uint8_t*>(v_codes);
  a.ks = k_scale; a.vs = v_scale;
  a.pages = static_cast<int>(pages);
  a.log_page = __builtin_ctzll(static_cast<unsigned long long>(page));
  a.heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(group);
  a.c2 = scale * 1.4426950408889634f;
  a.chunk = static_cast<int>(p.chunk);
  a.splits = static_cast<int>(p.splits);
  a.few = static_cast<int>(p.few);
  a.part_o = static_cast<float*>(workspace);
  a.wide_o = a.part_o + p.few_floats;
  a.part_ml = reinterpret_cast<float2*>(a.wide_o + p.wide_floats);
  a.wide_ml = a.part_ml + p.few_floats / head_dim;
  a.wide_chunk = static_cast<uint32_t>(p.wide_chunk);
  a.wide_splits = static_cast<int>(p.wide_splits);
  hipStream_t st = as_stream(stream);
  int rc = MOC_OK;
  if (p.units > 0) {
    MOC_REQUIRE(p.units * kv_heads < (1LL << 31) && p.wide_splits <= 65535,
                "moc_paged_attention_bf16: too many rows for one call");
    const dim3 grid(static_cast<unsigned>(p.units * kv_heads), static_cast<unsigned>(p.wide_splits));
#define MOC_PW(D)                                                                  \
  do {                                                                             \
    if (code == MOC_I8) paged_wide_kernel<D, true><<<grid, kPaThreads, 0, st>>>(a); \
    else paged_wide_kernel<D, false><<<grid, kPaThreads, 0, st>>>(a);              \
  } while (0)
    if (head_dim == 64) MOC_PW(64);
    else if (head_dim == 128) MOC_PW(128);
    else MOC_PW(256);
#undef MOC_PW
    rc = check_launch("paged_wide_kernel");
    if (rc != MOC_OK) return rc;
    if (p.wide_splits > 1) {
      const dim3 jg(static_cast<unsigned>(p.units * kv_heads), static_cast<unsigned>(kPaWide * head_dim / 8 / kPaThreads));
      if (head_dim == 64) paged_wide_join_kernel<64><<<jg, kPaThreads, 0, st>>>(a);
      else if (head_dim == 128) paged_wide_join_kernel<128><<<jg, kPaThreads, 0, st>>>(a);
      else paged_wide_join_kernel<256><<<jg, kPaThreads, 0, st>>>(a);
      rc = check_launch("paged_wide_join_kernel");
      if (rc != MOC_OK) return rc;
    }
  }
  if (p.tiles == 0) return rc;
  MOC_REQUIRE(p.tiles * kv_heads * p.splits < (1LL << 31), "moc_paged_attention_bf16: too many rows for one call");
  const dim3 grid(static_cast<unsigned>(p.tiles * kv_heads * p.splits));
#define MOC_PA(D)                                                                  \
  do {                                                                             \
    if (code == MOC_I8) paged_attn_kernel<D, true><<<grid, kPaThreads, 0, st>>>(a); \
    else paged_attn_kernel<D, false><<<grid, kPaThreads, 0, st>>>(a);              \
  } while (0)
  if (head_dim == 64) MOC_PA(64);
  else if (head_dim == 128) MOC_PA(128);
  else MOC_PA(256);
#undef MOC_PA
  rc = check_launch("paged_attn_kernel");
  if (rc != MOC_OK || p.splits == 1) return rc;
  const dim3 jg(static_cast<unsigned>(p.tiles), static_cast<unsigned>(kv_heads),
                static_cast<unsigned>(cu != nullptr ? 16 : std::min<int64_t>(group, 16)));
  if (head_dim == 64) paged_join_kernel<64><<<jg, kPaThreads, 0, st>>>(a);
  else if (head_dim == 128) paged_join_kernel<128><<<jg, kPaThreads, 0, st>>>(a);
  else paged_join_kernel<256><<<jg, kPaThreads, 0, st>>>(a);
  return check_launch("paged_join_kernel");
}
