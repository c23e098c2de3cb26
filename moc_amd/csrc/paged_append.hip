// New tokens into a paged 8-bit cache, queries and keys rotated on the way
// (gfx950): the cache half of a decode or prompt step of several sequences, as
// decode_qkv_kernel's last lines are of one (attn_decode.hip).
//
// Rotation: pairs (x[2i], x[2i+1]) by the angle of (position, i), cos and sin
// given, in f32; q is rounded to bf16 once, k goes to its code from f32.
//
// A block is a page's places of one head, of K or of V.  Its scale is the least
// power of two s with |x| <= largest * s for every x that it holds, at least
// 2^-100: what the block held gives its old scale (none where the call writes
// its first place), the call's tokens their largest magnitude.  Powers of two
// make x / s exact, and where s grows the older codes are encoded again without
// loss (e4m3 above its subnormals) or with one rounding to the coarser grid
// (int8).  Codes: nearest, ties to even; no finite value exceeds the largest.
//
// One wave takes one block (or one query head) of the tokens that one page gets
// in this call: its scale needs them all, and no workgroup has to meet.
// Bound for prompts by HBM traffic and by arithmetic beside it (9 of up to 1000
// tokens, 32 heads of 64: 132 MB in 30 us, where a copy of the 113 MB needed takes
// 22; VALU instructions issue in 45 % of the clocks: each head turns its own angles
// to f32, a key's or value's wave reads its rows, and turns a key's, once for the
// largest value and once for the codes), by the chain length -> page -> scale ->
// store for single tokens (64 of them, 8 key heads: 4.4 us).
#include "abi.h"
#include "paged.h"

namespace moc {
namespace {

struct AppendArgs {
  PagedSeqs s;
  const uint16_t *q, *k, *v;
  int64_t q_ld, q_lh, k_ld, k_lh, v_ld, v_lh;  // elements between tokens, heads
  uint16_t* q_out;
  int64_t o_ld, o_lh;
  const void *cos, *sin;  // [angles, dim / 2]
  int angles;
  uint8_t *kc, *vc;
  float *ks, *vs;
  int pages, log_page, q_heads, kv_heads;
};

// Least power of two s >= 2^-100 with x <= largest * s, largest = m 2^e with m
// in [1, 2): the exponent of x, one more where x's mantissa exceeds m.
template <bool INT8>
__device__ __forceinline__ float scale_for(float x) {
  constexpr uint32_t kMant = INT8 ? 0x7E0000u : 0x600000u;  // 127 = 1.984375 2^6, 448 = 1.75 2^8
  constexpr int kExp = INT8 ? 6 : 8;
  const uint32_t u = __float_as_uint(x);
  const int e = static_cast<int>(u >> 23) - kExp + ((u & 0x7FFFFFu) > kMant ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 27)) << 23);
}

// The least power of two >= x (x >= 0, finite), at least 2^-100.
__device__ __forceinline__ float power_above(float x) {
  const uint32_t u = __float_as_uint(x);
  return __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(u >> 23) + ((u & 0x7FFFFFu) ? 1 : 0), 27)) << 23);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.4028234e38f ? a : 0.f;
}

// Four values, already divided by the scale, as codes.  Not finite: the NaN
// code (e4m3); int8 has none, NaN becomes 0 and infinities the ends.
template <bool INT8>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (INT8) {
    auto one = [](float x) -> uint32_t {
      const float r = x != x ? 0.f : fminf(fmaxf(rintf(x), -127.f), 127.f);
      return static_cast<uint32_t>(static_cast<int>(r)) & 0xFFu;
    };
    return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
  } else {
    const float nan = __uint_as_float(0x7FC00000u);
    auto ok = [nan](float x) { return fabsf(x) <= 448.f ? x : nan; };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(ok(a), ok(b), 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(ok(c), ok(d), w, true));
  }
}

template <bool INT8>
__device__ __forceinline__ void decode4(uint32_t w, float (&x)[4]) {
  if constexpr (INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  } else {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = lo.x; x[1] = lo.y; x[2] = hi.x; x[3] = hi.y;
  }
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// Eight values of a row from its 16-byte chunk, rotated if cos is given.
template <bool TF32>
__device__ __forceinline__ void load8(const uint16_t* p, const AppendArgs& a, bool turn, int64_t angle, float (&x)[8]) {
  const uint4 t = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  if (!turn) return;
  float c[4], s[4];
  if (TF32) {
    const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(a.cos) + angle);
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(a.sin) + angle);
    c[0] = u.x; c[1] = u.y; c[2] = u.z; c[3] = u.w;
    s[0] = v.x; s[1] = v.y; s[2] = v.z; s[3] = v.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.cos) + angle);
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.sin) + angle);
    c[0] = __uint_as_float(u.x << 16); c[1] = __uint_as_float(u.x & 0xFFFF0000u);
    c[2] = __uint_as_float(u.y << 16); c[3] = __uint_as_float(u.y & 0xFFFF0000u);
    s[0] = __uint_as_float(v.x << 16); s[1] = __uint_as_float(v.x & 0xFFFF0000u);
    s[2] = __uint_as_float(v.y << 16); s[3] = __uint_as_float(v.y & 0xFFFF0000u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float e = x[2 * i], o = x[2 * i + 1];
    x[2 * i] = e * c[i] - o * s[i];
    x[2 * i + 1] = e * s[i] + o * c[i];
  }
}

__device__ __forceinline__ int page_units(int n, int64_t len, int log_page) {
  return static_cast<int>(((len - 1) >> log_page) - ((len - n) >> log_page)) + 1;
}

template <int D, bool INT8, bool TF32>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  constexpr int kCh = D / 8, kRows = 64 / kCh;  // chunks a row, rows a pass
  const int lane = threadIdx.x & 63, heads = a.q_heads + 2 * a.kv_heads;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int unit = static_cast<int>(id / heads);
  int head = static_cast<int>(id - static_cast<int64_t>(unit) * heads);
  const int lp = a.log_page, page = 1 << lp;
  SeqSpan sp;
  if (a.s.cu == nullptr) {
    if (unit >= a.s.seqs) return;
    sp.seq = sp.row0 = unit;
    sp.n = 1;
    sp.unit = 0;
    sp.len = a.s.lens[unit];
  } else {
    sp = find_unit(a.s, unit, [lp](int n, int64_t len) { return page_units(n, len, lp); });
    if (sp.seq < 0) return;
  }
  // this unit's positions [lo, hi) and the row of the first
  const int64_t first = sp.len - sp.n, index = (first >> lp) + sp.unit;
  const int64_t lo = max(first, index << lp), hi = min(sp.len, (index + 1) << lp);
  const int row = sp.row0 + static_cast<int>(lo - first), n = static_cast<int>(hi - lo);
  const bool is_q = head < a.q_heads;
  // of these, the ones with a place in the table and an angle
  const int good = index >= 0 && index < a.s.width ? static_cast<int>(min(max(a.angles - lo, int64_t(0)), int64_t(n))) : 0;
  const int c = lane % kCh, r0 = lane / kCh;
  if (is_q) {
    // no place in the cache: zeros before position 0 (padding), else NaN
    for (int r = r0; r < n; r += kRows) {
      uint4 out;
      if (r < good) {
        float x[8];
        load8<TF32>(a.q + (row + r) * a.q_ld + head * a.q_lh + 8 * c, a, true, (lo + r) * (D / 2) + 4 * c, x);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((cvt_f32x2_t){x[2 * i], x[2 * i + 1]}, cvt_bf16x2_t));
        out = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        const uint32_t f = lo + r < 0 ? 0u : 0x7FC07FC0u;
        out = make_uint4(f, f, f, f);
      }
      *reinterpret_cast<uint4*>(a.q_out + (row + r) * a.o_ld + head * a.o_lh + 8 * c) = out;
    }
    return;
  }
  if (good == 0) return;
  const int id_page = a.s.table[sp.seq * a.s.ld_table + index];
  if (id_page < 0 || id_page >= a.pages) return;
  head -= a.q_heads;
  const bool is_k = head < a.kv_heads;
  if (!is_k) head -= a.kv_heads;
  const uint16_t* src = is_k ? a.k + head * a.k_lh : a.v + head * a.v_lh;
  const int64_t ld = is_k ? a.k_ld : a.v_ld;
  const int64_t block = static_cast<int64_t>(id_page) * a.kv_heads + head;
  uint8_t* codes = (is_k ? a.kc : a.vc) + (block << lp) * D;
  float* scale = (is_k ? a.ks : a.vs) + block;
  const int place = static_cast<int>(lo & (page - 1));
  const float old = place > 0 ? *scale : 0.f;
  float most = 0.f;
  for (int r = r0; r < good; r += kRows) {
    float x[8];
    load8<TF32>(src + (row + r) * ld + 8 * c, a, is_k, (lo + r) * (D / 2) + 4 * c, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, finite_abs(x[i]));
  }
  most = wave_max(most);
  const float s = fmaxf(scale_for<INT8>(most), power_above(finite_abs(old)));
  const float inv = 1.0f / s;
  for (int r = r0; r < good; r += kRows) {
    float x[8];
    load8<TF32>(src + (row + r) * ld + 8 * c, a, is_k, (lo + r) * (D / 2) + 4 * c, x);
    uint2 w;
    w.x = encode4<INT8>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    w.y = encode4<INT8>(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    *reinterpret_cast<uint2*>(codes + (place + r) * D + 8 * c) = w;
  }
  if (place > 0 && old != s) {  // the older codes, on the new scale
    const float f = old * inv;
    for (int i = lane; i < place * (D / 4); i += 64) {
      float x[4];
      decode4<INT8>(reinterpret_cast<const uint32_t*>(codes)[i], x);
      reinterpret_cast<uint32_t*>(codes)[i] = encode4<INT8>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
    }
  }
  if (lane == 0 && (place == 0 || old != s)) *scale = s;
}

}  // namespace
}  // namespace moc

using namespace moc;

extern "C" int moc_paged_append_bf16(const void* q, int64_t q_ld, int64_t q_lh, const void* k, int64_t k_ld,
                                     int64_t k_lh, const void* v, int64_t v_ld, int64_t v_lh, int64_t tokens,
                                     int64_t q_heads, int64_t kv_heads, int64_t head_dim, const void* cos,
                                     const void* sin, int table_dtype, int64_t angles, int code, void* k_codes,
                                     void* v_codes, float* k_scale, float* v_scale, int64_t pages, int64_t page,
                                     const int32_t* table, int64_t ld_table, int64_t width, const int32_t* lens,
                                     const int32_t* cu, int64_t seqs, void* q_out, int64_t o_ld, int64_t o_lh,
                                     void* stream) {
  MOC_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256,
              "moc_paged_append_bf16: head_dim must be 64, 128 or 256");
  MOC_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0,
              "moc_paged_append_bf16: page must be a power of two from 16 to 256");
  MOC_REQUIRE(code == MOC_E4M3 || code == MOC_I8, "moc_paged_append_bf16: codes must be e4m3 or int8");
  MOC_REQUIRE(table_dtype == MOC_BF16 || table_dtype == MOC_F32, "moc_paged_append_bf16: cos, sin must be bf16 or f32");
  MOC_REQUIRE(tokens >= 0 && seqs >= 0 && q_heads >= 0 && kv_heads >= 1 && width >= 0 && pages >= 0 && angles >= 0 &&
                  tokens < (1 << 28) && seqs < (1 << 28) && q_heads + 2 * kv_heads <= 65536 && pages < (1LL << 31) &&
                  width < (1LL << 31) && angles < (1LL << 31),
              "moc_paged_append_bf16: bad shape");
  MOC_REQUIRE(cu != nullptr || tokens == seqs, "moc_paged_append_bf16: one token a sequence without cu");
  if (tokens == 0 || seqs == 0) return MOC_OK;
  MOC_REQUIRE((q || q_heads == 0) && k && v && cos && sin && k_codes && v_codes && k_scale && v_scale && (table || width == 0) && lens &&
                  (q_out || q_heads == 0),
              "moc_paged_append_bf16: null pointer");
  MOC_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(cos) && aligned16(sin) &&
                  aligned16(k_codes) && aligned16(v_codes) && (q_ld | q_lh | k_ld | k_lh | v_ld | v_lh | o_ld | o_lh) % 8 == 0,
              "moc_paged_append_bf16: rows must be 16-byte aligned");
  AppendArgs a;
  a.s = PagedSeqs{cu, lens, table, ld_table, static_cast<int>(seqs), static_cast<int>(tokens), static_cast<int>(width)};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_ld = q_ld; a.q_lh = q_lh; a.k_ld = k_ld; a.k_lh = k_lh; a.v_ld = v_ld; a.v_lh = v_lh;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.o_ld = o_ld; a.o_lh = o_lh;
  a.cos = cos; a.sin = sin;
  a.angles = static_cast<int>(angles);
  a.kc = static_cast<uint8_t*>(k_codes);
  a.vc = static_cast<uint8_t*>(v_codes);
  a.ks = k_scale; a.vs = v_scale;
  a.pages = static_cast<int>(pages);
  a.log_page = __builtin_ctzll(static_cast<unsigned long long>(page));
  a.q_heads = static_cast<int>(q_heads);
  a.kv_heads = static_cast<int>(kv_heads);
  // pages that n tokens of a sequence reach: at most (n - 1) / page + 2
  const int64_t units = cu == nullptr ? seqs : tokens / page + 2 * std::min(seqs, tokens);
  const int64_t blocks = (units * (q_heads + 2 * kv_heads) + 3) / 4;
  MOC_REQUIRE(blocks < (1LL << 31), "moc_paged_append_bf16: too many tokens and heads for one call");
  const dim3 grid(static_cast<unsigned>(blocks)), threads(256);
  hipStream_t st = as_stream(stream);
#define MOC_APPEND(D, I, F) paged_append_kernel<D, I, F><<<grid, threads, 0, st>>>(a)
#define MOC_APPEND_D(D)                                                   \
  do {                                                                    \
    if (code == MOC_I8) {                                                 \
      if (table_dtype == MOC_F32) MOC_APPEND(D, true, true);              \
      else MOC_APPEND(D, true, false);                                    \
    } else {                                                              \
      if (table_dtype == MOC_F32) MOC_APPEND(D, false, true);             \
      else MOC_APPEND(D, false, false);                                   \
    }                                                                     \
  } while (0)
  if (head_dim == 64) MOC_APPEND_D(64);
  else if (head_dim == 128) MOC_APPEND_D(128);
  else MOC_APPEND_D(256);
#undef MOC_APPEND_D
#undef MOC_APPEND
  return check_launch("paged_append_kernel");
}
