// What the kernels over a paged 8-bit key/value cache share (gfx950).
//
// The cache: codes [pages, kv_heads, page, head_dim] of keys and of values (one
// byte each: OCP e4m3, or int8) and one f32 scale for each page and head; a
// value is code * scale.  A sequence's position p lies in place p % page of page
// table[sequence][p / page].  page is a power of two from 16 to 256, so the 16
// positions of an MFMA tile never cross a page.
#pragma once

#include "common.h"

namespace moc {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// Sequences of a ragged batch: sequence b's new tokens are rows cu[b] .. cu[b +
// 1] - 1 of q (cu null: row b alone), the last of them at position lens[b] - 1.
struct PagedSeqs {
  const int32_t* cu;
  const int32_t* lens;
  const int32_t* table;  // [seqs, width]
  int64_t ld_table;
  int seqs, tokens, width;
};

struct SeqSpan {
  int seq;       // -1: none
  int row0, n;   // its rows of q
  int unit;      // which of its units
  int64_t len;   // tokens in the cache, new ones among them
};

// Sequence `seq`'s rows, kept inside [0, tokens] whatever cu holds.
__device__ __forceinline__ void seq_rows(const PagedSeqs& s, int seq, int& row0, int& n) {
  if (s.cu == nullptr) {
    row0 = min(seq, s.tokens);
    n = row0 < s.tokens ? 1 : 0;
    return;
  }
  row0 = min(max(s.cu[seq], 0), s.tokens);
  n = max(min(s.cu[seq + 1], s.tokens) - row0, 0);
}

// The sequence that holds the unit'th of all sequences' units, units_of(row0, n,
// len) each, by a whole wave: 64 sequences at a time, one a lane.
template <typename F>
__device__ __forceinline__ SeqSpan find_unit(const PagedSeqs& s, int unit, F units_of) {
  const int lane = threadIdx.x & 63;
  SeqSpan out;
  out.seq = -1;
  out.row0 = out.n = out.unit = 0;
  out.len = 0;
  int before = 0;
  for (int b0 = 0; b0 < s.seqs; b0 += 64) {
    const int b = b0 + lane;
    int row0 = 0, n = 0, len = 0, units = 0;
    if (b < s.seqs) {
      seq_rows(s, b, row0, n);
      len = s.lens[b];
      units = n > 0 ? units_of(n, static_cast<int64_t>(len)) : 0;
    }
    const int upto = static_cast<int>(wave_inclusive_scan(static_cast<uint32_t>(units)));
    const int total = __builtin_amdgcn_readlane(upto, 63);
    if (unit < before + total) {
      const uint64_t past = __ballot(before + upto > unit);
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      out.seq = b0 + at;
      out.row0 = __builtin_amdgcn_readlane(row0, at);
      out.n = __builtin_amdgcn_readlane(n, at);
      out.len = __builtin_amdgcn_readlane(len, at);
      out.unit = unit - (before + __builtin_amdgcn_readlane(upto - units, at));
      return out;
    }
    before += total;
  }
  return out;
}

}  // namespace moc
