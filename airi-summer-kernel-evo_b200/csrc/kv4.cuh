// What the kernels of the 4-bit paged cache share: the layout of a page, the batch that a call
// works on, and the places of its tokens.
//
// A page holds page_size tokens of every kv head of one layer; the block of a head is
//   [K codes: page_size x D/2 B | K scales: page_size x D/16 B | V codes | V scales]
// with e2m1 codes (two to a byte, the even element in the low nibble) and one e4m3 scale for
// 16 consecutive elements: value = code * scale * (k_scale or v_scale), 4.5 bits an element.
// e2m1 x e4m3 has at most 6 significant bits and lies in [2^-10, 2688]: exact in f16.
//
// Token i of the n new tokens of sequence b sits at position lens[row] - n + i, row = rows[b].
// Whatever the device-side lists say, no kernel reads or writes out of bounds: a row, page or
// position outside of its range records B2F_DEV_BAD_ARGS in the device status word and the
// token (key) is left out.
#pragma once
#include "common.cuh"

namespace b2f {

struct Kv4Cache {
  uint8_t* storage;
  long long page_stride;
  int pages, kv_heads, head_dim, page_size;
  float k_scale, v_scale;
  const int* table;
  int table_rows, table_cols;
  long long table_ld;
  const int* lens;
  // derived
  int page_log2, block_bytes, codes_bytes, scales_bytes;  // of one part of one block
};

struct Kv4Batch {
  int seqs, tokens;
  const int* rows;
  const int* starts;
  int each;  // tokens of a sequence without starts
};

struct Kv4Seq {
  int row;    // table row, -1: not a row of the table
  int start;  // first token of the batch
  int n;      // new tokens
  int len;    // cached tokens, the new ones among them; at most what the table can hold
};

__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Cache& c, const Kv4Batch& bt, int b) {
  Kv4Seq s;
  s.row = bt.rows != nullptr ? bt.rows[b] : b;
  if (bt.starts != nullptr) {
    s.start = bt.starts[b];
    const int end = bt.starts[b + 1];
    if (s.start < 0 || end < s.start || end > bt.tokens) {
      record_error(kDevBadArgs);
      s.start = 0;
      s.n = 0;
    } else {
      s.n = end - s.start;
    }
  } else {
    s.start = b * bt.each;
    s.n = bt.each;
  }
  s.len = 0;
  if (s.row < 0 || s.row >= c.table_rows) {
    record_error(kDevBadArgs);
    s.row = -1;
  } else {
    s.len = c.lens[s.row];
    const long long room = (long long)c.table_cols << c.page_log2;
    if (s.len < 0 || s.len > room) {
      record_error(kDevBadArgs);
      s.len = s.len < 0 ? 0 : (int)room;
    }
  }
  return s;
}

// The sequence of packed token t, -1 for a row outside of all sequences.  All lanes of a warp ask
// for the same token; each round probes 32 places, so that 1024 sequences take two.
__device__ __forceinline__ int kv4_owner(const Kv4Batch& bt, int t) {
  if (bt.starts == nullptr) return t / bt.each;
  const int lane = threadIdx.x & 31;
  int lo = 0, n = bt.seqs;  // starts[lo] <= t < starts[lo + n], if t is in a sequence at all
  if (t < bt.starts[0] || t >= bt.starts[bt.seqs]) return -1;
  while (n > 1) {
    const int step = (n + 31) >> 5, at = lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < n && bt.starts[lo + at] <= t);
    const int k = below == 0 ? 0 : 31 - __clz(below);
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}

// Page and slot of packed token t (the same for all lanes of a warp); page -1 where it has none,
// -2 outside of all sequences.
__device__ __forceinline__ int kv4_place(const Kv4Cache& c, const Kv4Batch& bt, int t, int& slot) {
  slot = 0;
  Kv4Seq s;
  if (bt.starts != nullptr && bt.seqs < 32) {
    // every lane looks up one sequence, so that the lookups do not wait for the search
    const int lane = threadIdx.x & 31;
    const int start = lane <= bt.seqs ? bt.starts[lane] : 0x7fffffff;
    int row = lane < bt.seqs ? (bt.rows != nullptr ? bt.rows[lane] : lane) : -1;
    if (row >= c.table_rows) row = -1;
    const int len = row >= 0 ? c.lens[row] : 0;
    const unsigned below = __ballot_sync(0xffffffffu, start <= t);
    const int b = below == 0 ? -1 : 31 - __clz(below);
    if (b < 0 || b >= bt.seqs) return -2;
    const int end = __shfl_sync(0xffffffffu, start, b + 1);
    s.start = __shfl_sync(0xffffffffu, start, b);
    s.n = end - s.start;
    if (s.start < 0 || end > bt.tokens) s.start = s.n = 0;  // not a part of the batch: as kv4_seq has it
    s.row = __shfl_sync(0xffffffffu, row, b);
    s.len = __shfl_sync(0xffffffffu, len, b);
  } else {
    const int b = kv4_owner(bt, t);
    if (b < 0) return -2;
    s = kv4_seq(c, bt, b);
    if (s.row >= 0) s.len = c.lens[s.row];
  }
  const int pos = s.len - s.n + (t - s.start);
  if (s.row < 0 || pos < 0 || t < s.start || t - s.start >= s.n ||
      s.len > (long long)c.table_cols << c.page_log2) {
    record_error(kDevBadArgs);
    return -1;
  }
  const int page = c.table[(long long)s.row * c.table_ld + (pos >> c.page_log2)];
  if (page < 0 || page >= c.pages) {
    record_error(kDevBadArgs);
    return -1;
  }
  slot = pos & (c.page_size - 1);
  return page;
}

// Host: argument checks shared by the entry points (nullptr: fine).
const char* kv4_check_cache(const b2f_kv4_cache& c, Kv4Cache* out);
const char* kv4_check_batch(const b2f_kv4_cache& c, const b2f_kv4_batch& b, Kv4Batch* out);

}  // namespace b2f
