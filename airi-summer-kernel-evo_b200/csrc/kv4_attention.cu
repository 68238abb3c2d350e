// Attention of new tokens over the 4-bit paged cache (C ABI: b2f_kv4_attention; the layout of
// the cache stands in kv4.cuh).
//
//   out[t, h] = sum_j softmax_j(q_h . k_j * sm_scale) v_j [* sigmoid(gate)] / ctx_scale
// over the keys j <= position of t (causal) or all cached keys of its sequence.
//
// Bound: a step of one token per sequence reads 9/8 D bytes per key and kv head and does
// 4 D * (heads / kv_heads) operations on them: HBM, if the codes become matrix operands cheaply
// enough.  At the copy rate (6.5 TB/s) an SM receives one key (D = 128, 144 B) in 6.2 clocks; in
// these a scheduler issues about 4.5 instructions of it (575 a warp for 32 keys), of which the
// conversions (cvt.rn.f16x2.e2m1x2) and the scalings (multiplications of f16 pairs) take 2 clocks
// each and the matrix instructions another 2, on three different pipes.
//
// Measured (device time in a replayed graph, bytes of the cache over it), head_dim 128, 8 kv heads of
// 4 query heads, calls without starts:
//   2 sequences of 131072 keys             64 us   4.7 TB/s   issue slots 55 %, DRAM 54 % busy
//   64 sequences of up to 8191, 273K keys  74 us   4.2 TB/s
//   1 sequence of 197                       9.2 us (launch, one unit's latency; no join, for the table
//                                          holds 208 tokens; 11.1 with a table of 8192)
//   head_dim 256, 4 kv heads, gate, e4m3; 16 sequences of up to 4000, 40K keys
//                                          26.5 us  1.7 TB/s
// About 10 us of each are ends, by the call on 197 keys in a wide table: finding the run of units, the
// first pages' latency, cold instructions, and the join.  Without these the long case has 5.6 TB/s
// and the batch 4.9, and neither the issue slots nor DRAM are full.
//
// How the work is laid out
//  - Keys on the rows of the matrix instruction (m16n8k16, f16 in, f32 out): S^T = K Q^T and
//    O^T = V^T P^T, up to 8 query rows (query heads of the kv head x new tokens) a column
//    tile, so that the 16-row operand that has to be made from codes is never padding.
//  - The sums over d and over keys may run in any order, which lets every thread use codes
//    where they lie: thread (r, c) = (lane / 4, lane % 4) reads 16 consecutive bytes of the K
//    row of its key, whose byte pairs are the k slots (2c, 2c+1), (2c+8, 2c+9) of eight
//    steps; q is read in the same order.  For V it reads the D / 8 elements r D / 8 .. of the
//    keys c, c + 4, c + 8, c + 12 of 16, merges the codes of two keys nibble by nibble, and
//    has the pairs along the keys that the instruction wants.  Slot s of 16 is key
//    (s & 7) / 2 + (s & 1) * 4 + (s & 8): the K rows are taken in that order.
//  - e2m1 x e4m3 is exact in f16.  A query row is brought to [2^14, 2^15) by a power of two:
//    bf16 and f16 queries lose nothing that is above 2^-39 of the row's largest.  P is held
//    in f16, at most 2^15 and scaled so that the row's largest is at least 2^7: a rounding of
//    2^-11, and of 2^-31 of the largest for the smallest.  Sums, maxima and O are f32.
//  - Each of four warps walks over 32 keys at a time (16 at D = 256, for its registers) with a
//    maximum, a sum and an O of its own (the maximum moves only when a score passes it by 2^8,
//    so most steps need no exchange); the four are joined when a piece of work ends.
//  - A fifth warp keeps a ring of units filled: one bulk copy a page, for the block of a kv head
//    is one piece of memory (with four copies a page, of K, V and their scales, the copies were
//    the bound), and lays the queries of the next item out as matrix operands.
//  - What a row may not see (keys behind the end or its position, pages that are not there, NaN in
//    such places) is taken out of the ring by a lane a key, in a loop of its own, before it is
//    used: the loop over all other units has no test for it (batch 76 -> 74 us, long 67 -> 64; its
//    instructions stay in the first cache).
//  - The keys of all (sequence, kv head, row tile) items are cut into units of 128 keys, and
//    every CTA takes an equal run of consecutive units, whatever the lengths: at most its
//    first and its last item are shared with other CTAs.  Their partial (O, max, sum) go to a
//    workspace and a second kernel joins them in order of the keys: same bits in every run.
#include <cfloat>

#include "kv4_attention.cuh"

namespace b2f {
namespace {

constexpr int kWarps = 4;                 // that work on keys; one more fetches them
constexpr int kWork = 32 * kWarps;
constexpr int kThreads = kWork + 32;


__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with zeros for d.
__device__ __forceinline__ void mma16816_from0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Barrier of `threads` threads; whether `mine` holds for all of them.
__device__ __forceinline__ bool named_bar_all(int id, int threads, bool mine) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(id), "r"(threads), "r"((uint32_t)mine)
      : "memory");
  return all != 0;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// kChunk: keys of a step of a warp; kUnit: of a unit of work, and of a stage of the ring.
template <int D, int NT, int STAGES>
struct Layout {
  static constexpr int R = 8 * NT;
  static constexpr int kChunk = D == 256 ? 16 : 32, kUnit = kChunk * kWarps;
  static constexpr int kStage = kUnit * D / 8 * 9;       // the blocks of a unit's pages, one after the other
  static constexpr int kRow = 64 + 4;                    // floats of a row of the join: 64 elements at a time
  static constexpr int kRing = STAGES * kStage;
  static constexpr int kJoin = kWarps * R * kRow * 4;
  static constexpr int kBytes = kRing + kJoin;
};

// What the fetching warp tells the others of the piece of an item that comes next.
struct Piece {
  int first, take;     // units [first, first + take) of the item; take 0: no more pieces
  int keys;            // of the item
  int start, n, seen;  // first token, tokens, and keys that are older than the first token
  int h, row0;         // kv head, first row of the tile
  int whole;           // the piece is the whole item
};

template <int D, int NT, int STAGES, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) kv4_attention_kernel(const Kv4AttnParams p) {
  using L = Layout<D, NT, STAGES>;
  constexpr int R = L::R, U = L::kUnit, kUnit = U, kChunk = L::kChunk;
  constexpr int G = kChunk / 16;            // sixteens of keys of a step
  constexpr int kTiles = D / 16;            // m16 tiles of O^T
  constexpr int kRuns = D == 256 ? 2 : 1;   // runs of neighbouring K codes of a thread and key
  constexpr int kWordsK = D / 32 / kRuns;   // 32-bit words of a run: two steps each
  constexpr int kWordsV = D / 64;           // words of V codes of a thread and key
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Scan sc;
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES], q_full[2], q_empty[2];
  __shared__ unsigned stage_ok[STAGES];  // bit i: page i of the unit is there
  __shared__ int aborted;                // a wait ran out: no more work, no more copies
  __shared__ Piece pieces[2];
  __shared__ uint4 q_frag[2][NT * D / 32][32];  // B operands of two steps of a lane
  __shared__ float q_drop[2][R];
  __shared__ float join_ms[kWarps][R][2];

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  float* join = reinterpret_cast<float*>(smem + L::kRing);
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], kWarps);
    }
    aborted = 0;
    fence_mbarrier_init();
  }
  pdl_wait();
  pdl_trigger();

  long long u0, u1;
  bool blank;
  const Runs runs = find_run<R, U, kThreads>(p, sc, u0, u1, blank);
  // No item yet; stored by the lane that stores the descriptor of one (below), for nothing else
  // orders the two.
  if (p.split && threadIdx.x == kWork) p.shared[blockIdx.x].more = 0;
  if (blank) blank_rows<D, R, kThreads>(p);
  if (u0 >= u1) return;

  int stage = 0, buf = 0;
  uint32_t phase = 0, q_phase = 0;
  const int log2p = p.c.page_log2;

  if (warp == kWarps) {
    // ---- the fetching warp: a lane for each page of a unit; the block of a head is one piece
    Item it;
    int first = 0;
    if (p.split) {
      first = find_item<R, U>(p, sc.b[0], u0 - sc.at[0], it);
    } else if (find_item<R, U>(p, sc.b[0], runs.begin(blockIdx.x) - sc.at[0], it) > 0) {
      next_item<R, U>(p, it);
    }
    long long left = u1 - u0;
    const bool copies = lane < (kUnit >> log2p);
    const uint64_t policy = policy_evict_normal();
    int fetched = 0, told = 0;
    bool ok = true;
    while (left > 0) {
      const int take = (int)min((long long)(it.units - first), left);
      const uint8_t* const block = p.c.storage + (long long)it.h * p.c.block_bytes;
      const int* const pages = p.c.table + (long long)it.s.row * p.c.table_ld;
      auto page_at = [&](int unit) {
        const int key = unit * kUnit + (lane << log2p);
        return copies && unit < first + take && key < it.keys ? pages[key >> log2p] : -1;
      };
      auto fetch = [&](int u, int page) {
        if (fetched >= STAGES)
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, kDevTimeoutProducer, &aborted));
        if (!ok) return;
        const bool there = (unsigned)page < (unsigned)p.c.pages;
        if (!there && copies && u * kUnit + (lane << log2p) < it.keys) record_error(kDevBadArgs);
        const unsigned good = __ballot_sync(0xffffffffu, there);
        if (lane == 0) {
          stage_ok[stage] = good;
          mbar_arrive_expect_tx(&full[stage], (uint32_t)__popc(good) * (uint32_t)p.c.block_bytes);
        }
        __syncwarp();
        if (there)
          bulk_load(smem + stage * L::kStage + lane * p.c.block_bytes, block + page * p.c.page_stride,
                    (uint32_t)p.c.block_bytes, &full[stage], policy);
        ++fetched;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      };
      int page = page_at(first);
      // the queries of the tile: thread (r, c) takes the elements of row r in the order of its codes
      float x[NT][kRuns][4 * kWordsK * 2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        int head;
        const int t = row_token(p, it.rt * R + nt * 8 + r, it.h, it.s.start, it.s.n, head);
        const long long at = (long long)t * p.q_ld + (long long)head * D + c * (8 * kWordsK);
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
#pragma unroll
          for (int k = 0; k < 8 * kWordsK; k += 4) {
            float* y = x[nt][i] + k;
            const long long e = at + i * 128 + k;
            if (t < 0) {
              y[0] = y[1] = y[2] = y[3] = 0.f;
            } else if (p.q_dtype == kBF16) {
              load4<kBF16>(p.q, e, y);
            } else if (p.q_dtype == kF16) {
              load4<kF16>(p.q, e, y);
            } else {
              load4<kE4M3>(p.q, e, y);
            }
          }
      }
      int next = page_at(first + 1);
      fetch(first, page);
      if (told >= 2)
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&q_empty[buf], q_phase ^ 1, kDevTimeoutProducer, &aborted));
      if (!ok) break;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
#pragma unroll
          for (int k = 0; k < 8 * kWordsK; ++k) top = fmaxf(top, fabsf(x[nt][i][k]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(14 - exponent of top), and its inverse; 1 for a row of zeros or with an infinity
        const int ex = (__float_as_int(top) >> 23) & 0xff;
        const int up = ex == 0 || ex == 255 ? 0 : min(max(127 + 14 - ex, -120), 120);
        const float lift = __int_as_float((127 + up) << 23), drop = __int_as_float((127 - up) << 23);
        if (c == 0) q_drop[buf][nt * 8 + r] = drop;
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
#pragma unroll
          for (int k = 0; k < kWordsK; ++k) {
            const float* y = x[nt][i] + 8 * k;
            q_frag[buf][(nt * kRuns + i) * kWordsK + k][lane] =
                make_uint4(pack_f16x2(y[0] * lift, y[1] * lift), pack_f16x2(y[2] * lift, y[3] * lift),
                           pack_f16x2(y[4] * lift, y[5] * lift), pack_f16x2(y[6] * lift, y[7] * lift));
          }
      }
      if (lane == 0) {
        const bool to_end = first + take == it.units;
        pieces[buf] = Piece{first, take, it.keys, it.s.start, it.s.n, it.s.len - it.s.n, it.h, it.rt * R, first == 0 && to_end};
        if (first == 0 && !to_end) {
          const int last = runs.of(u1 - left + it.units - 1);  // the CTA with the item's last unit
          p.shared[blockIdx.x] = Shared{last - (int)blockIdx.x, it.s.start, it.s.n, it.h * p.group, it.rt * R};
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[buf]);
      ++told;
      if (++buf == 2) {
        buf = 0;
        q_phase ^= 1;
      }
      for (int u = first + 1; u < first + take; ++u) {
        page = next;
        next = page_at(u + 1);
        fetch(u, page);
      }
      left -= take;
      if (left > 0) {
        next_item<R, U>(p, it);
        first = 0;
      }
    }
    if (ok) {
      if (told >= 2) mbar_wait(&q_empty[buf], q_phase ^ 1, kDevTimeoutProducer, &aborted);
      if (lane == 0) {
        pieces[buf].take = 0;
        mbar_arrive(&q_full[buf]);
      }
    }
    // no copy is left in flight when the CTA ends, whoever has given up
    for (int s = 0; s < min(fetched, STAGES); ++s) {
      if (--stage < 0) {
        stage = STAGES - 1;
        phase ^= 1;
      }
      mbar_wait(&full[stage], phase, kDevTimeoutDrain, nullptr);
    }
    return;
  }

  // Where the warp's codes and scales lie in a stage (of K; those of V are v_part behind), and how
  // far a second 16 of its keys are from the first; the bits of their pages in stage_ok.
  const int page0 = (warp * kChunk) >> log2p, slot0 = (warp * kChunk) & (p.c.page_size - 1);
  const int codes_at = page0 * p.c.block_bytes + slot0 * (D / 2);
  const int scales_at = page0 * p.c.block_bytes + p.c.codes_bytes + slot0 * (D / 16);
  const int v_part = p.c.codes_bytes + p.c.scales_bytes;
  const int codes_2nd = log2p == 4 ? p.c.block_bytes : 16 * (D / 2);
  const int scales_2nd = log2p == 4 ? p.c.block_bytes : 16 * (D / 16);
  const int page1 = page0 + (log2p == 4 && G == 2 ? 1 : 0);
  const unsigned mine = 1u << page0 | 1u << page1;

  for (;;) {
    // The barrier lets the four warps agree (a warp that gave up must not leave the others at the
    // next one), and the join of the piece before has been read when it is passed.
    if (!named_bar_all(1, kWork, mbar_wait(&q_full[buf], q_phase, kDevTimeoutMma, &aborted))) return;
    bool alive = true;
    const Piece it = pieces[buf];
    if (it.take == 0) return;
    float mul[NT][2];
    int limit[NT][2];  // keys that the column sees
    int lowest = 0x7fffffff;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mul[nt][j] = fmaxf(q_drop[buf][nt * 8 + 2 * c + j] * p.scale_log2, FLT_MIN);  // -infinity * 0 is none
        const int i = by_group(it.row0 + nt * 8 + 2 * c + j, p.group_inv);
        limit[nt][j] = p.causal ? min(it.seen + i + 1, it.keys) : it.keys;
        if (i < it.n) lowest = min(lowest, limit[nt][j]);
      }
    lowest = __reduce_min_sync(0xffffffffu, lowest);

    // P = 2^(score - base); base is 7 below the largest score seen when it was last moved
    float base[NT][2], sum[NT][2], o[kTiles][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        base[nt][j] = -FLT_MAX;  // no score yet: any is far above it, and -infinity stays -infinity
        sum[nt][j] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[t][nt][j] = 0.f;
    }

    for (int u = it.first; u < it.first + it.take; ++u) {
      const int key0 = u * kUnit + warp * kChunk;
      alive = alive && __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, kDevTimeoutMma, &aborted));
      if (alive && key0 < it.keys) {
        const uint8_t* kc = smem + stage * L::kStage + codes_at;
        const uint8_t* ks = smem + stage * L::kStage + scales_at;
        const unsigned okay = stage_ok[stage];
        const bool edge = key0 + kChunk > lowest || (okay & mine) != mine;
        // ---- S^T: 16 keys x R rows, G times
        float s[G][NT][4];
        const int kr = (r >> 1) + (r & 1) * 4;  // key of slot r (of the first 16); slot r + 8: kr + 8
#pragma unroll
        for (int i = 0; i < kRuns; ++i) {
          uint32_t w[2 * G][kWordsK], m[2 * G];  // codes of the keys kr + 8 k, scales of two groups as f16
#pragma unroll
          for (int k = 0; k < 2 * G; ++k) {
            const int key = kr + 8 * (k & 1);
            const uint8_t* codes = kc + (k >= 2 ? codes_2nd : 0);
            const uint8_t* scales = ks + (k >= 2 ? scales_2nd : 0);
            if (D == 64) {
              const uint2 a = *reinterpret_cast<const uint2*>(codes + key * 32 + c * 8);
              w[k][0] = a.x; w[k][1] = a.y;
              m[k] = e4m3x2_to_f16x2(scales[key * 4 + c]);
            } else {
              const uint4 a = *reinterpret_cast<const uint4*>(codes + key * (D / 2) + i * 64 + c * 16);
              w[k][0] = a.x; w[k][1] = a.y; w[k][kWordsK - 2] = a.z; w[k][kWordsK - 1] = a.w;
              m[k] = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(scales + key * (D / 16) + 8 * i + 2 * c));
            }
          }
#pragma unroll
          for (int x = 0; x < kWordsK; ++x) {  // a word is two steps; two words share a scale
            uint4 q[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) q[nt] = q_frag[buf][(nt * kRuns + i) * kWordsK + x][lane];
#pragma unroll
            for (int g = 0; g < G; ++g) {
              uint32_t f0[4], f1[4];
              e2m1x8_to_f16x2(w[2 * g][x], f0);
              e2m1x8_to_f16x2(w[2 * g + 1][x], f1);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                f0[j] = hmul2_by(f0[j], m[2 * g], x / 2);
                f1[j] = hmul2_by(f1[j], m[2 * g + 1], x / 2);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (i == 0 && x == 0) mma16816_from0(s[g][nt], f0[0], f1[0], f0[1], f1[1], q[nt].x, q[nt].y);
                else mma16816(s[g][nt], f0[0], f1[0], f0[1], f1[1], q[nt].x, q[nt].y);
                mma16816(s[g][nt], f0[2], f1[2], f0[3], f1[3], q[nt].z, q[nt].w);
              }
            }
          }
        }
        // ---- scores to P
        float x[G][NT][4];
        if (__builtin_expect(edge, 0)) {
          // Keys that a row may not see: score -infinity.  Their values must not reach it either:
          // 0 * NaN would.  NaN scales of values that not all rows see are set to 0 in the ring,
          // and a row that does see one gets it through its score.  A lane looks at one key.
          const uint32_t gone = (okay >> page0 & 1 ? 0u : 0xffffu) | (okay >> page1 & 1 ? 0u : 0xffff0000u);
          bool nan = false;
          if (lane < kChunk) {
            uint32_t* row = reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(
                ks + v_part + (lane >= 16 ? scales_2nd : 0) + (lane & 15) * (D / 16)));
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
              const uint32_t v = row[i], is = ((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bytes 0x7f, 0xff
              if (is != 0 && (key0 + lane >= lowest || (gone >> lane & 1))) {
                row[i] = v & ~((is >> 7) * 0xffu);
                nan = true;
              }
            }
          }
          fence_async_shared();  // the next copy into the stage comes after these stores
          const uint32_t nans = __ballot_sync(0xffffffffu, nan);
          __syncwarp();  // the scales are read by other lanes below
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int key = g * 16 + kr + (j >> 1) * 8;
                if (nans >> key & 1) s[g][nt][j] = NAN;
                if (key0 + key >= limit[nt][j & 1] || (gone >> key & 1)) s[g][nt][j] = -INFINITY;
              }
        }
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              x[g][nt][j] = fmaf(s[g][nt][j], mul[nt][0], -base[nt][0]);
              x[g][nt][j + 1] = fmaf(s[g][nt][j + 1], mul[nt][1], -base[nt][1]);
              top = fmax3(top, x[g][nt][j], x[g][nt][j + 1]);  // a first score is infinitely far above the base
            }
        if (__builtin_expect(__any_sync(0xffffffffu, top > kSlack + kLift), 0)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float m = fmaxf(s[0][nt][j], s[0][nt][j + 2]);
              if (G == 2) m = fmax3(m, s[G - 1][nt][j], s[G - 1][nt][j + 2]);
              m *= mul[nt][j];
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              m = fmaxf(m - kLift, base[nt][j]);
              const float f = m == base[nt][j] ? 1.f : ex2(base[nt][j] - m);
              base[nt][j] = m;
              sum[nt][j] *= f;
#pragma unroll
              for (int t = 0; t < kTiles; ++t) {
                o[t][nt][j] *= f;
                o[t][nt][j + 2] *= f;
              }
#pragma unroll
              for (int g = 0; g < G; ++g) {
                x[g][nt][j] = fmaf(s[g][nt][j], mul[nt][j], -m);
                x[g][nt][j + 2] = fmaf(s[g][nt][j + 2], mul[nt][j], -m);
              }
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[g][nt][j] = ex2(x[g][nt][j]);
              sum[nt][j & 1] += x[g][nt][j];
            }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int g = 0; g < G; ++g) {
          uint32_t pf[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            pf[nt][0] = transpose8x8(pack_f16x2(x[g][nt][0], x[g][nt][1]));
            pf[nt][1] = transpose8x8(pack_f16x2(x[g][nt][2], x[g][nt][3]));
          }
          // codes and scales of keys c, c + 4, c + 8, c + 12 of the 16
          const uint8_t* vk = kc + v_part + (g ? codes_2nd : 0) + c * (D / 2) + r * (D / 16);
          const uint8_t* vsk = ks + v_part + (g ? scales_2nd : 0) + c * (D / 16) + (r * (D / 8)) / 16;
          uint32_t v[4][kWordsV], vm[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (D == 64) {
              v[i][0] = *reinterpret_cast<const uint32_t*>(vk + i * 4 * (D / 2));
              vm[i] = vsk[i * 4 * (D / 16)];
            } else if (D == 128) {
              const uint2 a = *reinterpret_cast<const uint2*>(vk + i * 4 * (D / 2));
              v[i][0] = a.x;
              v[i][kWordsV - 1] = a.y;
              vm[i] = vsk[i * 4 * (D / 16)];
            } else {
              const uint4 a = *reinterpret_cast<const uint4*>(vk + i * 4 * (D / 2));
              v[i][0] = a.x;
              v[i][kWordsV / 4] = a.y;
              v[i][kWordsV / 2] = a.z;
              v[i][kWordsV - 1] = a.w;
              vm[i] = *reinterpret_cast<const uint16_t*>(vsk + i * 4 * (D / 16));
            }
          }
          uint32_t vm01[D == 256 ? 2 : 1], vm23[D == 256 ? 2 : 1];  // scales of two keys as f16 pairs
          if (D == 256) {
            vm01[0] = e4m3x2_to_f16x2(__byte_perm(vm[0], vm[1], 0x0040));
            vm23[0] = e4m3x2_to_f16x2(__byte_perm(vm[2], vm[3], 0x0040));
            vm01[D == 256] = e4m3x2_to_f16x2(__byte_perm(vm[0], vm[1], 0x0051));
            vm23[D == 256] = e4m3x2_to_f16x2(__byte_perm(vm[2], vm[3], 0x0051));
          } else {
            vm01[0] = e4m3x2_to_f16x2(vm[0] + vm[1] * 256);
            vm23[0] = e4m3x2_to_f16x2(vm[2] + vm[3] * 256);
          }
#pragma unroll
          for (int w = 0; w < kWordsV; ++w) {  // a word: four tiles
            const uint32_t m01 = D == 256 ? vm01[w / 2] : vm01[0], m23 = D == 256 ? vm23[w / 2] : vm23[0];
            uint32_t lo01[4], hi01[4], lo23[4], hi23[4];
            e2m1x8_to_f16x2((v[0][w] & 0x0f0f0f0fu) | ((v[1][w] << 4) & 0xf0f0f0f0u), lo01);
            e2m1x8_to_f16x2(((v[0][w] >> 4) & 0x0f0f0f0fu) | (v[1][w] & 0xf0f0f0f0u), hi01);
            e2m1x8_to_f16x2((v[2][w] & 0x0f0f0f0fu) | ((v[3][w] << 4) & 0xf0f0f0f0u), lo23);
            e2m1x8_to_f16x2(((v[2][w] >> 4) & 0x0f0f0f0fu) | (v[3][w] & 0xf0f0f0f0u), hi23);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a0 = hmul2(lo01[i], m01), a1 = hmul2(hi01[i], m01);
              const uint32_t a2 = hmul2(lo23[i], m23), a3 = hmul2(hi23[i], m23);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816(o[4 * w + i][nt], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
            }
          }
        }
      }
      __syncwarp();  // the stage has been read by all lanes
      if (lane == 0) mbar_arrive(&empty[stage]);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    // the queries and the piece have been read
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_empty[buf]);
    if (++buf == 2) {
      buf = 0;
      q_phase ^= 1;
    }

    // ---- the piece is done: join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = sum[nt][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int row = nt * 8 + 2 * c + j;
        if (r == 0) {
          join_ms[warp][row][0] = base[nt][j];
          join_ms[warp][row][1] = l;
        }
        sum[nt][j] = l;
      }
    const int slot = 2 * blockIdx.x + (it.first == 0 ? 1 : 0);
    float* part_o = p.partial + (long long)slot * R * D;
    float* part_ms = p.partial + 2ll * p.ctas * R * D + (long long)slot * R * 2;
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {  // 8 of the D / 8 elements of a thread at a time
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* to = join + (warp * R + nt * 8 + 2 * c + j) * L::kRow + r * 8;
#pragma unroll
          for (int t = 0; t < 4; t += 2)
            *reinterpret_cast<float4*>(to + 2 * t) = make_float4(o[4 * h + t][nt][j], o[4 * h + t][nt][j + 2],
                                                                 o[4 * h + t + 1][nt][j], o[4 * h + t + 1][nt][j + 2]);
        }
      named_bar_sync(1, kWork);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int row = i * 8 + threadIdx.x / 16, e = threadIdx.x % 16 * 4;
        const int d0 = (e >> 3) * (D / 8) + 8 * h + (e & 7);
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, join_ms[w][row][0]);
        float l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float mw = join_ms[w][row][0], lw = join_ms[w][row][1];
          const float f = mw == m ? 1.f : ex2(mw - m);  // a warp without a key: 0, or 1 of nothing
          const float4 y = *reinterpret_cast<const float4*>(join + (w * R + row) * L::kRow + e);
          l += lw * f;
          acc[0] += y.x * f; acc[1] += y.y * f; acc[2] += y.z * f; acc[3] += y.w * f;
        }
        if (it.whole) {
          int head;
          const int t = row_token(p, it.row0 + row, it.h, it.start, it.n, head);
          if (t >= 0) {
            finish_row<4>(p, t, head, d0, acc, l);
            if (d0 == 0) finish_lse(p, t, head, m, l);
          }
        } else {
          *reinterpret_cast<float4*>(part_o + row * D + d0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
          if (d0 == 0) {
            part_ms[2 * row] = m;
            part_ms[2 * row + 1] = l;
          }
        }
      }
      if (h + 1 < D / 64) named_bar_sync(1, kWork);
    }
  }
}

constexpr int kMaxPerSm = 4;

int tile_rows(int head_dim, long long rows) { return head_dim == 256 || rows <= 8 ? 8 : 16; }

template <int D, int NT, int STAGES, int CTAS>
int launch_attention(Kv4AttnParams& p, int sms, cudaStream_t s) {
  using L = Layout<D, NT, STAGES>;
  static_assert(CTAS <= kMaxPerSm && CTAS * (L::kBytes + NT * D * 32 + 2048) <= 227 * 1024, "CTAS CTAs fit on an SM");
  static FuncAttrOnce once;
  p.ctas = sms * CTAS;
  p.shared = reinterpret_cast<Shared*>(p.partial + 2ll * p.ctas * L::R * (D + 2));
  // Where no sequence can have more than two units, items are not cut: a CTA is done with one
  // before the pieces of several could be joined, and a launch is saved.  8 kv heads, head_dim
  // 128, whole against cut: 128 keys 8.1 us against 11.4, 256 keys 9.3 against 11.1, 512 keys 11.4
  // against 11.2, 16 sequences of 512 14.1 against 13.3.
  p.split = (long long)p.c.table_cols * p.c.page_size > 2 * L::kUnit;
  B2F_CUDA_TRY(once.max_smem(kv4_attention_kernel<D, NT, STAGES, CTAS>, L::kBytes));
  B2F_CUDA_TRY(launch_pdl(kv4_attention_kernel<D, NT, STAGES, CTAS>, dim3((unsigned)p.ctas), dim3(kThreads), L::kBytes, s, p));
  if (p.split)
    B2F_CUDA_TRY(launch_pdl(kv4_attention_join_kernel<D, L::R>, dim3((unsigned)p.ctas, L::R), dim3(kJoinThreads), 0, s, p));
  return B2F_OK;
}

}  // namespace
}  // namespace b2f

extern "C" {

void b2f_kv4_attn_args_init(b2f_kv4_attn_args* a) {
  if (a == nullptr) return;
  *a = b2f_kv4_attn_args{};
  a->causal = 1;
  a->q_dtype = a->out_dtype = B2F_DTYPE_BF16;
  a->gate_dtype = B2F_DTYPE_E4M3;
  a->q_scale = a->gate_scale = a->ctx_scale = 1.0f;
  a->cache.k_scale = a->cache.v_scale = 1.0f;
}

// Query rows of a kv head that a sequence brings, on average: what chooses between the kernels.
static long long rows_of_a_sequence(const b2f_kv4_attn_args* a) {
  if (a->batch.seqs <= 0 || a->batch.tokens <= 0 || a->cache.kv_heads <= 0) return 0;
  return (long long)a->batch.tokens * (a->heads / a->cache.kv_heads) / a->batch.seqs;
}

static long long attention_workspace(const b2f_kv4_attn_args* a, int sms) {
  if (sms <= 0) return -1;
  const int d = a->cache.head_dim;
  if (b2f::kv4_tiles_fit(rows_of_a_sequence(a))) return b2f::kv4_tiles_workspace(d, sms);
  const long long rows = d == 256 ? 8 : 16, ctas = (long long)sms * b2f::kMaxPerSm;
  return ctas * (2ll * rows * (d + 2) * 4 + (long long)sizeof(b2f::Shared));
}

long long b2f_kv4_attention_workspace_bytes(const b2f_kv4_attn_args* a) {
  return a == nullptr ? -1 : attention_workspace(a, b2f::sm_count());
}

int b2f_kv4_attention(const b2f_kv4_attn_args* a, b2f_stream_t stream) {
  using namespace b2f;
  if (a == nullptr) return fail(B2F_ERR_ARG, "kv4_attention: null args");
  Kv4AttnParams p = {};
  const char* e = kv4_check_cache(a->cache, &p.c);
  if (e == nullptr) e = kv4_check_batch(a->cache, a->batch, &p.b);
  if (e != nullptr) return fail(B2F_ERR_ARG, std::string("kv4_attention: ") + e);
  const int d = a->cache.head_dim, hk = a->cache.kv_heads;
  if (a->heads <= 0 || a->heads % hk) return fail(B2F_ERR_ARG, "kv4_attention: heads must be a multiple of kv_heads");
  if (a->heads / hk > 1024) return fail(B2F_ERR_ARG, "kv4_attention: more than 1024 query heads a kv head");
  if (a->batch.tokens > (1 << 23) || (long long)a->batch.tokens * a->heads > 0x3fffffffll) return fail(B2F_ERR_ARG, "kv4_attention: too many rows");
  if (a->q == nullptr || a->out == nullptr) return fail(B2F_ERR_ARG, "kv4_attention: null tensor");
  for (int dt : {a->q_dtype, a->out_dtype})
    if (dt != B2F_DTYPE_BF16 && dt != B2F_DTYPE_F16 && dt != B2F_DTYPE_E4M3)
      return fail(B2F_ERR_ARG, "kv4_attention: q and out must be bf16, f16 or e4m3");
  const int qs = a->q_dtype == B2F_DTYPE_E4M3 ? 1 : 2, os = a->out_dtype == B2F_DTYPE_E4M3 ? 1 : 2;
  const long long cols = (long long)a->heads * d;
  if (a->q_ld < cols || a->out_ld < cols || (a->q_ld * qs) % 16 || (a->out_ld * os) % 16 ||
      ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 15))
    return fail(B2F_ERR_ARG, "kv4_attention: q and out need 16-byte aligned rows of heads * head_dim elements");
  if (a->gate != nullptr) {
    if (a->gate_dtype != B2F_DTYPE_E4M3 && a->gate_dtype != B2F_DTYPE_BF16)
      return fail(B2F_ERR_ARG, "kv4_attention: gate must be e4m3 or bf16");
    if (a->gate_head_stride < d || a->gate_ld < (long long)(a->heads - 1) * a->gate_head_stride + d)
      return fail(B2F_ERR_ARG, "kv4_attention: gate row pitch or head stride too small");
    if (a->gate_dtype == B2F_DTYPE_BF16 && (reinterpret_cast<uintptr_t>(a->gate) & 1))
      return fail(B2F_ERR_ARG, "kv4_attention: misaligned gate");
  }
  if (!(a->q_scale > 0.f) || !std::isfinite(a->q_scale)) return fail(B2F_ERR_ARG, "kv4_attention: q_scale must be > 0");
  if (!std::isfinite(a->sm_scale)) return fail(B2F_ERR_ARG, "kv4_attention: sm_scale must be finite");
  const float sm = a->sm_scale > 0.f ? a->sm_scale : 1.0f / std::sqrt((float)d);
  p.scale_log2 = sm * a->q_scale * a->cache.k_scale * 1.4426950408889634f;
  if (!std::isfinite(p.scale_log2)) return fail(B2F_ERR_ARG, "kv4_attention: sm_scale * q_scale * k_scale passes f32");
  if (!(a->ctx_scale > 0.f) || !std::isfinite(a->ctx_scale)) return fail(B2F_ERR_ARG, "kv4_attention: ctx_scale must be > 0");
  if (a->out_dtype != B2F_DTYPE_E4M3 && a->ctx_scale != 1.0f)
    return fail(B2F_ERR_ARG, "kv4_attention: ctx_scale belongs to an e4m3 output");
  if (reinterpret_cast<uintptr_t>(a->lse) & 3) return fail(B2F_ERR_ARG, "kv4_attention: misaligned lse");
  const int sms = sm_count();
  const long long need = attention_workspace(a, sms);
  if (need < 0) return fail(B2F_ERR_CUDA, "kv4_attention: no device");
  if (a->workspace == nullptr || a->workspace_bytes < need || (reinterpret_cast<uintptr_t>(a->workspace) & 15))
    return fail(B2F_ERR_ARG, "kv4_attention: workspace too small or misaligned");
  p.heads = a->heads; p.group = a->heads / hk; p.causal = a->causal != 0;
  p.group_inv = ((1ull << 40) + p.group - 1) / p.group;
  p.q = reinterpret_cast<const char*>(a->q); p.q_dtype = a->q_dtype; p.q_ld = a->q_ld;
  p.out_mul = a->cache.v_scale;
  p.gate = reinterpret_cast<const char*>(a->gate); p.gate_dtype = a->gate_dtype;
  const int four = a->gate_dtype == B2F_DTYPE_BF16 ? 8 : 4;
  p.gate_aligned = reinterpret_cast<uintptr_t>(a->gate) % four == 0 && a->gate_ld % 4 == 0 && a->gate_head_stride % 4 == 0;
  p.gate_ld = a->gate_ld; p.gate_hstride = a->gate_head_stride; p.gate_scale = a->gate_scale;
  p.out = reinterpret_cast<char*>(a->out); p.out_dtype = a->out_dtype; p.out_ld = a->out_ld;
  p.ctx_scale = a->ctx_scale; p.lse = a->lse;
  p.partial = reinterpret_cast<float*>(a->workspace);
  cudaStream_t s = (cudaStream_t)stream;
  if (kv4_tiles_fit(rows_of_a_sequence(a))) return kv4_tiles_launch(p, sms, s);
  // 16 rows a tile read every key half as often as 8 do, once there are more than 8.  With starts the
  // host knows no lengths, and takes all tokens for one sequence's: 64 single tokens of 4 query heads
  // a kv head, 273K keys, 116 us with starts and 77 without (head_dim 64: 81 and 57).
  const long long most = a->batch.starts != nullptr ? a->batch.tokens : a->batch.tokens / a->batch.seqs;
  const int rows = tile_rows(d, most * p.group);
  if (d == 64) return rows == 8 ? launch_attention<64, 1, 4, 3>(p, sms, s) : launch_attention<64, 2, 4, 2>(p, sms, s);
  if (d == 128) return rows == 8 ? launch_attention<128, 1, 3, 3>(p, sms, s) : launch_attention<128, 2, 3, 2>(p, sms, s);
  return launch_attention<256, 1, 3, 3>(p, sms, s);
}

}  // extern "C"
