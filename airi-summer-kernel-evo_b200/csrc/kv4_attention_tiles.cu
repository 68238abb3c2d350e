// Attention over the 4-bit paged cache for many rows of queries (chunks of prompts): the product
// form of kv4_attention.cu on the tensor cores (tcgen05, accumulators in tensor memory).
//
// A CTA works on TILES tiles of 128 query rows (query heads of one kv head x new tokens) and
// walks over the keys 128 at a time:
//   products (1 warp)         S = Q K^T into tensor memory; O += P V with P read from there, then S
//                             of the next step over it
//   dequantisation (7 warps)  K and V codes of the step from the pages to f16 operands in shared
//                             memory, 128-byte-swizzled rows of 64 elements: K-major for Q.K^T,
//                             MN-major for P.V, the same bytes.  e2m1 x e4m3 is exact in f16.
//                             The codes of the next step are in registers while these are
//                             converted, and the page numbers of the one after that.  K and V share
//                             a ring of NS operands.
//   softmax (4 warps a tile)  a thread a row: the row of S from tensor memory, twice (its maximum,
//                             then P = 2^(s - base) as f16 over S), the sum in f32; O is rescaled
//                             only when a score passes the running maximum by 2^8
// Queries are brought to [2^14, 2^15) by a power of two of their row, as in kv4_attention.cu; P is
// at most 2^15, its largest at least 2^7.
//
// The runs of CTAs are as there (equal numbers of units, pieces joined by a second kernel); a unit
// is a step.
//
// Measured: chunks of 512, 83 and 497 tokens of sequences of up to 8192 keys, head_dim 128, 32 heads
// on 8 kv heads: 193 us with the join, 0.60 PFLOP/s.
// Bound: at D = 128 a step of two tiles is 2048 clocks of the tensor pipe, which is busy 35 % of the
// time.  A step takes some 5400: the chain of a tile, S to P (two threads a lane of a scheduler, 128
// exponentials each: 2048 clocks of the exponential unit) to P V to S, is longer than the other
// tile's share can hide.  Tried and no faster: S in halves of 64 keys (199 us against 193), two
// warps for the products (219; with halves 199), rings of two for K and for V apart (the same).
// The 128 registers of a thread do not hold all that the roles have: spilled are, stored and loaded, 8
// and 20 bytes at D = 128, 40 and 80 at 64, 56 and 116 at 256.  At D = 256 a CTA has one tile and a ring
// of two operands, so that the parts of a step follow one another: a chunk of 512 tokens, 16 heads on
// 4, 8192 keys, 175 us; 32 heads of 64 on 8, 92 us.
#include <cfloat>
#include <climits>

#include "kv4_attention.cuh"

namespace b2f {
namespace {

constexpr int kStep = 128;        // keys of a step: also the unit in which items are cut
constexpr int kDequantWarps = 7;

template <int D, int TILES, int NS>
struct Tiles {
  static constexpr int R = 128 * TILES;
  static constexpr int kThreads = 256 + 128 * TILES;
  static constexpr int kQ = 128 * D * 2, kKV = kStep * D * 2;
  static constexpr int kBytes = TILES * kQ + NS * kKV + 1024;
  static constexpr int kSCol(int t) { return t * 128; }
  static constexpr int kOCol(int t) { return TILES * 128 + t * D; }
  static_assert(TILES * (128 + D) <= 512, "tensor memory");
};

__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return make_sdesc_sw128(addr, sbo, lbo);
}

// The products are issued by one lane from code that the whole warp runs: the operands of a converged
// warp are in uniform registers, those of a single lane's branch are moved there one by one (a
// chunk of prompts: 242 us so, 212 us this way, with a first version of the loop below).
__device__ __forceinline__ void mma_ss(bool mine, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)add), "r"((uint32_t)mine)
      : "memory");
}
__device__ __forceinline__ void mma_ts(bool mine, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
      "r"((uint32_t)add), "r"((uint32_t)mine)
      : "memory");
}
__device__ __forceinline__ void commit(bool mine, uint64_t* bar) {
  if (mine) mma_commit(bar);
  __syncwarp();
}

// A wait of the products' warp that is not over at once: out of line, for its loop has to stay in
// the first instruction cache beside those of the other roles.
__device__ __noinline__ bool products_wait(uint64_t* bar, uint32_t parity, int* aborted) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, kDevTimeoutMma, aborted));
}

// A place in the ring and how often it has been gone round.
template <int NS>
struct RingAt {
  uint32_t slot = 0, round = 0;
  __device__ __forceinline__ void next() {
    if (++slot == NS) {
      slot = 0;
      round ^= 1;
    }
  }
};

// The power of two that brings a row of queries, by its largest magnitude, to [2^14, 2^15); and 2^n.
__device__ __forceinline__ int lift_of(float top) {
  const int ex = (__float_as_int(top) >> 23) & 0xff;
  return ex == 0 || ex == 255 ? 0 : min(max(127 + 14 - ex, -120), 120);
}
__device__ __forceinline__ float exp2_of(int n) { return __int_as_float((127 + n) << 23); }

// What the dequantising warps need of a step.
struct StepKeys {
  const uint8_t* block;  // of the kv head in page 0
  const int* pages;      // of the sequence
  int key0, keys;        // first key; keys of the item
  int lowest;            // keys from here on are not seen by every row
};

// Walks over the steps of a CTA's run of units.
template <int R>
struct Cursor {
  Item it;
  int unit, end;   // of the item
  long long left;  // units behind this piece
  __device__ __forceinline__ void open(int first, long long all) {
    unit = first;
    const int take = (int)min((long long)(it.units - first), all);
    end = first + take;
    left = all - take;
  }
  __device__ __forceinline__ bool next_piece(const Kv4AttnParams& p) {
    if (left <= 0) return false;
    next_item<R, kStep>(p, it);
    open(0, left);
    return true;
  }
};

template <int D, int TILES, int NS>
__global__ void __launch_bounds__(Tiles<D, TILES, NS>::kThreads, 1) kv4_attention_tiles_kernel(const Kv4AttnParams p) {
  using C = Tiles<D, TILES, NS>;
  constexpr int R = C::R;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const sq = smem;
  uint8_t* const ring = sq + TILES * C::kQ;  // K of a step, then its V, then the next K, ...
  __shared__ Scan sc;
  __shared__ __align__(8) uint64_t q_full, kv_full[NS], kv_empty[NS],
      s_full[TILES], p_full[TILES], o_full[TILES], drain;
  // Of the eights of keys of a step: those on a bad page; the keys with a NaN value (bits; written
  // with V, in steps that not all rows see to the end).  The pages' flags come with K, whose place is
  // free as soon as S is made, while the softmax warps may still have to read them: K of step m is
  // made when they are at step m - NS / 2 or later, so there are NS / 2 + 1 of them.
  constexpr int kFlags = NS / 2 + 1;
  __shared__ uint32_t bad[kFlags];
  __shared__ __align__(16) uint8_t nan[NS][16];
  __shared__ uint32_t tmem_slot;
  __shared__ int aborted;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 4 * TILES);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&kv_full[s], kDequantWarps);
      mbar_init(&kv_empty[s], 1);
    }
    for (int t = 0; t < TILES; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(&drain, 1);
    aborted = 0;
    fence_mbarrier_init();
  }
  if (warp == 0) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_trigger();

  long long u0, u1;
  bool blank;
  const Runs runs = find_run<R, kStep, C::kThreads>(p, sc, u0, u1, blank);
  // No item yet; stored by the thread that stores the descriptor of one (below).
  if (threadIdx.x == 32 * (1 + kDequantWarps)) p.shared[blockIdx.x].more = 0;
  if (blank) blank_rows<D, R, C::kThreads>(p);
  Cursor<R> cur;
  if (u0 < u1) {
    const int first = find_item<R, kStep>(p, sc.b[0], u0 - sc.at[0], cur.it);
    cur.open(first, u1 - u0);
  }
  auto tiles_of = [&](const Item& it) { return TILES == 1 ? 1 : it.s.n * p.group - it.rt * R > 128 ? 2 : 1; };

  if (u0 >= u1) {
    // nothing to do but to free the tensor memory
  } else if (warp == 0) {
    // -------------------------------------------------------------- products
    constexpr uint32_t idesc_s = make_idesc_f16(128, kStep, 0), idesc_o = make_idesc_f16(128, D, 1);
    const bool mine = elect_one();
    bool ok = true;
    uint32_t piece = 0;
    RingAt<NS> at;
    uint32_t done[2] = {0, 0};  // steps of each tile
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_test(bar, parity & 1)) || products_wait(bar, parity & 1, &aborted);
    };
    auto scores = [&](int t, uint32_t stage) {
      const uint64_t ad = smem_desc(smem_u32(sq + t * C::kQ), 16, 1024);
      const uint64_t bd = smem_desc(smem_u32(ring + stage * C::kKV), 16, 1024);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k >> 2) * 128 * 128 + (k & 3) * 32;  // 64 elements a block of rows
        mma_ss(mine, tmem + C::kSCol(t), ad + (off >> 4), bd + (off >> 4), idesc_s, k != 0);
      }
      commit(mine, &s_full[t]);
    };
    while (ok) {
      const int tiles = __reduce_max_sync(0xffffffffu, tiles_of(cur.it));
      const int take = __reduce_max_sync(0xffffffffu, cur.end - cur.unit);
      ok = wait(&q_full, piece) && wait(&kv_full[at.slot], at.round);
      if (!ok) break;
      tc_fence_after();
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) scores(t, at.slot);
      commit(mine, &kv_empty[at.slot]);
      at.next();
      for (int j = 0; j < take && ok; ++j) {
        const bool more = j + 1 < take;
        const uint32_t vs = at.slot;
        ok = wait(&kv_full[vs], at.round);
        at.next();  // K of the next step
        if (!ok) break;
        const uint64_t vd = smem_desc(smem_u32(ring + vs * C::kKV), kStep * 128, 1024);
#pragma unroll 1
        for (int t = 0; t < tiles && ok; ++t) {
          ok = wait(&p_full[t], done[t]++);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            mma_ts(mine, tmem + C::kOCol(t), tmem + C::kSCol(t) + k * 8, vd + ((k * 2048) >> 4), idesc_o, (j | k) != 0);
          if (more) {  // S of the next step, over the P that has just been used
            if (t == 0) ok = wait(&kv_full[at.slot], at.round);
            if (!ok) break;
            tc_fence_after();
            scores(t, at.slot);
          } else {
            commit(mine, &o_full[t]);
          }
        }
        commit(mine, &kv_empty[vs]);
        if (more) {
          commit(mine, &kv_empty[at.slot]);
          at.next();
        }
      }
      ++piece;
      if (!ok || !cur.next_piece(p)) break;
    }
    commit(mine, &drain);
    mbar_wait(&drain, 0, kDevTimeoutDrain, nullptr);
  } else if (warp <= kDequantWarps) {
    // ------------------------------------------------------------ dequantisation
    // Work is dealt in blocks of eight keys of K or V (q: 0 .. 15 K, 16 .. 31 V): lane = 4 * key + c,
    // c a quarter of the row.
    constexpr int kWords = D / 32;                // 32-bit words of codes of a lane
    constexpr int kMine = (32 + kDequantWarps - 1) / kDequantWarps;  // blocks of a warp, all in flight
    constexpr int kScaleBytes = D / 64;
    const int key8 = lane >> 2, c = lane & 3, first_q = warp - 1;
    const int log2p = p.c.page_log2;
    bool over = false;  // no more steps to look ahead to
    auto look = [&](StepKeys& s) {  // the next step, and the page of lane's block of eight keys
      int page = INT_MIN;           // not needed
      if (cur.unit >= cur.end && !cur.next_piece(p)) over = true;
      if (over) {
        s.keys = -1;
        return page;
      }
      s.block = p.c.storage + (long long)cur.it.h * p.c.block_bytes;
      s.pages = p.c.table + (long long)cur.it.s.row * p.c.table_ld;
      s.key0 = cur.unit * kStep;
      s.keys = cur.it.keys;
      s.lowest = p.causal ? min(cur.it.s.len - cur.it.s.n + by_group(cur.it.rt * R, p.group_inv) + 1, s.keys) : s.keys;
      ++cur.unit;
      const int key = s.key0 + lane * 8;
      if (lane < 16 && key < s.keys) page = max(s.pages[key >> log2p], -1);
      return page;
    };
    uint32_t codes[kMine][kWords], scales[kMine];
    auto load = [&](const StepKeys& s, int page, int q, int i) {
      if (q >= 32) return;
      const int b = q & 15, key = s.key0 + b * 8 + key8;
      const int pg = __shfl_sync(0xffffffffu, page, b);
#pragma unroll
      for (int w = 0; w < kWords; ++w) codes[i][w] = 0;
      scales[i] = 0;
      if ((unsigned)pg >= (unsigned)p.c.pages || key >= s.keys) return;
      const int slot = key & (p.c.page_size - 1);
      const uint8_t* from = s.block + (long long)pg * p.c.page_stride + (q >= 16 ? p.c.codes_bytes + p.c.scales_bytes : 0);
      const uint8_t* row = from + slot * (D / 2) + c * (kWords * 4);
      if constexpr (kWords == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(row);
        codes[i][0] = v.x; codes[i][1] = v.y;
      } else {
#pragma unroll
        for (int w = 0; w < kWords; w += 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(row + w * 4);
          codes[i][w] = v.x; codes[i][w + 1] = v.y; codes[i][w + 2] = v.z; codes[i][w + 3] = v.w;
        }
      }
      const uint8_t* sr = from + p.c.codes_bytes + slot * (D / 16) + c * kScaleBytes;
      if constexpr (kScaleBytes == 1) scales[i] = *sr;
      else if constexpr (kScaleBytes == 2) scales[i] = *reinterpret_cast<const uint16_t*>(sr);
      else scales[i] = *reinterpret_cast<const uint32_t*>(sr);
    };

    StepKeys now, next;
    int page = look(now);
#pragma unroll
    for (int i = 0; i < kMine; ++i) load(now, page, first_q + kDequantWarps * i, i);
    int now_page = page, next_page = look(next);
    bool ok = true;
    RingAt<NS> at;
    RingAt<kFlags> flags;
    while (ok && now.keys >= 0) {
      RingAt<NS> ka = at;  // of K, and of V behind it
      at.next();
      StepKeys after;
      const int after_page = look(after);
      const bool some_hidden = now.key0 + kStep > now.lowest;
      ok = __all_sync(0xffffffffu, mbar_wait(&kv_empty[ka.slot], ka.round ^ 1, kDevTimeoutProducer, &aborted));
      if (ok && warp == 1) {
        const unsigned wrong = __ballot_sync(0xffffffffu, now_page != INT_MIN && (unsigned)now_page >= (unsigned)p.c.pages);
        if (lane == 0) {
          bad[flags.slot] = wrong;
          if (wrong) record_error(kDevBadArgs);
        }
      }
      bool v_free = false;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int q = first_q + kDequantWarps * i;
        if (!ok || q >= 32) break;
        if (q >= 16 && !v_free) {  // K is done
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&kv_full[ka.slot]);
          ok = __all_sync(0xffffffffu, mbar_wait(&kv_empty[at.slot], at.round ^ 1, kDevTimeoutProducer, &aborted));
          if (!ok) break;
          v_free = true;
        }
        const int b = q & 15;
        if (q >= 16 && some_hidden) {
          // A NaN in a value that some row may not see: 0 here, and flagged for the rows that do
          // see it (0 * NaN would reach the others).
          bool flag = false;
          if (now.key0 + b * 8 + key8 >= now.lowest) {
#pragma unroll
            for (int k = 0; k < kScaleBytes; ++k)
              if ((scales[i] >> (8 * k) & 0x7f) == 0x7f) {
                scales[i] &= ~(0xffu << (8 * k));
                flag = true;
              }
          }
          const unsigned any = __ballot_sync(0xffffffffu, flag);
          const unsigned of8 = __ballot_sync(0xffffffffu, lane < 8 && (any >> (4 * (lane & 7)) & 15) != 0);
          if (lane == 0) nan[at.slot][b] = (uint8_t)of8;
        }
        uint8_t* const to = ring + (q < 16 ? ka.slot : at.slot) * C::kKV + (b * 8 + key8) * 128;
        uint32_t m[(kScaleBytes + 1) / 2];
#pragma unroll
        for (int k = 0; k < (kScaleBytes + 1) / 2; ++k) m[k] = e4m3x2_to_f16x2(scales[i] >> (16 * k));
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          uint32_t f[4];
          e2m1x8_to_f16x2(codes[i][w], f);
#pragma unroll
          for (int k = 0; k < 4; ++k) f[k] = hmul2_by(f[k], m[w / 4], (w / 2) & 1);
          const int ch = c * kWords + w;  // sixteen bytes of the row
          *reinterpret_cast<uint4*>(to + (ch >> 3) * (kStep * 128) + (((ch & 7) ^ key8) << 4)) =
              make_uint4(f[0], f[1], f[2], f[3]);
        }
        if (next.keys >= 0) load(next, next_page, q, i);
      }
      if (ok) {
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kv_full[at.slot]);
      }
      at.next();
      flags.next();
      now = next;
      now_page = next_page;
      next = after;
      next_page = after_page;
    }
  } else {
    // ------------------------------------------------------------ softmax, queries and results
    const int t = (warp - 1 - kDequantWarps) >> 2;  // tile
    const int r = (warp & 3) * 32 + lane;        // row of the tile: its lane of tensor memory
    const uint32_t t_lane = tmem + (uint32_t((warp & 3) * 32) << 16);
    bool ok = true;
    uint32_t steps = 0;  // of this tile
    uint32_t pieces = 0, mine = 0;  // of the CTA, and those with rows in this tile
    RingAt<NS> place;               // of the step's K
    RingAt<kFlags> flags;           // and of its pages' flags
    while (ok) {
      const Item& it = cur.it;
      const bool active = t < tiles_of(it);
      const int row = it.rt * R + t * 128 + r, first = cur.unit, take = cur.end - cur.unit;
      int head;
      const int token = row_token(p, row, it.h, it.s.start, it.s.n, head);
      float mul = 0.f;
      int limit = it.keys;
      const int lowest = p.causal ? min(it.s.len - it.s.n + by_group(it.rt * R, p.group_inv) + 1, it.keys) : it.keys;
      if (active) {
        // Q of the warp's 32 rows, eight elements a lane, and each row's power of two
        constexpr int kLanes = D / 8, kRows = 32 / kLanes;  // lanes of a row, rows at once
        const int e = (lane % kLanes) * 8;
        const long long mine_at = (long long)token * p.q_ld + (long long)head * D;
        uint8_t* const to = sq + t * C::kQ + (e >> 6) * (128 * 128);
        float own = 0.f;  // the largest of this lane's row
#pragma unroll 4
        for (int i = 0; i < kLanes; ++i) {
          const int x = i * kRows + lane / kLanes, rr = (warp & 3) * 32 + x;
          const int there = __shfl_sync(0xffffffffu, token, x);
          const long long at = __shfl_sync(0xffffffffu, mine_at, x) + e;
          float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (there >= 0) {
            if (p.q_dtype == kBF16) { load4<kBF16>(p.q, at, y); load4<kBF16>(p.q, at + 4, y + 4); }
            else if (p.q_dtype == kF16) { load4<kF16>(p.q, at, y); load4<kF16>(p.q, at + 4, y + 4); }
            else { load4<kE4M3>(p.q, at, y); load4<kE4M3>(p.q, at + 4, y + 4); }
          }
          float top = 0.f;
#pragma unroll
          for (int k = 0; k < 8; k += 2) top = fmax3(top, fabsf(y[k]), fabsf(y[k + 1]));
#pragma unroll
          for (int k = 1; k < kLanes; k *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
          const float lift = exp2_of(lift_of(top));
          *reinterpret_cast<uint4*>(to + rr * 128 + ((((e >> 3) & 7) ^ (rr & 7)) << 4)) =
              make_uint4(pack_f16x2(y[0] * lift, y[1] * lift), pack_f16x2(y[2] * lift, y[3] * lift),
                         pack_f16x2(y[4] * lift, y[5] * lift), pack_f16x2(y[6] * lift, y[7] * lift));
          const float theirs = __shfl_sync(0xffffffffu, top, lane % kRows * kLanes);
          if (lane / kRows == i) own = theirs;
        }
        mul = fmaxf(exp2_of(-lift_of(own)) * p.scale_log2, FLT_MIN);  // -infinity * 0 is none
        if (p.causal && token >= 0) limit = min(it.s.len - it.s.n + (token - it.s.start) + 1, it.keys);
      }
      fence_async_shared();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      ++pieces;
      if (!active) {  // the next queries wait until the piece is done: q_full counts all eight warps once
        for (int j = 0; j < take; ++j) {
          place.next();
          place.next();
          flags.next();
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&o_full[0], (pieces - 1) & 1, kDevTimeoutEpilogue, &aborted));
        if (!ok || !cur.next_piece(p)) break;
        continue;
      }
      ++mine;

      float base = -INFINITY, sum = 0.f;
      for (int j = 0; j < take && ok; ++j, ++steps) {
        const int key0 = (first + j) * kStep;
        place.next();
        const bool some_hidden = key0 + kStep > lowest;
        const uint32_t col = t_lane + C::kSCol(t);
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], steps & 1, kDevTimeoutEpilogue, &aborted));
        if (!ok) break;
        tc_fence_after();
        const uint32_t wrong = bad[flags.slot];
        if (some_hidden) {  // V of the step has come: its flags can be read
          ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[place.slot], place.round, kDevTimeoutEpilogue, &aborted));
          if (!ok) break;
        }
        if (some_hidden || wrong != 0) {
          // Scores that the row may not see become -infinity, and NaN those that bring a NaN value
          // (its scale was set to 0), in place: a loop of its own keeps the code below short.
#pragma unroll 1
          for (int k = 0; k < kStep; k += 16) {
            uint32_t x[16];
            tmem_ld16(col + k, x);
            const uint32_t b2 = wrong >> (k / 8);
            const uint32_t n2 = some_hidden ? *reinterpret_cast<const uint16_t*>(nan[place.slot] + k / 8) : 0;
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              if (n2 >> u & 1) x[u] = 0x7fffffffu;
              if (key0 + k + u >= limit || (b2 >> (u / 8) & 1)) x[u] = 0xff800000u;
            }
            tmem_st16(col + k, x);
          }
          tmem_st_wait();
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains of maxima, of sums below
        uint32_t a[32], b[32];
#pragma unroll 1
        for (int k = 0; k < kStep; k += 64) {
          tmem_ld32_async(col + k, a);
          tmem_ld32_async(col + k + 32, b);
          tmem_ld_wait_regs(a);
          reg_fence32(b);
#pragma unroll
          for (int u = 0; u < 32; u += 2) {
            tops[u / 2 & 1] = fmax3(tops[u / 2 & 1], __uint_as_float(a[u]), __uint_as_float(a[u + 1]));
            tops[2 + (u / 2 & 1)] = fmax3(tops[2 + (u / 2 & 1)], __uint_as_float(b[u]), __uint_as_float(b[u + 1]));
          }
        }
        tmem_ld32_async(col, a);  // again, for the weights: on its way while the maxima are joined
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * mul;
        // as in kv4_attention.cu: the base follows a new maximum only when it is 2^8 ahead
        float f = 1.f;
        const bool jump = top - base > kSlack + kLift;
        if (jump) {
          f = ex2(base - (top - kLift));
          base = top - kLift;
        }
        if (__any_sync(0xffffffffu, jump) && j > 0) {  // O is complete up to the step before: S came after it
#pragma unroll 1
          for (int k = 0; k < D; k += 16) {
            uint32_t o[16];
            tmem_ld16(t_lane + C::kOCol(t) + k, o);
#pragma unroll
            for (int u = 0; u < 16; ++u) o[u] = __float_as_uint(__uint_as_float(o[u]) * f);
            tmem_st16(t_lane + C::kOCol(t) + k, o);
          }
        }
        const float ref = base == -INFINITY ? 0.f : base;
        float2 part[4] = {};
        const float2 mul2 = make_float2(mul, mul), ref2 = make_float2(-ref, -ref);
        auto weights = [&](int k, uint32_t (&s)[32]) {  // P of 32 keys, over the columns of S
          uint32_t pk[16];
#pragma unroll
          for (int u = 0; u < 32; u += 2) {
            const float2 x = ffma2(make_float2(__uint_as_float(s[u]), __uint_as_float(s[u + 1])), mul2, ref2);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            part[u / 2 & 3] = fadd2(part[u / 2 & 3], e);
            pk[u / 2] = pack_f16x2(e.x, e.y);
          }
          tmem_st16(col + k / 2, pk);
        };
#pragma unroll 1
        for (int k = 0; k < kStep; k += 64) {
          tmem_ld_wait_regs(a);
          tmem_ld32_async(col + k + 32, b);
          weights(k, a);
          tmem_ld_wait_regs(b);
          if (k + 64 < kStep) tmem_ld32_async(col + k + 64, a);
          weights(k + 32, b);
        }
        part[0] = fadd2(fadd2(part[0], part[1]), fadd2(part[2], part[3]));
        sum = sum * f + (part[0].x + part[0].y);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        place.next();
        flags.next();
      }
      if (!ok) break;
      // ---- the piece is done
      ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], (mine - 1) & 1, kDevTimeoutEpilogue, &aborted));
      if (!ok) break;
      tc_fence_after();
      const bool from_start = first == 0, to_end = cur.end == it.units, whole = from_start && to_end;
      const int slot = 2 * blockIdx.x + (from_start ? 1 : 0);
      if (from_start && !to_end && threadIdx.x == 32 * (1 + kDequantWarps)) {
        const int last = runs.of(u1 - (cur.left + take) + it.units - 1);
        p.shared[blockIdx.x] = Shared{last - (int)blockIdx.x, it.s.start, it.s.n, it.h * p.group, it.rt * R};
      }
      float* const part_o = p.partial + ((long long)slot * R + t * 128) * D;
      float* const part_ms = p.partial + 2ll * p.ctas * R * D + ((long long)slot * R + t * 128 + r) * 2;
      // O of the warp's rows through shared memory (where their queries were), sixteen columns at a
      // time: a lane then stores four elements, and four lanes the 64 bytes of a row.
      constexpr int kLd = 20;  // floats of a row there: sixteen and a pad
      float* const turn = reinterpret_cast<float*>(sq + t * C::kQ + (warp & 3) * 32 * 128);
#pragma unroll 1
      for (int d = 0; d < D; d += 16) {
        uint32_t o[16];
        tmem_ld16(t_lane + C::kOCol(t) + d, o);
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 16; u += 4)
          *reinterpret_cast<uint4*>(turn + lane * kLd + u) = make_uint4(o[u], o[u + 1], o[u + 2], o[u + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = i * 8 + (lane >> 2), c = (lane & 3) * 4;
          const float4 v = *reinterpret_cast<const float4*>(turn + x * kLd + c);
          if (whole) {
            const float y[4] = {v.x, v.y, v.z, v.w};
            const int t2 = __shfl_sync(0xffffffffu, token, x), h2 = __shfl_sync(0xffffffffu, head, x);
            const float sum2 = __shfl_sync(0xffffffffu, sum, x);
            if (t2 >= 0) finish_row<4>(p, t2, h2, d + c, y, sum2);
          } else {
            *reinterpret_cast<float4*>(part_o + ((warp & 3) * 32 + x) * D + d + c) = v;
          }
        }
      }
      __syncwarp();
      if (whole) {
        if (token >= 0) finish_lse(p, token, head, base, sum);
      } else {
        part_ms[0] = base;
        part_ms[1] = sum;
      }
      tc_fence_before();
      if (!cur.next_piece(p)) break;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The join for tiles: a warp for each row of the item that begins in the run of CTA blockIdx.x.
template <int D, int R>
__global__ void __launch_bounds__(kJoinThreads) kv4_tiles_join_kernel(const Kv4AttnParams p) {
  constexpr int kPer = D / 32;
  pdl_wait();
  pdl_trigger();
  const int me = blockIdx.x, lane = threadIdx.x & 31;
  const Shared it = p.shared[me];
  if (it.more == 0) return;
  const float* all_ms = p.partial + 2ll * p.ctas * R * D;
  for (int row = blockIdx.y * (kJoinThreads / 32) + (threadIdx.x >> 5); row < R; row += gridDim.y * (kJoinThreads / 32)) {
    const int i = by_group(it.row0 + row, p.group_inv);
    if (i >= it.n) return;
    const int t = it.start + i, head = it.head0 + (it.row0 + row) - i * p.group;
    float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
#pragma unroll 2
    for (int x = 0; x <= it.more; ++x) {
      const long long slot = (2ll * (me + x) + (x == 0 ? 1 : 0)) * R + row;
      const float2 ms = *reinterpret_cast<const float2*>(all_ms + slot * 2);
      const float* o = p.partial + slot * D + lane * kPer;
      const float top = fmaxf(m, ms.x);
      const float f = m == top ? 1.f : ex2(m - top), g = ms.x == top ? 1.f : ex2(ms.x - top);
      m = top;
      l = l * f + ms.y * g;
#pragma unroll
      for (int k = 0; k < kPer; k += 2) {
        const float2 v = *reinterpret_cast<const float2*>(o + k);
        acc[k] = acc[k] * f + v.x * g;
        acc[k + 1] = acc[k + 1] * f + v.y * g;
      }
    }
    finish_row<kPer>(p, t, head, lane * kPer, acc, l);
    if (lane == 0) finish_lse(p, t, head, m, l);
  }
}

template <int D, int TILES, int NS>
int launch_tiles(Kv4AttnParams& p, int sms, cudaStream_t s) {
  using C = Tiles<D, TILES, NS>;
  static_assert(C::kBytes + 2048 <= 227 * 1024, "a CTA fits on an SM");
  static FuncAttrOnce once;
  p.ctas = sms;
  p.split = 1;
  p.shared = reinterpret_cast<Shared*>(p.partial + 2ll * p.ctas * C::R * (D + 2));
  B2F_CUDA_TRY(once.max_smem(kv4_attention_tiles_kernel<D, TILES, NS>, C::kBytes));
  B2F_CUDA_TRY(launch_pdl(kv4_attention_tiles_kernel<D, TILES, NS>, dim3((unsigned)p.ctas), dim3(C::kThreads), C::kBytes, s, p));
  B2F_CUDA_TRY(launch_pdl(kv4_tiles_join_kernel<D, C::R>, dim3((unsigned)p.ctas, 16), dim3(kJoinThreads), 0, s, p));
  return B2F_OK;
}

}  // namespace

// Rows a sequence (new tokens x query heads of a kv head), on average, from which this form is the
// faster one.  Microseconds, this form / the one of kv4_attention.cu, full sequences:
//   rows                            64         128        512
//   D  64, 4 sequences of 4096    27 / 21    30 / 28    45 / 72
//   D 128, 4 sequences of 4096    47 / 39    49 / 61    78 / 194
//   D 128, 16 sequences of 1024   24 / 22    26 / 30    46 / 75
//   D 128, 1 sequence of 1024     21 / 16    23 / 18    31 / 31
//   D 256, 4 sequences of 2048    38 / 34    43 / 52    79 / 150
// The average is all that the host knows of a call with starts, and misjudges mixed ones: D 128, 512
// tokens over 8192 keys take 117 us in this form, 63 single tokens over 265K keys 116 in the other, and
// both in one call 466 (36 rows on average, the other form; with 2048 tokens, 132 rows, this one: 740).
bool kv4_tiles_fit(long long rows) { return rows >= 96; }

long long kv4_tiles_workspace(int head_dim, int sms) {
  const int rows = head_dim == 256 ? 128 : 256;
  return (long long)sms * (2ll * rows * (head_dim + 2) * 4 + (long long)sizeof(Shared));
}

int kv4_tiles_launch(Kv4AttnParams& p, int sms, cudaStream_t s) {
  if (p.c.head_dim == 64) return launch_tiles<64, 2, 8>(p, sms, s);
  if (p.c.head_dim == 128) return launch_tiles<128, 2, 5>(p, sms, s);
  return launch_tiles<256, 1, 2>(p, sms, s);
}

}  // namespace b2f
