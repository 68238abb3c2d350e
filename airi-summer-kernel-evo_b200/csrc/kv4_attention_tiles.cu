// Attention over the 4-bit paged cache for many rows of queries (chunks of prompts): the product
// form of kv4_attention.cu on the tensor cores (tcgen05, accumulators in tensor memory).
//
// A CTA works on TILES tiles of 128 query rows (query heads of one kv head x new tokens) and
// walks over the keys 128 at a time:
//   dequantisation (3 warps)  K and V codes of the step from the pages to f16 operands in shared
//                             memory, 128-byte-swizzled rows of 64 elements: K-major for Q.K^T,
//                             MN-major for P.V, the same bytes.  e2m1 x e4m3 is exact in f16.
//                             The codes of the next step are in registers while these are
//                             converted, and the page numbers of the one after that.
//   products (1 thread)       S = Q K^T into tensor memory; O += P V with P read from there
//   softmax (4 warps a tile)  a thread a row: the row of S into registers, P = 2^(s - base) as f16
//                             over S, the sum in f32; O is rescaled only when a score passes the
//                             running maximum by 2^8
// With two tiles the tensor cores work on one while the other is exponentiated.  Queries are
// brought to [2^14, 2^15) by a power of two of their row, as in kv4_attention.cu; P is at most
// 2^15, its largest at least 2^7.
//
// Bound: a step of two tiles is 4 * 2 * 128 * 128 * D operations: 2100 clocks of an SM at D =
// 128, about what the softmax warps take for it; converting its codes is the third of the three
// warpgroups' work beside them.
#include <climits>

#include "kv4_attention.cuh"

namespace b2f {
namespace {

constexpr int kStep = 128;        // keys of a step: also the unit in which items are cut
constexpr int kDequantWarps = 7;

template <int D, int TILES, int ST>
struct Tiles {
  static constexpr int R = 128 * TILES;
  static constexpr int kThreads = 256 + 128 * TILES;
  static constexpr int kQ = 128 * D * 2, kKV = kStep * D * 2;
  static constexpr int kBytes = TILES * kQ + 2 * ST * kKV + 1024;
  static constexpr int kSCol(int t) { return t * 128; }
  static constexpr int kOCol(int t) { return TILES * 128 + t * D; }
  static_assert(TILES * (128 + D) <= 512, "tensor memory");
};

__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return make_sdesc_sw128(addr, sbo, lbo);
}

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

template <int D, int TILES, int ST>
__global__ void __launch_bounds__(Tiles<D, TILES, ST>::kThreads, 1) kv4_attention_tiles_kernel(const Kv4AttnParams p) {
  using C = Tiles<D, TILES, ST>;
  constexpr int R = C::R;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const sq = smem;
  uint8_t* const sk = sq + TILES * C::kQ;
  uint8_t* const sv = sk + ST * C::kKV;
  __shared__ Scan sc;
  __shared__ __align__(8) uint64_t q_full, k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], s_full[TILES],
      p_full[TILES], o_full[TILES], drain;
  // Of the eights of keys of a step: those on a bad page; the keys with a NaN value (bits; written
  // in steps that not all rows see to the end).
  __shared__ uint32_t bad[ST];
  __shared__ __align__(16) uint8_t nan[ST][16];
  __shared__ uint32_t tmem_slot;
  __shared__ int aborted;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 4 * TILES);
    for (int s = 0; s < ST; ++s) {
      mbar_init(&k_full[s], kDequantWarps);
      mbar_init(&v_full[s], kDequantWarps);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_empty[s], 1);
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
  if (blank) blank_rows<D, R, C::kThreads>(p);
  if (threadIdx.x == 0) p.shared[blockIdx.x].more = 0;
  Cursor<R> cur;
  if (u0 < u1) {
    const int first = find_item<R, kStep>(p, sc.b[0], u0 - sc.at[0], cur.it);
    cur.open(first, u1 - u0);
  }
  auto tiles_of = [&](const Item& it) { return TILES == 1 ? 1 : it.s.n * p.group - it.rt * R > 128 ? 2 : 1; };

  if (u0 >= u1) {
    // nothing to do but to free the tensor memory
  } else if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ products
      constexpr uint32_t idesc_s = make_idesc_f16(128, kStep, 0), idesc_o = make_idesc_f16(128, D, 1);
      bool ok = true;
      uint32_t piece = 0;
      long long n = 0;         // steps
      uint32_t done[2] = {0, 0};  // steps of each tile
      auto scores = [&](int t, int stage) {
        const uint32_t qa = smem_u32(sq + t * C::kQ), ka = smem_u32(sk + stage * C::kKV);
        const uint64_t ad = smem_desc(qa, 16, 1024), bd = smem_desc(ka, 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t at = (k >> 2) * 128 * 128 + (k & 3) * 32;  // 64 elements a block of rows
          mma_bf16(tmem + C::kSCol(t), ad + (at >> 4), bd + (at >> 4), idesc_s, k != 0);
        }
        mma_commit(&s_full[t]);
      };
      while (ok) {
        const int tiles = tiles_of(cur.it), take = cur.end - cur.unit;
        ok = mbar_wait(&q_full, piece & 1, kDevTimeoutMma, &aborted) &&
             mbar_wait(&k_full[n % ST], (n / ST) & 1, kDevTimeoutMma, &aborted);
        if (!ok) break;
        tc_fence_after();
        for (int t = 0; t < tiles; ++t) scores(t, n % ST);
        mma_commit(&k_empty[n % ST]);
        for (int j = 0; j < take && ok; ++j, ++n) {
          const bool more = j + 1 < take;
          const int st = n % ST, nst = (n + 1) % ST;
          ok = mbar_wait(&v_full[st], (n / ST) & 1, kDevTimeoutMma, &aborted);
          if (!ok) break;
          const uint64_t vd = smem_desc(smem_u32(sv + st * C::kKV), kStep * 128, 1024);
          for (int t = 0; t < tiles && ok; ++t) {
            ok = mbar_wait(&p_full[t], done[t] & 1, kDevTimeoutMma, &aborted);
            if (!ok) break;
            ++done[t];
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < kStep / 16; ++k)
              mma_bf16_ts(tmem + C::kOCol(t), tmem + C::kSCol(t) + k * 8, vd + ((k * 2048) >> 4), idesc_o,
                          (j | k) != 0);
            if (!more) {
              mma_commit(&o_full[t]);
            } else {
              if (t == 0) ok = mbar_wait(&k_full[nst], ((n + 1) / ST) & 1, kDevTimeoutMma, &aborted);
              if (!ok) break;
              tc_fence_after();
              scores(t, nst);
            }
          }
          mma_commit(&v_empty[st]);
          if (more) mma_commit(&k_empty[nst]);
        }
        ++piece;
        if (!ok || !cur.next_piece(p)) break;
      }
      mma_commit(&drain);
      mbar_wait(&drain, 0, kDevTimeoutDrain, nullptr);
    }
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
      if (lane < 16 && key < s.keys) page = s.pages[key >> log2p];
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
    for (long long n = 0; ok && now.keys >= 0; ++n) {
      const int st = n % ST;
      const uint32_t ph = ((n / ST) & 1) ^ 1;
      StepKeys after;
      const int after_page = look(after);
      const bool some_hidden = now.key0 + kStep > now.lowest;
      ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], ph, kDevTimeoutProducer, &aborted));
      bool v_free = false;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int q = first_q + kDequantWarps * i;
        if (!ok || q >= 32) break;
        if (q >= 16 && !v_free) {  // K is done
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&k_full[st]);
          ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[st], ph, kDevTimeoutProducer, &aborted));
          if (!ok) break;
          v_free = true;
          if (warp == 1) {
            const unsigned wrong = __ballot_sync(0xffffffffu, now_page != INT_MIN && (unsigned)now_page >= (unsigned)p.c.pages);
            if (lane == 0) {
              bad[st] = wrong;
              if (wrong) record_error(kDevBadArgs);
            }
          }
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
          if (lane == 0) nan[st][b] = (uint8_t)of8;
        }
        uint8_t* const to = (q < 16 ? sk : sv) + st * C::kKV + (b * 8 + key8) * 128;
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
        if (lane == 0) mbar_arrive(&v_full[st]);
      }
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
    uint32_t n = 0;                 // steps of the CTA
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
        // the row of Q: the power of two, then the operand
        const long long at = (long long)token * p.q_ld + (long long)head * D;
        float top = 0.f;
        auto q4 = [&](int e, float* y) {
          if (p.q_dtype == kBF16) load4<kBF16>(p.q, at + e, y);
          else if (p.q_dtype == kF16) load4<kF16>(p.q, at + e, y);
          else load4<kE4M3>(p.q, at + e, y);
        };
        if (token >= 0) {
#pragma unroll 4
          for (int e = 0; e < D; e += 4) {
            float y[4];
            q4(e, y);
            top = fmax3(top, fabsf(y[0]), fabsf(y[1]));
            top = fmax3(top, fabsf(y[2]), fabsf(y[3]));
          }
        }
        const int ex = (__float_as_int(top) >> 23) & 0xff;
        const int up = ex == 0 || ex == 255 ? 0 : min(max(127 + 14 - ex, -120), 120);
        const float lift = __int_as_float((127 + up) << 23);
        mul = __int_as_float((127 - up) << 23) * p.scale_log2;
        uint8_t* const to = sq + t * C::kQ + r * 128;
#pragma unroll 4
        for (int e = 0; e < D; e += 8) {
          float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          if (token >= 0) {
            q4(e, y);
            q4(e + 4, y + 4);
          }
          *reinterpret_cast<uint4*>(to + (e >> 6) * (128 * 128) + ((((e >> 3) & 7) ^ (r & 7)) << 4)) =
              make_uint4(pack_f16x2(y[0] * lift, y[1] * lift), pack_f16x2(y[2] * lift, y[3] * lift),
                         pack_f16x2(y[4] * lift, y[5] * lift), pack_f16x2(y[6] * lift, y[7] * lift));
        }
        if (p.causal && token >= 0) limit = min(it.s.len - it.s.n + (token - it.s.start) + 1, it.keys);
      }
      fence_async_shared();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
      ++pieces;
      if (!active) {  // the next queries wait until the piece is done: q_full counts all eight warps once
        n += take;
        ok = __all_sync(0xffffffffu, mbar_wait(&o_full[0], (pieces - 1) & 1, kDevTimeoutEpilogue, &aborted));
        if (!ok || !cur.next_piece(p)) break;
        continue;
      }
      ++mine;

      float base = -INFINITY, sum = 0.f;
      for (int j = 0; j < take && ok; ++j, ++steps, ++n) {
        const int st = n % ST, key0 = (first + j) * kStep;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], steps & 1, kDevTimeoutEpilogue, &aborted));
        if (!ok) break;
        tc_fence_after();
        // V of the step has come: its flags can be read
        ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (n / ST) & 1, kDevTimeoutEpilogue, &aborted));
        if (!ok) break;
        const uint32_t wrong = bad[st];
        const bool some_hidden = key0 + kStep > lowest;
        if (some_hidden || wrong != 0) {
          // Scores that the row may not see become -infinity, and NaN those that bring a NaN value
          // (its scale was set to 0), in place: a loop of its own keeps the code below short.
#pragma unroll 1
          for (int k = 0; k < kStep; k += 16) {
            uint32_t x[16];
            tmem_ld16(t_lane + C::kSCol(t) + k, x);
            const uint32_t b2 = wrong >> (k / 8);
            const uint32_t n2 = some_hidden ? *reinterpret_cast<const uint16_t*>(nan[st] + k / 8) : 0;
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              if (n2 >> u & 1) x[u] = 0x7fffffffu;
              if (key0 + k + u >= limit || (b2 >> (u / 8) & 1)) x[u] = 0xff800000u;
            }
            tmem_st16(t_lane + C::kSCol(t) + k, x);
          }
          tmem_st_wait();
        }
        // Two passes over the row of S, 32 columns at a time, the next ones on their way: the
        // registers of a whole row would halve the warps of the CTA.
        uint32_t a[32], b[32];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains of maxima, of sums below
        tmem_ld32_async(t_lane + C::kSCol(t), a);
#pragma unroll
        for (int k = 0; k < kStep; k += 64) {
          tmem_ld_wait_regs(a);
          tmem_ld32_async(t_lane + C::kSCol(t) + k + 32, b);
#pragma unroll
          for (int u = 0; u < 32; u += 2)
            tops[u / 2 & 3] = fmax3(tops[u / 2 & 3], __uint_as_float(a[u]), __uint_as_float(a[u + 1]));
          tmem_ld_wait_regs(b);
          tmem_ld32_async(t_lane + C::kSCol(t) + (k == 0 ? 64 : 0), a);  // behind the last: the first again
#pragma unroll
          for (int u = 0; u < 32; u += 2)
            tops[u / 2 & 3] = fmax3(tops[u / 2 & 3], __uint_as_float(b[u]), __uint_as_float(b[u + 1]));
        }
        tmem_ld_wait_regs(a);
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * mul;
        // as in kv4_attention.cu: the base follows a new maximum only when it is 2^8 ahead
        float f = 1.f;
        const bool jump = top - base > kSlack + kLift;
        if (jump) {
          f = ex2(base - (top - kLift));
          base = top - kLift;
        }
        if (__any_sync(0xffffffffu, jump) && j > 0) {
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
        // P of 32 keys goes over columns of S that have been read
        auto weights = [&](int k, uint32_t (&s)[32]) {
          uint32_t pk[16];
#pragma unroll
          for (int u = 0; u < 32; u += 2) {
            const float2 x = ffma2(make_float2(__uint_as_float(s[u]), __uint_as_float(s[u + 1])), mul2, ref2);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            part[u / 2 & 3] = fadd2(part[u / 2 & 3], e);
            pk[u / 2] = pack_f16x2(e.x, e.y);
          }
          tmem_st16(t_lane + C::kSCol(t) + k / 2, pk);
        };
#pragma unroll
        for (int k = 0; k < kStep; k += 64) {
          tmem_ld32_async(t_lane + C::kSCol(t) + k + 32, b);
          weights(k, a);
          tmem_ld_wait_regs(b);
          if (k == 0) tmem_ld32_async(t_lane + C::kSCol(t) + 64, a);
          weights(k + 32, b);
          if (k == 0) tmem_ld_wait_regs(a);
        }
        part[0] = fadd2(fadd2(part[0], part[1]), fadd2(part[2], part[3]));
        sum = sum * f + (part[0].x + part[0].y);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
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
      float* const part_o = p.partial + ((long long)slot * R + t * 128 + r) * D;
      float* const part_ms = p.partial + 2ll * p.ctas * R * D + ((long long)slot * R + t * 128 + r) * 2;
#pragma unroll 1
      for (int d = 0; d < D; d += 16) {
        uint32_t o[16];
        tmem_ld16(t_lane + C::kOCol(t) + d, o);
        float x[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) x[u] = __uint_as_float(o[u]);
        if (whole) {
          if (token >= 0) finish_row<16>(p, token, head, d, x, sum);
        } else {
#pragma unroll
          for (int u = 0; u < 16; u += 4)
            *reinterpret_cast<float4*>(part_o + d + u) = make_float4(x[u], x[u + 1], x[u + 2], x[u + 3]);
        }
      }
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

template <int D, int TILES, int ST>
int launch_tiles(Kv4AttnParams& p, int sms, cudaStream_t s) {
  using C = Tiles<D, TILES, ST>;
  static_assert(C::kBytes + 2048 <= 227 * 1024, "a CTA fits on an SM");
  static FuncAttrOnce once;
  p.ctas = sms;
  p.split = 1;
  p.shared = reinterpret_cast<Shared*>(p.partial + 2ll * p.ctas * C::R * (D + 2));
  B2F_CUDA_TRY(once.max_smem(kv4_attention_tiles_kernel<D, TILES, ST>, C::kBytes));
  B2F_CUDA_TRY(launch_pdl(kv4_attention_tiles_kernel<D, TILES, ST>, dim3((unsigned)p.ctas), dim3(C::kThreads), C::kBytes, s, p));
  B2F_CUDA_TRY(launch_pdl(kv4_tiles_join_kernel<D, C::R>, dim3((unsigned)p.ctas, 16), dim3(kJoinThreads), 0, s, p));
  return B2F_OK;
}

}  // namespace

bool kv4_tiles_fit(int head_dim, long long rows) { return rows >= 64; }

long long kv4_tiles_workspace(int head_dim, int sms) {
  const int rows = head_dim == 256 ? 128 : 256;
  return (long long)sms * (2ll * rows * (head_dim + 2) * 4 + (long long)sizeof(Shared));
}

int kv4_tiles_launch(Kv4AttnParams& p, int sms, cudaStream_t s) {
  if (p.c.head_dim == 64) return launch_tiles<64, 2, 2>(p, sms, s);
  if (p.c.head_dim == 128) return launch_tiles<128, 2, 2>(p, sms, s);
  return launch_tiles<256, 1, 1>(p, sms, s);
}

}  // namespace b2f
