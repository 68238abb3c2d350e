// What the two kernels of the attention over the 4-bit cache share: their parameters, how the
// work is cut among the CTAs, how rows are finished, and the kernel that joins cut items.
#pragma once
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "common.cuh"
#include "host_common.h"
#include "convert.cuh"
#include "kv4.cuh"

namespace b2f {

constexpr float kLift = 7.0f;             // P is scaled by 2^7 ...
constexpr float kSlack = 8.0f;            // ... and the maximum may lag behind by 2^8

// The item that begins in a CTA's run of units and goes on in those of the next `more` CTAs
// (0: there is none): what the join needs of it.
struct Shared {
  int more, start, n, head0, row0;
};

struct Kv4AttnParams {
  Kv4Cache c;
  Kv4Batch b;
  int heads, group, causal;
  unsigned long long group_inv;  // 2^40 / group, rounded up
  const char* q;
  int q_dtype;
  long long q_ld;
  float scale_log2;  // sm_scale * q_scale * k_scale * log2(e)
  float out_mul;     // v_scale
  const char* gate;
  int gate_dtype;
  long long gate_ld, gate_hstride;
  int gate_aligned;  // four neighbouring gates can be loaded at once
  float gate_scale;
  char* out;
  int out_dtype;
  long long out_ld;
  float ctx_scale;
  float* lse;
  float* partial;  // [2 * CTAs][R][D] O, then [2 * CTAs][R][2] (base, sum)
  Shared* shared;  // [CTAs]
  int ctas;
  int split;     // items may be cut; otherwise every item is one CTA's, and there is no join
};

// One (sequence, kv head, row tile): its keys and rows.
__device__ __forceinline__ int by_group(int row, unsigned long long group_inv) {
  // exact for row * group < 2^40 (row < 2^30, group <= 2^10)
  return (int)(row * group_inv >> 40);
}

struct Item {
  Kv4Seq s;
  int b, h, rt, rts;  // row tiles of the sequence
  int keys;           // keys that some row of the tile may see
  int units;
};

template <int R>
__device__ __forceinline__ int tile_keys(const Kv4AttnParams& p, const Kv4Seq& s, int rt) {
  if (!p.causal) return s.len;
  const int last = by_group(min((rt + 1) * R, s.n * p.group) - 1, p.group_inv);  // last token of the tile
  return max(s.len - s.n + last + 1, 0);
}

template <int U>
__device__ __forceinline__ int units_of(int keys) { return (keys + U - 1) / U; }

// Units of one kv head of a sequence.
template <int R, int U>
__device__ __forceinline__ long long seq_units(const Kv4AttnParams& p, const Kv4Seq& s) {
  const int rts = (s.n * p.group + R - 1) / R;
  if (!p.causal || rts <= 1) return rts == 0 ? 0 : (long long)rts * units_of<U>(tile_keys<R>(p, s, 0));
  long long u = 0;
  for (int rt = 0; rt < rts; ++rt) u += units_of<U>(tile_keys<R>(p, s, rt));
  return u;
}

// x / y for 0 <= x, 0 < y; the 32-bit division where it does (a tenth of the other's time).
__device__ __forceinline__ long long divide(long long x, long long y) {
  return ((x | y) >> 32) == 0 ? (long long)((unsigned)x / (unsigned)y) : x / y;
}

// The units of all items, cut into `ctas` runs of consecutive ones.
struct Runs {
  long long each, more;  // the first `more` CTAs take each + 1 units, the others `each`
  __device__ __forceinline__ Runs(long long total, int ctas) {
    each = divide(total, ctas);
    more = total - each * ctas;
  }
  __device__ __forceinline__ long long begin(int cta) const { return each * cta + min((long long)cta, more); }
  __device__ __forceinline__ int of(long long unit) const {  // the CTA that has it
    const long long x = more * (each + 1);
    return (int)(unit < x ? divide(unit, each + 1) : more + divide(unit - x, each));
  }
};

struct Scan {
  long long warp_sum[32];
  long long at[2];  // units before the sequences of the run's ends
  int b[2];
};

// One round of THREADS sequences: units of thread's sequence base + threadIdx.x (`mine`), of
// those before it (returned), and `before` moved on.
template <int THREADS>
__device__ __forceinline__ long long scan_round(long long mine, long long& before, Scan& sc) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sc.warp_sum[warp] = x;
  __syncthreads();
  long long lead = before;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) lead += sc.warp_sum[w];
    before += sc.warp_sum[w];
  }
  return lead + x - mine;
}

template <int R, int U>
__device__ __forceinline__ void open_item(const Kv4AttnParams& p, Item& it) {
  it.keys = tile_keys<R>(p, it.s, it.rt);
  it.units = units_of<U>(it.keys);
}

// The item of unit `unit` of sequence b, and the unit's place in it.
template <int R, int U>
__device__ int find_item(const Kv4AttnParams& p, int b, long long unit, Item& it) {
  it.b = b;
  it.s = kv4_seq(p.c, p.b, b);
  it.rts = (it.s.n * p.group + R - 1) / R;
  const long long per = seq_units<R, U>(p, it.s);
  it.h = (int)divide(unit, per);
  long long rest = unit - it.h * per;
  for (it.rt = 0;; ++it.rt) {
    open_item<R, U>(p, it);
    if (rest < it.units || it.rt + 1 >= it.rts) break;
    rest -= it.units;
  }
  return (int)rest;
}

// The next item that has units.  There is one: the caller still has units to do.
template <int R, int U>
__device__ void next_item(const Kv4AttnParams& p, Item& it) {
  do {
    if (++it.rt >= it.rts) {
      it.rt = 0;
      if (++it.h >= p.c.kv_heads) {
        it.h = 0;
        do {
          if (++it.b >= p.b.seqs) {
            it.units = 0;
            it.keys = 0;
            return;
          }
          it.s = kv4_seq(p.c, p.b, it.b);
          it.rts = (it.s.n * p.group + R - 1) / R;
        } while (it.rts == 0);
      }
    }
    open_item<R, U>(p, it);
  } while (it.units == 0);
}

// This CTA's run of units [u0, u1), with the sequence of u0 in sc.b[0] and the units before it
// in sc.at[0].  Without splitting, the run is that of the items that begin in it.  `blank`: this CTA has to look after sequences with rows that see no key.
template <int R, int U, int THREADS>
__device__ __forceinline__ Runs find_run(const Kv4AttnParams& p, Scan& sc, long long& u0, long long& u1, bool& blank) {
  long long before = 0, mine = 0, start = 0;
  bool empty = false;
  for (int base = 0; base < p.b.seqs; base += THREADS) {
    const int b = base + (int)threadIdx.x;
    mine = 0;
    if (b < p.b.seqs) {
      const Kv4Seq s = kv4_seq(p.c, p.b, b);
      mine = seq_units<R, U>(p, s) * p.c.kv_heads;
      empty |= b % gridDim.x == blockIdx.x && s.n > 0 && tile_keys<R>(p, s, 0) <= 0;
    }
    start = scan_round<THREADS>(mine, before, sc);
  }
  const Runs runs(before, gridDim.x);
  u0 = runs.begin(blockIdx.x);
  u1 = runs.begin(blockIdx.x + 1);
  auto note = [&](int b) {
    if (u0 >= start && u0 < start + mine) {
      sc.b[0] = b;
      sc.at[0] = start;
    }
    if (u1 >= start && u1 < start + mine) {
      sc.b[1] = b;
      sc.at[1] = start;
    }
  };
  const long long total = before;
  if (p.b.seqs <= THREADS) {
    note(threadIdx.x);
  } else {
    before = 0;
    for (int base = 0; base < p.b.seqs; base += THREADS) {
      const int b = base + (int)threadIdx.x;
      mine = b < p.b.seqs ? seq_units<R, U>(p, kv4_seq(p.c, p.b, b)) * p.c.kv_heads : 0;
      start = scan_round<THREADS>(mine, before, sc);
      note(b);
    }
  }
  blank = __syncthreads_or(empty);
  if (!p.split) {
    Item it;
    if (u1 < total) {
      const int at = find_item<R, U>(p, sc.b[1], u1 - sc.at[1], it);
      if (at > 0) u1 += it.units - at;
    }
    if (u0 < total) {
      const int at = find_item<R, U>(p, sc.b[0], u0 - sc.at[0], it);
      if (at > 0) u0 += it.units - at;
    }
  }
  return runs;
}

// Two e4m3 bytes as an f16 pair (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)v));
  return r;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// a times the lower (upper) half of the pair b.
__device__ __forceinline__ uint32_t hmul2_by(uint32_t a, uint32_t b, int upper) {
  const __half2 x = *reinterpret_cast<const __half2*>(&a), y = *reinterpret_cast<const __half2*>(&b);
  const __half2 z = __hmul2(x, upper ? __high2half2(y) : __low2half2(y));
  return *reinterpret_cast<const uint32_t*>(&z);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float load1(const char* base, int dt, long long off) {
  switch (dt) {
    case kF32: return reinterpret_cast<const float*>(base)[off];
    case kBF16: return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[off]);
    case kF16: return __half2float(reinterpret_cast<const __half*>(base)[off]);
    default: return e4m3_to_f32(reinterpret_cast<const uint8_t*>(base)[off]);
  }
}

__device__ __forceinline__ void store1(char* base, int dt, long long off, float x) {
  switch (dt) {
    case kF32: reinterpret_cast<float*>(base)[off] = x; break;
    case kBF16: reinterpret_cast<__nv_bfloat16*>(base)[off] = __float2bfloat16_rn(x); break;
    case kF16: reinterpret_cast<__half*>(base)[off] = __float2half_rn(x); break;
    default: reinterpret_cast<uint8_t*>(base)[off] = uint8_t(f32x2_to_e4m3x2(x, 0.f)); break;
  }
}

// Where a row (query head x new token, of a kv head h) goes: its token and query head; -1: none.
__device__ __forceinline__ int row_token(const Kv4AttnParams& p, int row, int h, int start, int n, int& head) {
  const int i = by_group(row, p.group_inv);
  head = h * p.group + (row - i * p.group);
  return i < n ? start + i : -1;
}

template <int N>
__device__ __forceinline__ void store_row(const Kv4AttnParams& p, int t, int head, int d0, const float* x) {
  const long long at = (long long)t * p.out_ld + (long long)head * p.c.head_dim + d0;
  if (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      switch (p.out_dtype) {
        case kBF16: store4<kBF16>(p.out, at + i, x + i); break;
        case kF16: store4<kF16>(p.out, at + i, x + i); break;
        default: store4<kE4M3>(p.out, at + i, x + i); break;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) store1(p.out, p.out_dtype, at + i, x[i]);
  }
}

// Normalises, gates and stores N neighbouring elements (o, unnormalised) of one row.  A row that
// saw no key (sum 0) is zeros, whatever its gate.
template <int N>
__device__ __forceinline__ void finish_row(const Kv4AttnParams& p, int t, int head, int d0, const float* o,
                                           float sum) {
  float x[N];
  const float mul = p.out_mul / sum;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = o[i] * mul;
  if (p.gate != nullptr) {
    const long long at = (long long)t * p.gate_ld + head * p.gate_hstride + d0;
    float g[N];
    if (N % 4 == 0 && p.gate_aligned) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        if (p.gate_dtype == kBF16) load4<kBF16>(p.gate, at + i, g + i);
        else load4<kE4M3>(p.gate, at + i, g + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] = load1(p.gate, p.gate_dtype, at + i);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = x[i] / (1.0f + __expf(-g[i] * p.gate_scale));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (p.out_dtype == kE4M3) x[i] = __fdiv_rn(x[i], p.ctx_scale);
    if (sum == 0.f) x[i] = 0.f;
  }
  store_row<N>(p, t, head, d0, x);
}

// log sum exp of a row: P was 2^(score * log2 e - ref), sum over the keys.
__device__ __forceinline__ void finish_lse(const Kv4AttnParams& p, int t, int head, float ref, float sum) {
  if (p.lse == nullptr) return;
  const float l2 = log2f(sum) + ref;
  p.lse[(long long)t * p.heads + head] = sum > 0.f ? l2 * 0.69314718055994531f
                                         : sum != sum ? sum : -INFINITY;
}

// Zeros for the rows that see no key at all, of the sequences that are this CTA's to look after.
template <int D, int R, int THREADS>
__device__ __forceinline__ void blank_rows(const Kv4AttnParams& p) {
  for (int b = blockIdx.x; b < p.b.seqs; b += gridDim.x) {
    const Kv4Seq s = kv4_seq(p.c, p.b, b);
    const int rts = (s.n * p.group + R - 1) / R;
    for (int rt = 0; rt < rts; ++rt) {
      if (tile_keys<R>(p, s, rt) > 0) break;  // later tiles see more
      for (int x = threadIdx.x; x < p.c.kv_heads * R * (D / 4); x += THREADS) {
        const int h = x / (R * (D / 4)), y = x - h * (R * (D / 4));
        int head;
        const int t = row_token(p, rt * R + y / (D / 4), h, s.start, s.n, head);
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        if (t >= 0) {
          store_row<4>(p, t, head, (y % (D / 4)) * 4, zero);
          if (y % (D / 4) == 0) finish_lse(p, t, head, 0.f, 0.f);
        }
      }
    }
  }
}

constexpr int kJoinThreads = 128;

// Joins the pieces of the item that begins in the run of CTA blockIdx.x and goes on in the
// next ones.  A CTA for each row; each warp takes every fourth piece.
template <int D, int R>
__global__ void __launch_bounds__(kJoinThreads) kv4_attention_join_kernel(const Kv4AttnParams p) {
  constexpr int kPer = D / 32;  // elements of a lane
  __shared__ float acc_s[(kJoinThreads / 32)][D], ms[(kJoinThreads / 32)][2];
  pdl_wait();
  pdl_trigger();
  const int me = blockIdx.x, row = blockIdx.y;
  const Shared it = p.shared[me];
  if (it.more == 0) return;
  const int i = by_group(it.row0 + row, p.group_inv);
  if (i >= it.n) return;
  const int t = it.start + i, head = it.head0 + (it.row0 + row) - i * p.group;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* all_ms = p.partial + 2ll * p.ctas * R * D;

  float m = -INFINITY, l = 0.f, acc[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc[k] = 0.f;
#pragma unroll 4
  for (int x = warp; x <= it.more; x += (kJoinThreads / 32)) {
    const long long slot = 2ll * (me + x) + (x == 0 ? 1 : 0);
    const float2 msx = *reinterpret_cast<const float2*>(all_ms + (slot * R + row) * 2);
    const float* o = p.partial + (slot * R + row) * D + lane * kPer;
    float y[kPer];
#pragma unroll
    for (int k = 0; k < kPer; k += 2) {
      const float2 v = *reinterpret_cast<const float2*>(o + k);
      y[k] = v.x;
      y[k + 1] = v.y;
    }
    const float top = fmaxf(m, msx.x);
    const float f = m == top ? 1.f : ex2(m - top), g = msx.x == top ? 1.f : ex2(msx.x - top);
    m = top;
    l = l * f + msx.y * g;
#pragma unroll
    for (int k = 0; k < kPer; ++k) acc[k] = acc[k] * f + y[k] * g;
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) acc_s[warp][lane * kPer + k] = acc[k];
  if (lane == 0) {
    ms[warp][0] = m;
    ms[warp][1] = l;
  }
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < (kJoinThreads / 32); ++w) top = fmaxf(top, ms[w][0]);
  float f[(kJoinThreads / 32)];
  l = 0.f;
#pragma unroll
  for (int w = 0; w < (kJoinThreads / 32); ++w) {
    f[w] = ms[w][0] == top ? 1.f : ex2(ms[w][0] - top);
    l += ms[w][1] * f[w];
  }
  for (int d = threadIdx.x; d < D; d += kJoinThreads) {
    float x[1] = {0.f};
#pragma unroll
    for (int w = 0; w < (kJoinThreads / 32); ++w) x[0] += acc_s[w][d] * f[w];
    finish_row<1>(p, t, head, d, x, l);
  }
  if (threadIdx.x == 0) finish_lse(p, t, head, top, l);
}

// Raises a kernel's shared-memory limit once per device and context.
struct FuncAttrOnce {
  std::atomic<unsigned long long> done[64] = {};
  template <typename K>
  cudaError_t max_smem(K kernel, int bytes) {
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    const unsigned long long token = context_token();
    if (dev < 64 && token != 0 && done[dev].load(std::memory_order_acquire) == token) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done[dev].store(token, std::memory_order_release);
    return e;
  }
};

// The kernel for many rows of queries (kv4_attention_tiles.cu): whether it is for these rows, its
// workspace, and its launch.
bool kv4_tiles_fit(long long rows_of_a_sequence);
long long kv4_tiles_workspace(int head_dim, int sms);
int kv4_tiles_launch(Kv4AttnParams& p, int sms, cudaStream_t s);

}  // namespace b2f
