// Rotary positions of q and k at explicit positions (C ABI: b2f_rotary).
//
// Pair i of a head turns by the angle a = position * w_i:
//   (x, y) -> magnitude * (x cos a - y sin a, y cos a + x sin a)
// Pairs are (i, i + rotary_dim / 2) or (2 i, 2 i + 1); elements behind rotary_dim pass through.
// With weights the head is RMS-normalised first: x * rsqrt(mean(x^2) + eps) * (w + offset).
//
// Angles of far positions: w_i is handed over as the fraction of a turn per position in
// 64-bit fixed point (2^64 = one turn), so position * w_i modulo 2^64 IS the fraction of a
// turn, exact but for the rounding of w_i (2^-65 of a turn per position: 2^-34 of a turn at
// position 2^31, 2^-25 at 2^40).  Two integer multiply-adds give its top 32 bits; the f32 sincospi
// of those adds about 2^-24 of a half turn at any position.
//
// Bound: memory (each element is read and written once).  A lane owns four pairs of a head
// (8 elements), so a rotation needs no shuffle; a warp owns one token and walks over its
// heads with the four sines and cosines of the lane in registers (their cost is shared by
// all heads of q and k), the next head loaded ahead.  With few tokens the heads of a
// token are dealt to several warps (see the launch).
//
// Measured (bytes in and out over device time): 8192 tokens x 40 heads of 128, f32, interleaved
// 56 us, 6.0 TB/s; 4099 x 20 heads of 256, bf16, 64 elements rotated 21.9 us, 3.8 TB/s (84 MB: an
// elementwise copy of 42 MB, which moves as much, takes 29 us); 8 tokens, e4m3 and RMS weights
// 2.3 us, a launch.
#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "host_common.h"
#include "convert.cuh"

namespace b2f {
namespace {

struct RotaryParams {
  int rows, q_heads, k_heads, head_dim, rotary_dim;
  int lanes_log2;                              // lanes of a head
  int rounds, warps_per_row, rounds_per_warp;  // a round: the heads that a warp has at a time
  int inverse, position_bits;
  const char* q;
  const char* k;
  long long q_ld, q_hstride, k_ld, k_hstride;  // elements
  float in_scale;
  const float* q_weight;
  const float* k_weight;
  float weight_offset, eps;
  const void* positions;
  const unsigned long long* freqs;
  float magnitude;
  char* q_out;
  char* k_out;
  long long q_out_ld, k_out_ld;
  float out_scale;
};

constexpr int kRotaryWarps = 4;

// The lane's 8 elements sit at e0 .. e0 + 3 and e1 .. e1 + 3; in the half layout these are
// the first and the second member of its four pairs, else two times two neighbouring pairs.
template <int TI, int TO, bool INTERLEAVED, bool NORM, int AHEAD>
__global__ void __launch_bounds__(32 * kRotaryWarps) rotary_kernel(const RotaryParams p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * kRotaryWarps + (threadIdx.x >> 5);
  const long long row = w / p.warps_per_row;
  if (row >= p.rows) return;
  const int part = int(w - row * p.warps_per_row);

  const int lph = 1 << p.lanes_log2;       // lanes per head
  const int hpw = 32 >> p.lanes_log2;      // heads of a warp at a time
  const int j = lane & (lph - 1);          // lane within the head
  const int sub = lane >> p.lanes_log2;    // head of the warp
  const bool active = j * 8 < p.head_dim;
  const bool turns = j * 8 < p.rotary_dim;
  const int half = p.rotary_dim >> 1;
  int e0 = j * 8, e1 = j * 8 + 4;
  if (!INTERLEAVED && turns) {
    e0 = j * 4;
    e1 = half + j * 4;
  }

  // Rounds of hpw heads: first those of q, then those of k.  The elements of the next AHEAD rounds
  // are in flight while those of this one are turned, the first ones while the angles are made.
  const int q_rounds = (p.q_heads + hpw - 1) >> (5 - p.lanes_log2);
  const int first = part * p.rounds_per_warp;
  const int last = min(first + p.rounds_per_warp, p.rounds);
  constexpr int kIn = TI == kF32 ? 4 : TI == kE4M3 ? 1 : 2, kOut = TO == kF32 ? 4 : TO == kE4M3 ? 1 : 2;
  const char* in;
  char* out;
  auto start = [&](int it) {  // where the lane's head of round `it` is read
    in = it < q_rounds ? p.q + (row * p.q_ld + (it * hpw + sub) * p.q_hstride) * kIn
                       : p.k + (row * p.k_ld + ((it - q_rounds) * hpw + sub) * p.k_hstride) * kIn;
  };
  auto start_out = [&](int it) {
    out = it < q_rounds ? p.q_out + (row * p.q_out_ld + (long long)(it * hpw + sub) * p.head_dim) * kOut
                        : p.k_out + (row * p.k_out_ld + (long long)((it - q_rounds) * hpw + sub) * p.head_dim) * kOut;
  };
  auto there = [&](int it) {
    return active && (it < q_rounds ? it * hpw + sub < p.q_heads : (it - q_rounds) * hpw + sub < p.k_heads);
  };
  Raw4<TI> lo[AHEAD], hi[AHEAD];
  int next = first;  // the round that is loaded next
  auto load = [&](Raw4<TI>& x, Raw4<TI>& y) {
    if (next < last) {
      if (next == first || next == q_rounds) start(next);
      else in += (next < q_rounds ? p.q_hstride : p.k_hstride) * (hpw * kIn);
      if (there(next)) {
        x = load_raw4<TI>(in, e0);
        y = load_raw4<TI>(in, e1);
      }
      ++next;
    }
  };
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    lo[u] = hi[u] = Raw4<TI>{};
    load(lo[u], hi[u]);
  }

  float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
  if (turns) {
    const long long pos = p.position_bits == 64
                              ? reinterpret_cast<const long long*>(p.positions)[row]
                              : (long long)reinterpret_cast<const int*>(p.positions)[row];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long f = p.freqs[j * 4 + i];
      const int turn = int((unsigned long long)pos * f >> 32);  // signed fraction of a turn / 2^32
      sincospif(float(turn) * 0x1p-31f, &s[i], &c[i]);
      c[i] *= p.magnitude;
      s[i] *= p.inverse ? -p.magnitude : p.magnitude;
    }
  }

  float wt[8];
  start_out(first);
  for (int base = first; base < last; base += AHEAD) {
#pragma unroll
   for (int u = 0; u < AHEAD; ++u) {
    const int it = base + u;
    if (it >= last) break;
    const bool live = there(it);
    float x[8];
    unpack4<TI>(lo[u], x);
    unpack4<TI>(hi[u], x + 4);
    load(lo[u], hi[u]);
    if (NORM && (it == first || it == q_rounds)) {
      const char* weight = reinterpret_cast<const char*>(it < q_rounds ? p.q_weight : p.k_weight);
#pragma unroll
      for (int i = 0; i < 8; ++i) wt[i] = 0.f;
      if (active) {
        load4<kF32>(weight, e0, wt);
        load4<kF32>(weight, e1, wt + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) wt[i] += p.weight_offset;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= p.in_scale;
    if (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
      if (!live) sum = 0.f;
      for (int o = 1; o < lph; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float inv = rsqrtf(sum / float(p.head_dim) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * wt[i];
    }
    if (turns) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float& a = INTERLEAVED ? x[2 * i] : x[i];
        float& b = INTERLEAVED ? x[2 * i + 1] : x[i + 4];
        const float a0 = a, b0 = b;
        a = fmaf(-b0, s[i], a0 * c[i]);
        b = fmaf(a0, s[i], b0 * c[i]);
      }
    }
    if (live) {
      if (TO == kE4M3) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __fdiv_rn(x[i], p.out_scale);
      }
      store4<TO>(out, e0, x);
      store4<TO>(out, e1, x + 4);
    }
    if (it + 1 == q_rounds) start_out(it + 1);
    else out += (long long)p.head_dim * (hpw * kOut);
   }
  }
}

template <int TI, int TO>
cudaError_t launch_rotary(const RotaryParams& p, bool interleaved, cudaStream_t s) {
  const long long warps = (long long)p.rows * p.warps_per_row;
  const dim3 grid((unsigned)((warps + kRotaryWarps - 1) / kRotaryWarps));
  const dim3 block(32 * kRotaryWarps);
  constexpr int A = TI == kF32 ? 2 : 4;
  if (p.q_weight != nullptr)
    return interleaved ? launch_pdl(rotary_kernel<TI, TO, true, true, A>, grid, block, 0, s, p)
                       : launch_pdl(rotary_kernel<TI, TO, false, true, A>, grid, block, 0, s, p);
  return interleaved ? launch_pdl(rotary_kernel<TI, TO, true, false, A>, grid, block, 0, s, p)
                     : launch_pdl(rotary_kernel<TI, TO, false, false, A>, grid, block, 0, s, p);
}

template <int TI>
cudaError_t launch_rotary_to(const RotaryParams& p, int to, bool interleaved, cudaStream_t s) {
  switch (to) {
    case kF32: return launch_rotary<TI, kF32>(p, interleaved, s);
    case kBF16: return launch_rotary<TI, kBF16>(p, interleaved, s);
    case kF16: return launch_rotary<TI, kF16>(p, interleaved, s);
    default: return launch_rotary<TI, kE4M3>(p, interleaved, s);
  }
}

}  // namespace
}  // namespace b2f

extern "C" {

void b2f_rotary_args_init(b2f_rotary_args* a) {
  if (a == nullptr) return;
  *a = b2f_rotary_args{};
  a->in_dtype = a->out_dtype = B2F_DTYPE_BF16;
  a->in_scale = a->out_scale = a->magnitude = 1.0f;
  a->weight_offset = 1.0f;
  a->eps = 1e-6f;
  a->position_bits = 32;
}

int b2f_rotary(const b2f_rotary_args* a, b2f_stream_t stream) {
  using namespace b2f;
  if (a == nullptr) return fail(B2F_ERR_ARG, "rotary: null args");
  if (a->rows <= 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads + a->k_heads == 0)
    return fail(B2F_ERR_ARG, "rotary: empty shape");
  if (a->q_heads > 65536 || a->k_heads > 65536) return fail(B2F_ERR_ARG, "rotary: too many heads");
  const int d = a->head_dim;
  if (d < 8 || d > 256 || d % 8) return fail(B2F_ERR_ARG, "rotary: head_dim must be a multiple of 8 up to 256");
  if (a->rotary_dim < 8 || a->rotary_dim > d || a->rotary_dim % 8)
    return fail(B2F_ERR_ARG, "rotary: rotary_dim must be a multiple of 8 up to head_dim");
  for (int dt : {a->in_dtype, a->out_dtype})
    if (dt < B2F_DTYPE_F32 || dt > B2F_DTYPE_F16) return fail(B2F_ERR_ARG, "rotary: unknown dtype");
  if (a->position_bits != 32 && a->position_bits != 64)
    return fail(B2F_ERR_ARG, "rotary: positions are int32 or int64");
  if (a->positions == nullptr || a->freqs == nullptr)
    return fail(B2F_ERR_ARG, "rotary: null positions or frequencies");
  if ((reinterpret_cast<uintptr_t>(a->positions) % (a->position_bits / 8)) ||
      (reinterpret_cast<uintptr_t>(a->freqs) & 7))
    return fail(B2F_ERR_ARG, "rotary: misaligned positions or frequencies");
  if (!(a->out_scale > 0.0f) || !std::isfinite(a->out_scale))
    return fail(B2F_ERR_ARG, "rotary: out_scale must be > 0");
  if (a->out_dtype != B2F_DTYPE_E4M3 && a->out_scale != 1.0f)
    return fail(B2F_ERR_ARG, "rotary: out_scale belongs to an e4m3 output");
  // the weight of a side that is not there does not stand in for one that is
  if ((a->q_heads && !a->q_weight && a->k_weight) || (a->k_heads && !a->k_weight && a->q_weight))
    return fail(B2F_ERR_ARG, "rotary: q_weight and k_weight go together");
  if ((reinterpret_cast<uintptr_t>(a->q_weight) | reinterpret_cast<uintptr_t>(a->k_weight)) & 15)
    return fail(B2F_ERR_ARG, "rotary: weights must be 16-byte aligned");
  if ((a->q_weight || a->k_weight) && a->inverse)
    return fail(B2F_ERR_ARG, "rotary: the head norm has no inverse");
  const int is = a->in_dtype == B2F_DTYPE_F32 ? 4 : a->in_dtype == B2F_DTYPE_E4M3 ? 1 : 2;
  const int os = a->out_dtype == B2F_DTYPE_F32 ? 4 : a->out_dtype == B2F_DTYPE_E4M3 ? 1 : 2;
  struct Side { const void* in; long long ld, hs; void* out; long long old; int heads; };
  for (const Side& x : {Side{a->q, a->q_ld, a->q_head_stride, a->q_out, a->q_out_ld, a->q_heads},
                        Side{a->k, a->k_ld, a->k_head_stride, a->k_out, a->k_out_ld, a->k_heads}}) {
    if (x.heads == 0) continue;
    if (x.in == nullptr || x.out == nullptr) return fail(B2F_ERR_ARG, "rotary: null tensor");
    if (x.hs < d || x.hs % 8 || x.ld < (long long)(x.heads - 1) * x.hs + d ||
        x.old < (long long)x.heads * d)
      return fail(B2F_ERR_ARG, "rotary: row pitch or head stride too small, or stride not a multiple of 8");
    if (reinterpret_cast<uintptr_t>(x.in) % (4 * is) || reinterpret_cast<uintptr_t>(x.out) % (4 * os) ||
        x.ld % 4 || x.old % 4)
      return fail(B2F_ERR_ARG, "rotary: tensors and rows must be aligned to four elements");
  }
  RotaryParams p = {};
  p.rows = a->rows; p.q_heads = a->q_heads; p.k_heads = a->k_heads;
  p.head_dim = d; p.rotary_dim = a->rotary_dim;
  p.lanes_log2 = d <= 64 ? 3 : d <= 128 ? 4 : 5;
  p.inverse = a->inverse; p.position_bits = a->position_bits;
  p.q = reinterpret_cast<const char*>(a->q); p.k = reinterpret_cast<const char*>(a->k);
  p.q_ld = a->q_ld; p.q_hstride = a->q_head_stride; p.k_ld = a->k_ld; p.k_hstride = a->k_head_stride;
  p.in_scale = a->in_scale;
  p.q_weight = a->q_weight != nullptr ? a->q_weight : a->k_weight;
  p.k_weight = a->k_weight != nullptr ? a->k_weight : a->q_weight;
  p.weight_offset = a->weight_offset; p.eps = a->eps;
  p.positions = a->positions; p.freqs = a->freqs; p.magnitude = a->magnitude;
  p.q_out = reinterpret_cast<char*>(a->q_out); p.k_out = reinterpret_cast<char*>(a->k_out);
  p.q_out_ld = a->q_out_ld; p.k_out_ld = a->k_out_ld; p.out_scale = a->out_scale;
  // One warp per token where tokens fill the GPU (32 warps on each of 148 SMs); fewer tokens
  // have their heads dealt to more warps.
  const int hpw = 32 >> p.lanes_log2;
  p.rounds = (p.q_heads + hpw - 1) / hpw + (p.k_heads + hpw - 1) / hpw;
  const int want = std::max(1, std::min(p.rounds, (32 * 148 + p.rows - 1) / p.rows));
  p.rounds_per_warp = (p.rounds + want - 1) / want;
  p.warps_per_row = (p.rounds + p.rounds_per_warp - 1) / p.rounds_per_warp;
  if ((long long)p.rows * p.warps_per_row / kRotaryWarps >= 0x7fffffffll)
    return fail(B2F_ERR_ARG, "rotary: too many rows");
  cudaStream_t s = (cudaStream_t)stream;
  const bool il = a->interleaved != 0;
  switch (a->in_dtype) {
    case kF32: B2F_CUDA_TRY(launch_rotary_to<kF32>(p, a->out_dtype, il, s)); break;
    case kBF16: B2F_CUDA_TRY(launch_rotary_to<kBF16>(p, a->out_dtype, il, s)); break;
    case kF16: B2F_CUDA_TRY(launch_rotary_to<kF16>(p, a->out_dtype, il, s)); break;
    default: B2F_CUDA_TRY(launch_rotary_to<kE4M3>(p, a->out_dtype, il, s)); break;
  }
  return B2F_OK;
}

}  // extern "C"
