// Keys and values into the pages of the 4-bit cache, and back (C ABI: b2f_kv4_write,
// b2f_kv4_read; the layout stands in kv4.cuh).
//
//   s8   = e4m3(amax(|x_0..15|) / (6 * scale))        (6 = the largest e2m1 value; saturating)
//   code = e2m1(x / (s8 * scale))                     (ties to even, saturating; 0 when s8 is 0)
// The code is that of the quotient as f32 rounds it; with a scale that is a power of two the divisor
// has 4 significant bits, a quotient of a 16-bit x that is not on a border between two codes is far
// from it, and the codes are those of exact arithmetic.  A NaN makes the scale of its group NaN, an
// infinity saturates.
//
// Quotients.  With r the rounded reciprocal of s, two corrections q <- q + (x - q s) r of q = x r
// end in the rounded quotient (P. Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990: the first brings q within a unit of the last place, of such a q the
// second makes the rounded quotient; x - q s is exact in one fused multiply-add).  s lies within
// 2^-73 and 2^73, quotients that matter within 1/8 and 16: nothing leaves the range of f32; below 1/8
// only the sign of q matters, which is taken from x.  Groups whose scale saturates, where quotients
// have no bound, are divided one by one.
//
// Bound: memory.  One lane owns one group: 32 bytes of 16-bit input in, 8 bytes of codes and
// a scale byte out; a warp owns a token (its place is found once, all lanes alike) and runs
// over its groups, K heads then V heads, neighbouring lanes on neighbouring groups.
//
// Measured: 4251 tokens of four prompts, bf16, 8 kv heads of head_dim 128 (22 MB): written and read
// back 16.0 us, written alone 7.5 (7.3 from e4m3), read alone 7.7; 16 IEEE divisions a group in place of
// the corrections cost 4 more.  Nothing is full: the write has half of its issue slots busy, the read
// a third, with 38 % of the warps, which wait for their loads.  24 single tokens, both calls:
// 4.4 us, of launches and two dependent loads (a token's sequence, its page).
#include <algorithm>
#include <cmath>
#include <string>

#include "common.cuh"
#include "host_common.h"
#include "convert.cuh"
#include "kv4.cuh"

namespace b2f {

const char* kv4_check_cache(const b2f_kv4_cache& c, Kv4Cache* o) {
  if (c.storage == nullptr || c.table == nullptr || c.lens == nullptr) return "null cache buffer";
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return "head_dim must be 64, 128 or 256";
  if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64) return "page_size must be 16, 32 or 64";
  if (c.pages <= 0 || c.kv_heads <= 0 || c.kv_heads > 1024) return "empty cache, or more than 1024 kv heads";
  if (c.table_rows <= 0 || c.table_cols <= 0 || c.table_ld < c.table_cols) return "table shape";
  if ((long long)c.table_cols * c.page_size > 0x3fffffffll) return "a table row holds at most 2^30 tokens";
  const int block = c.page_size * c.head_dim / 8 * 9;
  if (c.page_stride < (long long)block * c.kv_heads || c.page_stride % 16)
    return "page_stride smaller than a page, or not a multiple of 16";
  if (reinterpret_cast<uintptr_t>(c.storage) & 15) return "storage must be 16-byte aligned";
  if ((reinterpret_cast<uintptr_t>(c.table) | reinterpret_cast<uintptr_t>(c.lens)) & 3)
    return "misaligned table or lens";
  for (float s : {c.k_scale, c.v_scale})
    if (!(s >= 0x1p-64f && s <= 0x1p64f)) return "k_scale and v_scale must lie in [2^-64, 2^64]";
  *o = Kv4Cache{reinterpret_cast<uint8_t*>(c.storage), c.page_stride, c.pages, c.kv_heads,
                c.head_dim, c.page_size, c.k_scale, c.v_scale, c.table, c.table_rows,
                c.table_cols, c.table_ld, c.lens, 0, 0, 0, 0};
  o->page_log2 = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : 6;
  o->block_bytes = block;
  o->codes_bytes = c.page_size * c.head_dim / 2;
  o->scales_bytes = c.page_size * c.head_dim / 16;
  return nullptr;
}

const char* kv4_check_batch(const b2f_kv4_cache& c, const b2f_kv4_batch& b, Kv4Batch* o) {
  if (b.seqs <= 0 || b.tokens <= 0) return "empty batch";
  if (b.starts == nullptr && b.tokens % b.seqs) return "without starts, tokens must be a multiple of seqs";
  if (b.rows == nullptr && b.seqs > c.table_rows) return "more sequences than table rows";
  if ((reinterpret_cast<uintptr_t>(b.rows) | reinterpret_cast<uintptr_t>(b.starts)) & 3)
    return "misaligned rows or starts";
  *o = Kv4Batch{b.seqs, b.tokens, b.rows, b.starts, b.starts == nullptr ? b.tokens / b.seqs : 0};
  return nullptr;
}

namespace {

struct Kv4MoveParams {
  Kv4Cache c;
  Kv4Batch b;
  const char* k;
  const char* v;
  char* k_out;
  char* v_out;
  long long k_ld, v_ld;
  float k_in, v_in;
  int warps_per_token;
  int groups_log2;  // of the groups of 16 of a head
};

constexpr int kMoveWarps = 4;

__device__ __forceinline__ uint32_t e2m1x8(const float* y) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  return r;
}

// The largest magnitude of three; NaN when one of them is.
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// x / s as f32 rounds it, for |x| < 16 s and 2^-73 <= s <= 2^73 (see above; |q| < 1/8: about).
__device__ __forceinline__ void divide16(float (&x)[16], float s) {
  const float r = __frcp_rn(s);
  const float2 r2 = make_float2(r, r), minus_s = make_float2(-s, -s);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const float2 v = make_float2(x[i], x[i + 1]);
    float2 q = fmul2(v, r2);
    q = ffma2(ffma2(q, minus_s, v), r2, q);
    q = ffma2(ffma2(q, minus_s, v), r2, q);
    x[i] = copysignf(q.x, v.x);
    x[i + 1] = copysignf(q.y, v.y);
  }
}

// Where group g of a token lies: K (0) or V (1), the kv head, the group within the head.
struct Kv4Group {
  int part, head, in_head;
};
__device__ __forceinline__ Kv4Group kv4_group(const Kv4MoveParams& p, int g) {
  const int half = p.c.kv_heads << p.groups_log2;
  Kv4Group r;
  r.part = g >= half;
  const int x = g - (r.part ? half : 0);
  r.head = x >> p.groups_log2;
  r.in_head = x & ((1 << p.groups_log2) - 1);
  return r;
}
__device__ __forceinline__ long long kv4_element(const Kv4MoveParams& p, int t, const Kv4Group& at) {
  return (long long)t * (at.part ? p.v_ld : p.k_ld) + at.head * p.c.head_dim + at.in_head * 16;
}
__device__ __forceinline__ uint8_t* kv4_block(const Kv4Cache& c, int page, const Kv4Group& at) {
  return c.storage + (long long)page * c.page_stride + (long long)at.head * c.block_bytes +
         at.part * (c.codes_bytes + c.scales_bytes);
}

template <int DT>
__global__ void __launch_bounds__(32 * kMoveWarps, 8) kv4_write_kernel(const Kv4MoveParams p) {
  // Groups of a lane in flight.  Four, with the registers that they take (109), leave room for half the
  // warps: 16.5 us for the prompts above against 16.0.
  constexpr int N = DT == kF32 ? 1 : 2;
  pdl_wait();
  pdl_trigger();
  const long long w = (long long)blockIdx.x * kMoveWarps + (threadIdx.x >> 5);
  const int t = int(w / p.warps_per_token);
  if (t >= p.b.tokens) return;
  const Kv4Cache& c = p.c;
  const int groups = 2 * c.kv_heads << p.groups_log2, step = 32 * p.warps_per_token;
  int g0 = int(w - (long long)t * p.warps_per_token) * 32 + (threadIdx.x & 31);
  Raw16<DT> raw[N];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (g0 + u * step < groups) {
        const Kv4Group at = kv4_group(p, g0 + u * step);
        raw[u] = load_raw16<DT>(at.part ? p.v : p.k, kv4_element(p, t, at));
      }
  };
  load();  // in flight while the token's place is looked up
  int slot;
  const int page = kv4_place(p.c, p.b, t, slot);
  if (page < 0) return;
  while (true) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (g0 + u * step >= groups) break;
      const Kv4Group at = kv4_group(p, g0 + u * step);
      float x[16];
      unpack16<DT>(raw[u], x);
      const float in = at.part ? p.v_in : p.k_in, scale = at.part ? c.v_scale : c.k_scale;
      const float2 in2 = make_float2(in, in);
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float2 y = fmul2(make_float2(x[i], x[i + 1]), in2);
        x[i] = y.x;
        x[i + 1] = y.y;
        top = max3_abs_nan(top, y.x, y.y);
      }
      const uint16_t s8 = f32x2_to_e4m3x2(__fdiv_rn(top, 6.0f * scale), 0.f) & 0xff;
      const float s = e4m3_to_f32(uint8_t(s8)) * scale;
      if (s > 0.f && s8 < 0x7e) {
        divide16(x, s);
      } else {  // 0, NaN, or the largest scale, which may have been saturated
        const bool some = s > 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = some ? __fdiv_rn(x[i], s) : 0.f;
      }
      uint8_t* block = kv4_block(c, page, at);
      *reinterpret_cast<uint2*>(block + slot * (c.head_dim >> 1) + at.in_head * 8) =
          make_uint2(e2m1x8(x), e2m1x8(x + 8));
      block[c.codes_bytes + slot * (c.head_dim >> 4) + at.in_head] = uint8_t(s8);
    }
    g0 += N * step;
    if (g0 >= groups) return;
    load();
  }
}

template <int DT>
__global__ void __launch_bounds__(32 * kMoveWarps) kv4_read_kernel(const Kv4MoveParams p) {
  constexpr int N = 4;  // groups of a lane in flight
  pdl_wait();
  pdl_trigger();
  const long long w = (long long)blockIdx.x * kMoveWarps + (threadIdx.x >> 5);
  const int t = int(w / p.warps_per_token);
  if (t >= p.b.tokens) return;
  int slot;
  const int page = kv4_place(p.c, p.b, t, slot);
  if (page == -2) return;
  const Kv4Cache& c = p.c;
  const int groups = 2 * c.kv_heads << p.groups_log2, step = 32 * p.warps_per_token;
  for (int g0 = int(w - (long long)t * p.warps_per_token) * 32 + (threadIdx.x & 31); g0 < groups; g0 += N * step) {
    uint2 codes[N];
    uint8_t s8[N];
#pragma unroll
    for (int u = 0; u < N; ++u) {
      codes[u] = make_uint2(0, 0);
      s8[u] = 0;
      if (page >= 0 && g0 + u * step < groups) {
        const Kv4Group at = kv4_group(p, g0 + u * step);
        const uint8_t* block = kv4_block(c, page, at);
        codes[u] = *reinterpret_cast<const uint2*>(block + slot * (c.head_dim >> 1) + at.in_head * 8);
        s8[u] = block[c.codes_bytes + slot * (c.head_dim >> 4) + at.in_head];
      }
    }
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (g0 + u * step >= groups) break;
      const Kv4Group at = kv4_group(p, g0 + u * step);
      const float s = e4m3_to_f32(s8[u]) * (at.part ? c.v_scale : c.k_scale);
      float x[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t f[4];
        e2m1x8_to_f16x2(h ? codes[u].y : codes[u].x, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 v = unpack_f16x2(f[i]);
          x[8 * h + 2 * i] = v.x * s;
          x[8 * h + 2 * i + 1] = v.y * s;
        }
      }
      store16<DT>(at.part ? p.v_out : p.k_out, kv4_element(p, t, at), x);
    }
  }
}

int elem_bytes(int dt) { return dt == B2F_DTYPE_F32 ? 4 : dt == B2F_DTYPE_E4M3 ? 1 : 2; }

// Fills p and the grid; nullptr when the arguments are fine.
const char* prepare_move(const b2f_kv4_cache& c, const b2f_kv4_batch& b, const void* k, long long k_ld,
                         const void* v, long long v_ld, int dtype, Kv4MoveParams* p, dim3* grid) {
  if (const char* e = kv4_check_cache(c, &p->c)) return e;
  if (const char* e = kv4_check_batch(c, b, &p->b)) return e;
  if (k == nullptr || v == nullptr) return "null tensor";
  const long long cols = (long long)c.kv_heads * c.head_dim;
  const int es = elem_bytes(dtype);
  for (long long ld : {k_ld, v_ld})
    if (ld < cols || (ld * es) % 16) return "row pitch smaller than kv_heads * head_dim, or rows not 16-byte aligned";
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)
    return "tensors must be 16-byte aligned";
  p->k_ld = k_ld;
  p->v_ld = v_ld;
  p->groups_log2 = c.head_dim == 64 ? 2 : c.head_dim == 128 ? 3 : 4;
  // A warp a token once there are enough of them (8 for each of 148 SMs); fewer tokens have
  // their groups dealt to more warps, one round of 32 groups at the least.
  const int rounds = (int)((2 * cols / 16 + 31) / 32);
  p->warps_per_token = std::max(1, std::min(rounds, (8 * 148 + b.tokens - 1) / b.tokens));
  const long long ctas = ((long long)b.tokens * p->warps_per_token + kMoveWarps - 1) / kMoveWarps;
  if (ctas > 0x7fffffffll) return "too many tokens";
  *grid = dim3((unsigned)ctas);
  return nullptr;
}

}  // namespace
}  // namespace b2f

extern "C" {

void b2f_kv4_write_args_init(b2f_kv4_write_args* a) {
  if (a == nullptr) return;
  *a = b2f_kv4_write_args{};
  a->dtype = B2F_DTYPE_BF16;
  a->k_in_scale = a->v_in_scale = 1.0f;
  a->cache.k_scale = a->cache.v_scale = 1.0f;
}

int b2f_kv4_write(const b2f_kv4_write_args* a, b2f_stream_t stream) {
  using namespace b2f;
  if (a == nullptr) return fail(B2F_ERR_ARG, "kv4_write: null args");
  if (a->dtype < B2F_DTYPE_F32 || a->dtype > B2F_DTYPE_F16) return fail(B2F_ERR_ARG, "kv4_write: unknown dtype");
  Kv4MoveParams p = {};
  dim3 grid;
  if (const char* e = prepare_move(a->cache, a->batch, a->k, a->k_ld, a->v, a->v_ld, a->dtype, &p, &grid))
    return fail(B2F_ERR_ARG, std::string("kv4_write: ") + e);
  p.k = reinterpret_cast<const char*>(a->k);
  p.v = reinterpret_cast<const char*>(a->v);
  p.k_in = a->k_in_scale;
  p.v_in = a->v_in_scale;
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 block(32 * kMoveWarps);
  switch (a->dtype) {
    case kF32: B2F_CUDA_TRY(launch_pdl(kv4_write_kernel<kF32>, grid, block, 0, s, p)); break;
    case kBF16: B2F_CUDA_TRY(launch_pdl(kv4_write_kernel<kBF16>, grid, block, 0, s, p)); break;
    case kF16: B2F_CUDA_TRY(launch_pdl(kv4_write_kernel<kF16>, grid, block, 0, s, p)); break;
    default: B2F_CUDA_TRY(launch_pdl(kv4_write_kernel<kE4M3>, grid, block, 0, s, p)); break;
  }
  return B2F_OK;
}

void b2f_kv4_read_args_init(b2f_kv4_read_args* a) {
  if (a == nullptr) return;
  *a = b2f_kv4_read_args{};
  a->dtype = B2F_DTYPE_BF16;
  a->cache.k_scale = a->cache.v_scale = 1.0f;
}

int b2f_kv4_read(const b2f_kv4_read_args* a, b2f_stream_t stream) {
  using namespace b2f;
  if (a == nullptr) return fail(B2F_ERR_ARG, "kv4_read: null args");
  if (a->dtype != B2F_DTYPE_F32 && a->dtype != B2F_DTYPE_BF16 && a->dtype != B2F_DTYPE_F16)
    return fail(B2F_ERR_ARG, "kv4_read: out must be f32, bf16 or f16");
  Kv4MoveParams p = {};
  dim3 grid;
  if (const char* e = prepare_move(a->cache, a->batch, a->k, a->k_ld, a->v, a->v_ld, a->dtype, &p, &grid))
    return fail(B2F_ERR_ARG, std::string("kv4_read: ") + e);
  p.k_out = reinterpret_cast<char*>(a->k);
  p.v_out = reinterpret_cast<char*>(a->v);
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 block(32 * kMoveWarps);
  switch (a->dtype) {
    case kF32: B2F_CUDA_TRY(launch_pdl(kv4_read_kernel<kF32>, grid, block, 0, s, p)); break;
    case kBF16: B2F_CUDA_TRY(launch_pdl(kv4_read_kernel<kBF16>, grid, block, 0, s, p)); break;
    default: B2F_CUDA_TRY(launch_pdl(kv4_read_kernel<kF16>, grid, block, 0, s, p)); break;
  }
  return B2F_OK;
}

}  // extern "C"
