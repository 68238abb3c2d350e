// The pages of the 4-bit cache: handing out, forking, freeing, compacting, copying (C ABI:
// b2f_kv4_extend / _fork / _free / _compact / _copy_pages).
//
// refs[page] counts the table rows that use a page; a page is free exactly when its count is
// 0, and the free page with the lowest number is always taken first.  There is no free list
// to keep in order: counts are changed by integer atomics, so results do not depend on the
// order in which threads run, and a call captured in a graph does the same on every replay.
//
// A call that cannot be carried out (a row out of range, listed twice, a fork onto a row in
// use, a full table row, too few free pages) changes nothing and records B2F_DEV_BAD_ARGS or
// B2F_DEV_NO_PAGES in the device status word.
//
// extend, and the first half of fork and compact, are one CTA of 1024 threads: they read
// refs once or twice (4 bytes a page, 16 pages a thread in flight; once where the pool is at most
// 16384 pages: fork 12.1 -> 11.1 us, compact 46.7 -> 43.9) and are bound by latency.
// The pages themselves are moved by a second kernel, a warp for 2 KB, bound by memory.
//
// Measured (device time, 8 kv heads of head_dim 128, pages of 16 tokens, 4 layers): compact of a
// pool of 6000 pages 43.9 us: 6 for the plan, 28.5 for moving 100 MB (7.0 TB/s read and written:
// some of it stays in the L2 cache), the rest the rewriting of tables and two launches; fork of 8
// sequences of up to 1500 tokens eight times 11.1 us, 7.5 of them the plan: a chain of a few
// dependent loads and barriers; extend of 64 rows by a token 3.3 us with 8192 pages, 3.8 with 65536.
#include <algorithm>
#include <new>
#include <string>
#include <vector>

#include "common.cuh"
#include "host_common.h"

namespace b2f {
namespace {

struct Pool {
  uint8_t* storage;
  long long layer_stride, page_stride;
  int layers, pages, page_log2, page_bytes;
  int* table;
  int table_rows, table_cols;
  long long table_ld;
  int* lens;
  int* refs;
};

constexpr int kPlanThreads = 1024;
constexpr int kPerThread = 16;  // pages of a thread in one round of a scan
constexpr int kMaxRows = 1024;  // rows of one call (a thread each)

// Exclusive prefix of v over the CTA, and its total; `scratch` holds 33 ints.
__device__ __forceinline__ int block_scan(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // scratch may still be read from the call before
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = scratch[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    scratch[lane] = s;
  }
  __syncthreads();
  total = scratch[31];
  return x - v + (warp ? scratch[warp - 1] : 0);
}

// Bit i set: page first + i is free (of the kPerThread pages of this thread, in a round that
// starts at `base`).
__device__ __forceinline__ unsigned free_bits(const Pool& p, int base) {
  const int first = base + (int)threadIdx.x * kPerThread;
  unsigned bits = 0;
  if (first + kPerThread <= p.pages && (reinterpret_cast<uintptr_t>(p.refs) & 15) == 0) {
    const int4* v = reinterpret_cast<const int4*>(p.refs + first);
#pragma unroll
    for (int i = 0; i < kPerThread / 4; ++i) {
      const int4 a = v[i];
      bits |= (unsigned(a.x == 0) | unsigned(a.y == 0) << 1 | unsigned(a.z == 0) << 2 |
               unsigned(a.w == 0) << 3) << (4 * i);
    }
  } else {
    for (int i = 0; i < kPerThread; ++i)
      if (first + i < p.pages && p.refs[first + i] == 0) bits |= 1u << i;
  }
  return bits;
}

// Hands the `need` lowest free pages to take(rank, page), rank 0 .. need - 1, and returns true;
// returns false and takes none when there are fewer.  All threads of the CTA call it.
template <typename Take>
__device__ __forceinline__ bool take_free(const Pool& p, int need, int* scratch, Take take) {
  constexpr int kRound = kPlanThreads * kPerThread;
  const unsigned bits0 = free_bits(p, 0);  // of the first round, often the only one
  int total0;
  const int rank0 = block_scan(__popc(bits0), scratch, total0);
  int found = total0;
  for (int base = kRound; base < p.pages && found < need; base += kRound) {
    int total;
    block_scan(__popc(free_bits(p, base)), scratch, total);
    found += total;
  }
  if (found < need) return false;
  int rank = 0;
  for (int base = 0; base < p.pages && rank < need; base += kRound) {
    unsigned bits = bits0;
    int total = total0, r = rank0;
    if (base > 0) {
      bits = free_bits(p, base);
      r = rank + block_scan(__popc(bits), scratch, total);
    }
    for (; bits != 0 && r < need; bits &= bits - 1, ++r)
      take(r, base + (int)threadIdx.x * kPerThread + __ffs(bits) - 1);
    rank += total;
  }
  return true;
}

// Whether rows[i] of any thread i < n equals this thread's (i itself apart).
__device__ __forceinline__ bool listed_twice(const int* rows, int n, int mine) {
  bool twice = false;
  for (int j = 0; j < n; ++j) twice |= j != (int)threadIdx.x && rows[j] == mine;
  return twice;
}

__global__ void __launch_bounds__(kPlanThreads) kv4_extend_kernel(const Pool p, const int* rows,
                                                                  const int* counts, int n) {
  pdl_wait();
  pdl_trigger();
  __shared__ int scratch[33], row_of[kMaxRows], first[kMaxRows + 1], have[kMaxRows];
  const int i = threadIdx.x, page = 1 << p.page_log2;
  int row = -1, len = 0, more = 0, need = 0;
  bool bad = false;
  if (i < n) {
    row = rows != nullptr ? rows[i] : i;
    row_of[i] = row;
    bad = row < 0 || row >= p.table_rows;
  }
  __syncthreads();
  if (i < n && !bad) {
    len = p.lens[row];
    more = counts[i];
    bad = len < 0 || more < 0 || (long long)len + more > ((long long)p.table_cols << p.page_log2) ||
          (rows != nullptr && listed_twice(row_of, n, row));
    have[i] = (int)(((long long)len + page - 1) >> p.page_log2);
    need = bad ? 0 : (int)(((long long)len + more + page - 1) >> p.page_log2) - have[i];
  }
  if (__syncthreads_or(bad)) {
    if (i == 0) record_error(kDevBadArgs);
    return;
  }
  // a pool has at most 2^20 pages: 1024 needs, each cut off just above, sum up to less than 2^31
  int total;
  const int at = block_scan(min(need, p.pages + 1), scratch, total);
  if (i < n) first[i] = at;
  const bool too_many = __syncthreads_or(total < 0 || total > p.pages);
  const bool done = !too_many && take_free(p, total, scratch, [&](int rank, int pg) {
    int lo = 0, hi = n;  // the row with first[row] <= rank < first[row + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= rank) lo = mid;
      else hi = mid;
    }
    p.table[(long long)row_of[lo] * p.table_ld + have[lo] + rank - first[lo]] = pg;
    p.refs[pg] = 1;
  });
  if (!done) {
    if (i == 0) record_error(kDevNoPages);
    return;
  }
  if (i < n) p.lens[row] = len + more;
}

__global__ void __launch_bounds__(256) kv4_free_kernel(const Pool p, const int* rows) {
  pdl_wait();
  pdl_trigger();
  __shared__ int len;
  const int row = rows != nullptr ? rows[blockIdx.x] : (int)blockIdx.x;
  if (row < 0 || row >= p.table_rows) {
    if (threadIdx.x == 0) record_error(kDevBadArgs);
    return;
  }
  // the exchange lets a row that is listed twice be let go once
  if (threadIdx.x == 0) len = atomicExch(&p.lens[row], 0);
  __syncthreads();
  const long long page = 1 << p.page_log2;
  const int used = (int)min((max(len, 0) + page - 1) >> p.page_log2, (long long)p.table_cols);
  int* mine = p.table + (long long)row * p.table_ld;
  for (int c = threadIdx.x; c < used; c += 256) {
    const int pg = mine[c];
    mine[c] = -1;
    if (pg < 0 || pg >= p.pages) {
      record_error(kDevBadArgs);
    } else if (atomicSub(&p.refs[pg], 1) <= 0) {  // was free already: the lists disagree
      atomicAdd(&p.refs[pg], 1);
      record_error(kDevBadArgs);
    }
  }
}

// Copies pages src(k) -> dst(k), k < n, of all layers, a warp for 2 KB; dst(k) < 0: none.
template <typename Pair>
__device__ __forceinline__ void copy_pages(const Pool& p, int n, Pair pair) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
  const int slices = (p.page_bytes + 2047) >> 11;
  const long long per = (long long)p.layers * slices, total = n * per;
  for (long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total; w += warps) {
    const int k = (int)(w / per);
    const int rest = (int)(w - k * per), layer = rest / slices, at = (rest - layer * slices) << 11;
    int src, dst;
    pair(k, src, dst);
    if (src < 0 || dst < 0 || src >= p.pages || dst >= p.pages) continue;
    const uint8_t* from = p.storage + layer * p.layer_stride + src * p.page_stride + at;
    uint8_t* to = p.storage + layer * p.layer_stride + dst * p.page_stride + at;
    const int bytes = min(2048, p.page_bytes - at);
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int o = (i * 32 + lane) * 16;
      if (o < bytes) v[i] = __ldcs(reinterpret_cast<const uint4*>(from + o));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int o = (i * 32 + lane) * 16;
      if (o < bytes) *reinterpret_cast<uint4*>(to + o) = v[i];
    }
  }
}

// fork, first half: a fresh page for every child whose parent's last page is not full.
// plan[0]: 1 when the call can be carried out; plan[1 + i]: child i's fresh page or -1.
__global__ void __launch_bounds__(kPlanThreads) kv4_fork_plan_kernel(const Pool p, const int* src,
                                                                     const int* dst, int n, int* plan) {
  pdl_wait();
  pdl_trigger();
  __shared__ int scratch[33], to[kMaxRows], owner[kMaxRows];
  const int i = threadIdx.x;
  int from = -1, mine = -1, len = 0;
  bool bad = false;
  if (i < n) {
    from = src[i];
    mine = dst[i];
    to[i] = mine;
    plan[1 + i] = -1;
    bad = from < 0 || from >= p.table_rows || mine < 0 || mine >= p.table_rows;
  }
  __syncthreads();
  if (i < n && !bad) {
    len = p.lens[from];
    bad = len < 0 || len > ((long long)p.table_cols << p.page_log2) || p.lens[mine] != 0 ||
          listed_twice(to, n, mine);
    for (int j = 0; j < n; ++j) bad |= to[j] == from;  // no row is both parent and child
  }
  if (__syncthreads_or(bad)) {
    if (i == 0) {
      plan[0] = 0;
      record_error(kDevBadArgs);
    }
    return;
  }
  const int part = i < n && (len & ((1 << p.page_log2) - 1)) != 0;
  int total;
  const int at = block_scan(part, scratch, total);
  if (part) owner[at] = i;
  __syncthreads();
  const bool done = take_free(p, total, scratch, [&](int rank, int pg) {
    plan[1 + owner[rank]] = pg;
    p.refs[pg] = 1;
  });
  if (i == 0) {
    plan[0] = done;
    if (!done) record_error(kDevNoPages);
  }
  if (done && i < n) p.lens[mine] = len;
}

// fork, second half: the children's table rows, the counts of the shared pages, and the copies
// of the pages that are not full.
__global__ void __launch_bounds__(256) kv4_fork_kernel(const Pool p, const int* src, const int* dst,
                                                       int n, const int* plan) {
  pdl_wait();
  pdl_trigger();
  if (plan[0] == 0) return;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int full = p.lens[src[i]] >> p.page_log2, fresh = plan[1 + i];
    const int* from = p.table + (long long)src[i] * p.table_ld;
    int* to = p.table + (long long)dst[i] * p.table_ld;
    for (int c = threadIdx.x; c < full; c += 256) {
      const int pg = from[c];
      to[c] = pg;
      if (pg >= 0 && pg < p.pages) atomicAdd(&p.refs[pg], 1);
      else record_error(kDevBadArgs);
    }
    if (threadIdx.x == 0 && fresh >= 0) to[full] = fresh;
  }
  copy_pages(p, n, [&](int k, int& s, int& d) {
    d = plan[1 + k];
    s = d < 0 ? -1 : p.table[(long long)src[k] * p.table_ld + (p.lens[src[k]] >> p.page_log2)];
  });
}

// compact, first half: with L pages in use, the i-th used page at or behind L moves into the
// i-th free page before L.  plan: [L, moves, remap[pages], from[pages / 2 + 1], to[...]].
__global__ void __launch_bounds__(kPlanThreads) kv4_compact_plan_kernel(const Pool p, int* plan) {
  pdl_wait();
  pdl_trigger();
  __shared__ int scratch[33];
  constexpr int kRound = kPlanThreads * kPerThread;
  int* remap = plan + 2;
  int* from = remap + p.pages;
  int* to = from + p.pages / 2 + 1;
  const unsigned bits0 = free_bits(p, 0);  // of the first round, often the only one
  int live = p.pages;
  for (int base = 0; base < p.pages; base += kRound) {
    int total;
    block_scan(__popc(base == 0 ? bits0 : free_bits(p, base)), scratch, total);
    live -= total;
  }
  for (int pg = live + (int)threadIdx.x; pg < p.pages; pg += kPlanThreads) remap[pg] = pg;
  int holes = 0, moves = 0;
  for (int base = 0; base < p.pages; base += kRound) {
    const int first = base + (int)threadIdx.x * kPerThread;
    const unsigned bits = base == 0 ? bits0 : free_bits(p, base);
    const unsigned there = (1u << max(0, min(p.pages - first, kPerThread))) - 1;
    const unsigned front = (1u << max(0, min(live - first, kPerThread))) - 1;  // pages before L
    unsigned hole = bits & front, move = ~bits & there & ~front;
    int total;  // of both, at most 2^14 in a round, in one scan
    const int before = block_scan(__popc(hole) | __popc(move) << 16, scratch, total);
    int r = holes + (before & 0xffff);
    holes += total & 0xffff;
    for (; hole != 0; hole &= hole - 1) to[r++] = first + __ffs(hole) - 1;
    r = moves + (before >> 16);
    moves += total >> 16;
    for (; move != 0; move &= move - 1) from[r++] = first + __ffs(move) - 1;
  }
  __syncthreads();  // from and to are read by other threads than wrote them
  for (int k = threadIdx.x; k < moves; k += kPlanThreads) {
    const int a = from[k], b = to[k];
    remap[a] = b;
    p.refs[b] = p.refs[a];
    p.refs[a] = 0;
  }
  if (threadIdx.x == 0) {
    plan[0] = live;
    plan[1] = moves;
  }
}

__global__ void __launch_bounds__(256) kv4_compact_kernel(const Pool p, const int* plan) {
  pdl_wait();
  pdl_trigger();
  const int live = plan[0], moves = plan[1];
  if (moves == 0) return;
  const int* remap = plan + 2;
  const int* from = remap + p.pages;
  const int* to = from + p.pages / 2 + 1;
  for (int row = blockIdx.x; row < p.table_rows; row += gridDim.x) {
    const long long len = max(p.lens[row], 0);
    const int used = (int)min((len + (1 << p.page_log2) - 1) >> p.page_log2, (long long)p.table_cols);
    int* mine = p.table + (long long)row * p.table_ld;
    for (int c = threadIdx.x; c < used; c += 256) {
      const int pg = mine[c];
      if (pg >= live && pg < p.pages) mine[c] = remap[pg];
    }
  }
  copy_pages(p, moves, [&](int k, int& s, int& d) {
    s = from[k];
    d = to[k];
  });
}

constexpr int kPairsPerLaunch = 256;
struct PagePairs {
  int src[kPairsPerLaunch], dst[kPairsPerLaunch];
};

__global__ void __launch_bounds__(256) kv4_copy_pages_kernel(const Pool p, const __grid_constant__ PagePairs pairs, int n) {
  pdl_wait();
  pdl_trigger();
  copy_pages(p, n, [&](int k, int& s, int& d) {
    s = pairs.src[k];
    d = pairs.dst[k];
  });
}

const char* check_pool(const b2f_kv4_pool* a, Pool* o) {
  if (a == nullptr) return "null args";
  if (a->storage == nullptr || a->table == nullptr || a->lens == nullptr || a->refs == nullptr)
    return "null pool buffer";
  if (a->page_size != 16 && a->page_size != 32 && a->page_size != 64) return "page_size must be 16, 32 or 64";
  if (a->layers <= 0 || a->pages <= 0 || a->pages > (1 << 20)) return "empty pool, or more than 2^20 pages";
  if (a->table_rows <= 0 || a->table_cols <= 0 || a->table_ld < a->table_cols) return "table shape";
  if ((long long)a->table_cols * a->page_size > 0x3fffffffll) return "a table row holds at most 2^30 tokens";
  if (a->page_bytes <= 0 || a->page_bytes % 16 || a->page_stride < a->page_bytes || a->page_stride % 16)
    return "page_bytes and page_stride must be multiples of 16, the stride no smaller than a page";
  if (a->layers > 1 && (a->layer_stride < 0 || a->layer_stride % 16)) return "layer_stride must be a multiple of 16";
  if (reinterpret_cast<uintptr_t>(a->storage) & 15) return "storage must be 16-byte aligned";
  if ((reinterpret_cast<uintptr_t>(a->table) | reinterpret_cast<uintptr_t>(a->lens) |
       reinterpret_cast<uintptr_t>(a->refs)) & 3)
    return "misaligned table, lens or refs";
  *o = Pool{reinterpret_cast<uint8_t*>(a->storage), a->layer_stride, a->page_stride, a->layers, a->pages,
            a->page_size == 16 ? 4 : a->page_size == 32 ? 5 : 6, a->page_bytes, a->table, a->table_rows,
            a->table_cols, a->table_ld, a->lens, a->refs};
  return nullptr;
}

const char* check_rows(const Pool& p, const void* rows, int n, bool may_be_all) {
  if (n <= 0 || n > kMaxRows) return "a call takes 1 to 1024 rows";
  if (rows == nullptr && !may_be_all) return "null rows";
  if (rows == nullptr && n > p.table_rows) return "more rows than the table has";
  if (reinterpret_cast<uintptr_t>(rows) & 3) return "misaligned rows";
  return nullptr;
}

// CTAs of a page copy: a warp for each 2 KB, at most what fills the GPU (8 CTAs on an SM).
unsigned copy_grid(const Pool& p, long long pairs) {
  const long long warps = pairs * p.layers * ((p.page_bytes + 2047) / 2048);
  return (unsigned)std::max(1ll, std::min((warps + 7) / 8, (long long)std::max(sm_count(), 1) * 8));
}

}  // namespace
}  // namespace b2f

extern "C" {

long long b2f_kv4_fork_workspace_bytes(int n) { return n < 0 ? 0 : 4ll * (n + 1); }

long long b2f_kv4_compact_workspace_bytes(int pages) {
  return pages < 0 ? 0 : 4ll * (2 + (long long)pages + 2ll * (pages / 2 + 1));
}

int b2f_kv4_extend(const b2f_kv4_pool* pool, const int* rows, const int* counts, int n, b2f_stream_t stream) {
  using namespace b2f;
  Pool p;
  const char* e = check_pool(pool, &p);
  if (e == nullptr) e = check_rows(p, rows, n, true);
  if (e == nullptr) e = check_rows(p, counts, n, false);
  if (e != nullptr) return fail(B2F_ERR_ARG, std::string("kv4_extend: ") + e);
  B2F_CUDA_TRY(launch_pdl(kv4_extend_kernel, dim3(1), dim3(kPlanThreads), 0, (cudaStream_t)stream, p, rows, counts, n));
  return B2F_OK;
}

int b2f_kv4_free(const b2f_kv4_pool* pool, const int* rows, int n, b2f_stream_t stream) {
  using namespace b2f;
  Pool p;
  const char* e = check_pool(pool, &p);
  if (e == nullptr) e = check_rows(p, rows, n, true);
  if (e != nullptr) return fail(B2F_ERR_ARG, std::string("kv4_free: ") + e);
  B2F_CUDA_TRY(launch_pdl(kv4_free_kernel, dim3((unsigned)n), dim3(256), 0, (cudaStream_t)stream, p, rows));
  return B2F_OK;
}

int b2f_kv4_fork(const b2f_kv4_pool* pool, const int* src, const int* dst, int n, void* workspace,
                 long long workspace_bytes, b2f_stream_t stream) {
  using namespace b2f;
  Pool p;
  const char* e = check_pool(pool, &p);
  if (e == nullptr) e = check_rows(p, src, n, false);
  if (e == nullptr) e = check_rows(p, dst, n, false);
  if (e == nullptr && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 3) ||
                       workspace_bytes < b2f_kv4_fork_workspace_bytes(n)))
    e = "workspace too small or misaligned";
  if (e != nullptr) return fail(B2F_ERR_ARG, std::string("kv4_fork: ") + e);
  cudaStream_t s = (cudaStream_t)stream;
  int* plan = reinterpret_cast<int*>(workspace);
  B2F_CUDA_TRY(launch_pdl(kv4_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, src, dst, n, plan));
  B2F_CUDA_TRY(launch_pdl(kv4_fork_kernel, dim3(copy_grid(p, n)), dim3(256), 0, s, p, src, dst, n, (const int*)plan));
  return B2F_OK;
}

int b2f_kv4_compact(const b2f_kv4_pool* pool, void* workspace, long long workspace_bytes, b2f_stream_t stream) {
  using namespace b2f;
  Pool p;
  const char* e = check_pool(pool, &p);
  if (e == nullptr && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 3) ||
                       workspace_bytes < b2f_kv4_compact_workspace_bytes(p.pages)))
    e = "workspace too small or misaligned";
  if (e != nullptr) return fail(B2F_ERR_ARG, std::string("kv4_compact: ") + e);
  cudaStream_t s = (cudaStream_t)stream;
  int* plan = reinterpret_cast<int*>(workspace);
  B2F_CUDA_TRY(launch_pdl(kv4_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p, plan));
  B2F_CUDA_TRY(launch_pdl(kv4_compact_kernel, dim3(copy_grid(p, p.pages / 2 + 1)), dim3(256), 0, s, p, (const int*)plan));
  return B2F_OK;
}

int b2f_kv4_copy_pages(const b2f_kv4_pool* pool, const int* src, const int* dst, int n, b2f_stream_t stream) {
  using namespace b2f;
  Pool p;
  if (const char* e = check_pool(pool, &p)) return fail(B2F_ERR_ARG, std::string("kv4_copy_pages: ") + e);
  if (n <= 0 || src == nullptr || dst == nullptr) return fail(B2F_ERR_ARG, "kv4_copy_pages: empty list");
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= p.pages || dst[i] < 0 || dst[i] >= p.pages)
      return fail(B2F_ERR_ARG, "kv4_copy_pages: page out of range");
  try {  // the copies run side by side: no page is written twice, or both read and written
    std::vector<int> to(dst, dst + n);
    std::sort(to.begin(), to.end());
    if (std::adjacent_find(to.begin(), to.end()) != to.end())
      return fail(B2F_ERR_ARG, "kv4_copy_pages: a page is written twice");
    for (int i = 0; i < n; ++i)
      if (std::binary_search(to.begin(), to.end(), src[i]))
        return fail(B2F_ERR_ARG, "kv4_copy_pages: a page is both read and written");
  } catch (const std::bad_alloc&) {
    return fail(B2F_ERR_ARG, "kv4_copy_pages: out of host memory");
  }
  cudaStream_t s = (cudaStream_t)stream;
  for (int at = 0; at < n; at += kPairsPerLaunch) {
    PagePairs pairs = {};
    const int m = std::min(kPairsPerLaunch, n - at);
    std::copy(src + at, src + at + m, pairs.src);
    std::copy(dst + at, dst + at + m, pairs.dst);
    B2F_CUDA_TRY(launch_pdl(kv4_copy_pages_kernel, dim3(copy_grid(p, m)), dim3(256), 0, s, p, pairs, m));
  }
  return B2F_OK;
}

}  // extern "C"
