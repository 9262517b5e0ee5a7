// cache_pages.hip — a cache's pages forked and compacted, in all of its pools at once.
//
// Bound by the bytes copied, read once and written once. A copied page is cut into pieces of 16 KB, a workgroup each, whose loads are all
// on their way before its first store; pools go with the launch's arguments, kPools at a time. Measured: 212 MB in 4 layers' pools
// compacted in 48 us, 4.4 TB/s (a plain copy of 2 GB: 5.0); of that the plan, one workgroup's, takes 7. 32 sequences forked in 8 layers in
// 13 us (the parents' pages come from the caches).
#include "kernels.h"
#include "scan.h"

namespace vib3 {
namespace {

constexpr int kPools = 64;
constexpr int kPiece = 1024;  // 16-byte chunks of a piece
constexpr int kMaxCompact = 1 << 20;

// A pool as the kernels take it: 16-byte chunks of a page and of a token, and the divisions by a run's chunks and a token's.
struct Pool {
  uint8_t* base;
  int64_t page_stride, run_stride, token_stride;
  int chunks, per;
  Divisor by_run, by_token;
};
struct Pools {
  Pool pool[kPools];
};
static_assert(sizeof(Pools) <= 3584, "4 KB of arguments a launch, with what else it takes");

__host__ __device__ inline int64_t page_chunks(const vib3_page_pool& p, int page_size) {
  return (int64_t)p.runs * page_size * (p.token_bytes / 16);
}

// One piece of a page, of its first `tokens` tokens, to another page (256 threads). STREAM: past the caches, for what nothing reads soon.
template <bool STREAM>
__device__ __forceinline__ void copy_piece(const Pool& p, int page_size, int tokens, int from, int to, int piece) {
  const uint8_t* src = p.base + (int64_t)from * p.page_stride;
  uint8_t* dst = p.base + (int64_t)to * p.page_stride;
  const int run = p.per * page_size;
  u32x4 v[kPiece / 256];
  int64_t at[kPiece / 256];
  bool ok[kPiece / 256];
#pragma unroll
  for (int i = 0; i < kPiece / 256; i++) {
    const int c = piece * kPiece + i * 256 + (int)threadIdx.x;
    const int r = p.by_run.of(c), in = c - r * run, t = p.by_token.of(in);
    at[i] = (int64_t)r * p.run_stride + (int64_t)t * p.token_stride + (int64_t)(in - t * p.per) * 16;
    ok[i] = (c < p.chunks) & (t < tokens);
  }
  if (tokens == page_size && (piece + 1) * kPiece <= p.chunks) {  // all loads first: a branch would have each waited for
#pragma unroll
    for (int i = 0; i < kPiece / 256; i++) {
      const u32x4* from_at = (const u32x4*)(src + at[i]);
      v[i] = STREAM ? __builtin_nontemporal_load(from_at) : *from_at;
    }
#pragma unroll
    for (int i = 0; i < kPiece / 256; i++) {
      u32x4* to_at = (u32x4*)(dst + at[i]);
      if (STREAM) __builtin_nontemporal_store(v[i], to_at);
      else *to_at = v[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kPiece / 256; i++) v[i] = *(const u32x4*)(src + (at[i] & -(int64_t)ok[i]));
#pragma unroll
  for (int i = 0; i < kPiece / 256; i++)
    if (ok[i]) *(u32x4*)(dst + at[i]) = v[i];
}

// ------------------------------------------------------------------------- fork

// Workgroups 0..count - 1 write the children's rows of the table (in the first launch of a call), the others copy.
__global__ __launch_bounds__(256) void k_fork_pages(vib3_fork_pages a, Pools pools, int pieces, int table_blocks, unsigned blocks) {
  const unsigned block = wide_block();
  if (block >= blocks) return;
  const int b = (int)block - table_blocks, i = b < 0 ? (int)block : b / pieces % a.count;
  const int p = a.parents[i], c = a.children[i], fresh = a.new_pages[i];
  if ((unsigned)p >= (unsigned)a.num_seqs || (unsigned)c >= (unsigned)a.num_seqs) return;
  const int64_t cap = min((int64_t)a.max_pages * a.page_size, (int64_t)0x7fffffff);
  const int n = a.lens[p], len = n <= 0 ? 0 : n > cap ? (int)cap : n;
  const int full = len / a.page_size, rest = len - full * a.page_size;
  const int32_t* parent = a.block_table + (size_t)p * a.max_pages;
  if (b < 0) {
    int32_t* child = a.block_table + (size_t)c * a.max_pages;
    for (int k = (int)threadIdx.x; k < a.max_pages; k += 256) child[k] = k < full ? parent[k] : k == full ? fresh : -1;
    return;
  }
  if (rest == 0) return;
  const int from = parent[full];
  if ((unsigned)from >= (unsigned)a.num_pages || (unsigned)fresh >= (unsigned)a.num_pages) return;
  copy_piece<false>(pools.pool[b / pieces / a.count], a.page_size, rest, from, fresh, b % pieces);
}

// ------------------------------------------------------------------------- compaction

// Device workspace: the number of moves, their pages, and the pages' new numbers (of those that move).
struct CompactWs {
  int32_t* count;
  int32_t *from, *to;  // [num_pages / 2]: a move takes a page in use and one that is not
  int32_t* place;      // [num_pages]
};

inline size_t compact_ws(int num_pages, CompactWs* w, void* base) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return (int32_t*)((uint8_t*)base + p);
  };
  CompactWs r;
  r.count = take(4);
  r.from = take(4 * (size_t)(num_pages / 2));
  r.to = take(4 * (size_t)(num_pages / 2));
  r.place = take(4 * (size_t)num_pages);
  if (w) *w = r;
  return at;
}

__device__ __forceinline__ int used_entries(const vib3_compact_pages& a, int s) {
  const int n = a.lens[s];
  return n <= 0 ? 0 : min((n - 1) / a.page_size + 1, a.max_pages);
}

// Sum of v over the threads before this one, of 1024 threads; *all: over all of them.
__device__ int block_scan(int v, int* wave_sums, int* all) {
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int sum = add_up(v);
  __syncthreads();
  if (lane == 63) wave_sums[tid >> 6] = sum;
  __syncthreads();
  int before = 0, total = 0;
  for (int i = 0; i < 16; i++) {
    if (i < tid >> 6) before += wave_sums[i];
    total += wave_sums[i];
  }
  *all = total;
  return before + sum - v;
}

// One workgroup: a bit for each page in use, in LDS; the ranks of pages among those in use by a scan over its words.
__global__ __launch_bounds__(1024) void k_compact_plan(vib3_compact_pages a, CompactWs w) {
  __shared__ uint32_t bits[kMaxCompact / 32];
  __shared__ int sums[16];
  __shared__ int below;
  const int tid = (int)threadIdx.x;
  const int words = (a.num_pages + 31) / 32, per = (words + 1023) / 1024;
  for (int k = tid; k < words; k += 1024) bits[k] = 0;
  __syncthreads();
  // a wave a row, 4 rows of 64 entries on their way at a time
  auto mark = [&](int id) {
    if ((unsigned)id < (unsigned)a.num_pages) atomicOr(&bits[id / 32], 1u << (id % 32));
  };
  const int lane = tid & 63, wave = tid >> 6;
  for (int s0 = wave; s0 < a.num_seqs; s0 += 16 * 64) {
    const int used = s0 + 16 * lane < a.num_seqs ? used_entries(a, s0 + 16 * lane) : 0;
    for (int i = 0; i < 64 && s0 + 16 * i < a.num_seqs; i += 4) {
      int n[4], id[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        n[j] = __builtin_amdgcn_readlane(used, i + j);
        id[j] = lane < n[j] ? a.block_table[(size_t)(s0 + 16 * (i + j)) * a.max_pages + lane] : -1;
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        mark(id[j]);
        for (int k = 64 + lane; k < n[j]; k += 64) mark(a.block_table[(size_t)(s0 + 16 * (i + j)) * a.max_pages + k]);
      }
    }
  }
  __syncthreads();
  // a thread's words, in order
  const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
  int mine = 0, live;
  for (int k = w0; k < w1; k++) mine += __popc(bits[k]);
  const int before = block_scan(mine, sums, &live);
  // pages in use below `live`: the first of those from there on moves to the first place that is not in use
  {
    int n = before;
    for (int k = w0; k < w1; k++) {
      if (live >= 32 * k && live < 32 * k + 32) below = n + __popc(bits[k] & ((1u << (live % 32)) - 1));
      n += __popc(bits[k]);
    }
    if (tid == 0 && live >= 32 * words) below = live;  // all pages are in use
  }
  __syncthreads();
  const int kept = below;
  int n = before;
  for (int k = w0; k < w1; k++) {
    const uint32_t word = bits[k];
    for (int i = 0; i < 32; i++) {
      const int page = 32 * k + i;
      const bool used = word >> i & 1;
      if (used && page >= live) w.from[n - kept] = page;
      if (!used && page < live) w.to[page - n] = page;
      n += used;
    }
  }
  __syncthreads();
  const int moves = live - kept;
  for (int k = tid; k < moves; k += 1024) w.place[w.from[k]] = w.to[k];
  if (tid == 0) {
    *w.count = moves;
    *a.live = live;
  }
}

// Workgroups 0..table_blocks - 1 write the table (in the first launch of a call), the others go through the pieces of all moves.
__global__ __launch_bounds__(256) void k_compact_move(vib3_compact_pages a, CompactWs w, Pools pools, int num_pools, int pieces,
                                                      int table_blocks) {
  const int live = *a.live;
  if ((int)blockIdx.x < table_blocks) {
    for (int s = (int)blockIdx.x; s < a.num_seqs; s += table_blocks) {
      const int n = used_entries(a, s);
      const size_t row = (size_t)s * a.max_pages;
      for (int k = (int)threadIdx.x; k < a.max_pages; k += 256) {
        int id = -1;
        if (k < n) {
          id = a.block_table[row + k];
          if (id >= live && id < a.num_pages) id = w.place[id];
        }
        a.out_table[row + k] = id;
      }
    }
    return;
  }
  const int moves = *w.count, each = num_pools * pieces, step = (int)gridDim.x - table_blocks, first = (int)blockIdx.x - table_blocks;
  const int step_moves = step / each, step_rest = step - step_moves * each;
  int move = first / each, rest = first - move * each;
  while (move < moves) {
    const int pool = rest / pieces;
    copy_piece<true>(pools.pool[pool], a.page_size, a.page_size, w.from[move], w.to[move], rest - pool * pieces);
    move += step_moves;
    rest += step_rest;
    if (rest >= each) rest -= each, move++;
  }
}

// The most pieces of a page in pools [first, first + n), and these as arguments.
int gather_pools(const vib3_page_pool* pools, int n, int page_size, Pools* out) {
  int64_t most = 1;
  for (int i = 0; i < n; i++) {
    const vib3_page_pool& p = pools[i];
    const int64_t c = page_chunks(p, page_size);
    const int per = p.token_bytes / 16;
    out->pool[i] = Pool{(uint8_t*)p.base, p.page_stride, p.run_stride, p.token_stride, (int)c, per, divisor(per * page_size), divisor(per)};
    most = c > most ? c : most;
  }
  return (int)((most + kPiece - 1) / kPiece);
}

int check_pools(const vib3_page_pool* pools, int num_pools, int num_pages, int page_size, int num_seqs, int max_pages) {
  if (num_pools < 0 || num_pages < 0 || page_size < 1 || page_size > 65536 || num_seqs < 0 || max_pages < 0) return VIB3_ERR_BAD_COUNT;
  if (num_pools && !pools) return VIB3_ERR_BAD_POINTER;
  for (int i = 0; i < num_pools; i++) {
    const vib3_page_pool& p = pools[i];
    if (p.runs < 1 || p.token_bytes < 16 || p.page_stride < 0 || p.run_stride < 0 || p.token_stride < 0) return VIB3_ERR_BAD_COUNT;
    if ((num_pages && !p.base) || ((uintptr_t)p.base & 15) || p.token_bytes % 16 || p.page_stride % 16 || p.run_stride % 16 ||
        p.token_stride % 16)
      return VIB3_ERR_BAD_POINTER;
    if ((int64_t)p.runs * page_size > (0x7fffffff - kPiece) / (p.token_bytes / 16)) return VIB3_ERR_BAD_COUNT;  // page_chunks fits an int
  }
  return 0;
}

}  // namespace
}  // namespace vib3

using namespace vib3;

extern "C" int vib3_launch_fork_pages(const vib3_fork_pages* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_fork_pages& a = *args;
  if (const int rc = check_pools(a.pools, a.num_pools, a.num_pages, a.page_size, a.num_seqs, a.max_pages)) return rc;
  if (a.count < 0) return VIB3_ERR_BAD_COUNT;
  if (a.count == 0 || a.num_seqs == 0 || a.max_pages == 0) return 0;
  if (!a.block_table || !a.lens || !a.parents || !a.children || !a.new_pages) return VIB3_ERR_BAD_POINTER;
  int first = 0;
  do {
    const int n = a.num_pools - first < kPools ? a.num_pools - first : kPools;
    Pools pools{};
    const int pieces = gather_pools(a.pools + first, n, a.page_size, &pools);
    const int table_blocks = first == 0 ? a.count : 0;
    const int64_t blocks = table_blocks + (int64_t)a.count * n * pieces;
    if (blocks > 0x7fffffff) return VIB3_ERR_BAD_COUNT;
    hipLaunchKernelGGL(k_fork_pages, wide_grid(blocks), dim3(256), 0, (hipStream_t)stream, a, pools, pieces, table_blocks, (unsigned)blocks);
    first += n;
  } while (first < a.num_pools);
  VIB3_RETURN_LAUNCH();
}

extern "C" size_t vib3_compact_pages_workspace_bytes(const vib3_compact_pages* args) {
  if (!args || args->num_pages < 0 || args->num_pages > kMaxCompact) return 0;
  return compact_ws(args->num_pages, nullptr, nullptr);
}

extern "C" int vib3_launch_compact_pages(const vib3_compact_pages* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_compact_pages& a = *args;
  if (const int rc = check_pools(a.pools, a.num_pools, a.num_pages, a.page_size, a.num_seqs, a.max_pages)) return rc;
  if (a.num_pages > kMaxCompact) return VIB3_ERR_BAD_COUNT;
  if (!a.live || !a.workspace || ((uintptr_t)a.workspace & 255)) return VIB3_ERR_BAD_POINTER;
  if (a.num_seqs && (!a.lens || (a.max_pages && (!a.block_table || !a.out_table)))) return VIB3_ERR_BAD_POINTER;
  if (a.workspace_bytes < vib3_compact_pages_workspace_bytes(&a)) return VIB3_ERR_WORKSPACE;
  CompactWs w;
  compact_ws(a.num_pages, &w, a.workspace);
  hipLaunchKernelGGL(k_compact_plan, dim3(1), dim3(1024), 0, (hipStream_t)stream, a, w);
  int first = 0;
  do {
    const int n = a.num_pools - first < kPools ? a.num_pools - first : kPools;
    Pools pools{};
    const int pieces = gather_pools(a.pools + first, n, a.page_size, &pools);
    const int table_blocks = first == 0 ? (a.num_seqs < 256 ? a.num_seqs : 256) : 0;
    const int64_t most = (int64_t)(a.num_pages / 2) * n * pieces;
    const int64_t blocks = table_blocks + (most < 2048 ? most : 2048);
    if (blocks)
      hipLaunchKernelGGL(k_compact_move, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, w, pools, n, pieces, table_blocks);
    first += n;
  } while (first < a.num_pools);
  VIB3_RETURN_LAUNCH();
}
