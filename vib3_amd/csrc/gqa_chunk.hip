// gqa_chunk.hip — causal attention of each sequence's newest tokens over the paged key/value cache.
//
// Bound by the matrix cores for prompts, 4 dim flops per visible (query, token, head), by the cache's bytes for a few queries over
// many tokens. The queries of a sequence times the heads of one key/value head's group are rows; a block is 32 NB rows of each wave of a
// workgroup, which walks over the tokens, 64 at a time (a tile), with a running maximum and sum per row.
//
// Scores are formed transposed, S^T = K . Q^T, so that a lane holds one row's scores of 32 of the 64 tokens (the other lane
// of the pair l, l + 32 the rest): the maximum and sum are almost all within a lane, and the probabilities, packed in pairs of
// 16 bits, are as they stand the B operand of O^T = V^T . P^T (the tokens' order along k is free as long as V^T is read in the
// same one, which the transposing LDS reads allow). The scores of the next tile are formed next to the softmax of this one, so that
// the matrix cores and the vector units have work of one wave at a time.
//
// Keys and values go straight from memory to LDS, double-buffered. Each wave looks up the pages of a tile's 64 tokens, a token (or a
// group of them on one page) a lane, three tiles ahead for heads of 128, two for others, and hands the addresses to the lanes that load. 16-byte chunk c of an LDS row lies at c ^ a function of
// the row, which spreads the reads over the banks.
//
// Many blocks: a workgroup each, the longest of a sequence first. Few blocks: long ones are cut along the tokens into pieces, which a
// causal mask's unequal blocks and long caches under few queries need alike; a piece's sums go to the workspace as they lie in
// registers, and a second launch joins them. How long a piece is follows from the lengths alone, which every workgroup reads for
// itself, so a captured launch follows them.
//
// Measured: 12288 tokens of 32 heads over 8 of 128: 1.24 ms, 994 TFLOP/s (a library product of 8192^3: 1223, held down by the card's power),
// 64 heads of 64 1.51 ms, 16 over 2 of 256 1.77 ms. The matrix cores are busy for 43 % of the cycles and the vector units for 50 %, and
// the two add up: products and softmax of one wave interleaved by hand, sums a tile late, and 64 rows a wave were no faster (1.34 to 1.38
// and, with spilled registers, 2.7 ms). 16 sequences' 4 drafted tokens of 16 heads over 2 of 256 after 317 to 5642: 37 us and 10 to join.
#include <type_traits>

#include "gqa.h"
#include "scan.h"

namespace vib3 {
namespace {

constexpr int kTile = 64;         // tokens of one step
constexpr int kMaxBlocks = 1024;  // of a launch that may cut them, and its most sequences
// What a piece takes besides its tiles, and what the parts of as many pieces as there are workgroups on the card take on their way through
// memory and with the second launch, in tiles' time. (32 heads over 8: 2048 tokens cut 82 us, whole 78; 512 after 32768 tokens 301 and 950.)
constexpr int kPieceCost = 2, kPartsCost = 8, kJoinCost = 2;

// Workgroups on the card at a time.
__host__ __device__ constexpr int card_groups(int dim) { return dim == 64 ? 512 : 256; }

// What tokens that are not seen are read from.
__device__ const uint4 zero_token[256 / 8] = {};

// 16 bytes a lane from global memory, at a wave-uniform address and a lane's offset, to LDS at base + 16 * lane (see mla.h's load_to_lds16).
__device__ __forceinline__ void load_group_to_lds16(const void* g, uint32_t off, lds_u8* base) {
  const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)base);
  // (the address is a scalar select: a vector instruction that wrote it would need wait states that nobody sees here)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(g) : "memory", "m0");
}

// The queries of a sequence.
struct Queries {
  int seq, q0, nq, len;  // its row of the table, its first query, their number, its tokens
};

__device__ __forceinline__ Queries queries_of(const vib3_gqa_chunk& a, int s) {
  Queries q{s, 0, 0, 0};
  if (s < a.cache.num_seqs) {
    q.q0 = min(max(a.cu_q[s], 0), a.q_tokens);
    q.nq = max(min(a.cu_q[s + 1], a.q_tokens) - q.q0, 0);
    q.len = gqa_len(a.cache, a.lens[s]);
  }
  return q;
}

// What block b (of `size` rows) of a sequence sees, in tiles: `skip` tiles from the first token on (those with sinks), then from tile
// `first` on.
struct Block {
  Queries q;
  int row0, rows;        // its first row in the sequence, the sequence's rows
  int low, high;         // the positions of its first and its last query
  int skip, first, tiles;
  __device__ __forceinline__ int token(int t) const { return (t < skip ? t : first + t - skip) * kTile; }
};

__device__ __forceinline__ Block block_of(const vib3_gqa_chunk& a, const Queries& q, int b, int size, int group) {
  Block k;
  k.q = q;
  k.row0 = b * size;
  k.rows = q.nq * group;
  k.low = q.len - q.nq + k.row0 / group;
  k.high = q.len - q.nq + (min(k.row0 + size, k.rows) - 1) / group;
  const int start = window_start(max(k.low, 0), a.window);
  k.first = start / kTile;
  k.skip = min((min(a.sinks, start) + kTile - 1) / kTile, k.first);
  k.tiles = k.high < 0 ? 0 : k.high / kTile + 1 - k.first + k.skip;
  return k;
}

// Blocks of all sequences are numbered in order, a sequence's last block first (it sees the most tokens). Each wave finds block b
// by itself, 64 sequences at a time; false: there is no block b.
__device__ bool find_block(const vib3_gqa_chunk& a, int b, int size, int group, Block* out) {
  const int lane = lane_id();
  for (int s0 = 0; s0 < a.cache.num_seqs; s0 += 64) {
    const Queries q = queries_of(a, s0 + lane);
    int upto = (int)(((int64_t)q.nq * group + size - 1) / size);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const uint64_t hit = __ballot(b < upto);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const Queries mine{s0 + l, __builtin_amdgcn_readlane(q.q0, l), __builtin_amdgcn_readlane(q.nq, l),
                         __builtin_amdgcn_readlane(q.len, l)};
      *out = block_of(a, mine, __builtin_amdgcn_readlane(upto, l) - 1 - b, size, group);
      return true;
    }
    b -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// A block that was cut, for the joining: its first query's token, the rows of its sequence, its first row there, its pieces, and their
// first slot (of key/value head 0).
struct JoinBlock {
  int q0, rows, row0, pieces, slot, pad[3];
};

// Workspace of a launch that may cut blocks: fewer than 2 pieces for each workgroup on the card are of cut blocks.
struct ChunkWs {
  int32_t* head;     // [2]: cut blocks of a key/value head, their slots
  JoinBlock* join;   // [groups]
  float2* stat;      // [slots][rows] reference value (of unscaled scores) and sum
  float* part;       // [slots][rows][dim] unnormalised sums, as the lanes hold them
};

inline size_t chunk_ws(int size, int dim, ChunkWs* w, void* base) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return (uint8_t*)base + p;
  };
  ChunkWs r;
  r.head = (int32_t*)take(8);
  r.join = (JoinBlock*)take(sizeof(JoinBlock) * card_groups(dim));
  const size_t slots = 2 * (size_t)card_groups(dim);
  r.stat = (float2*)take(8 * slots * size);
  r.part = (float*)take(4 * slots * size * dim);
  if (w) *w = r;
  return at;
}

struct ChunkArgs {
  vib3_gqa_chunk a;
  ChunkWs w;
  int group;
};

// The plan of a launch that may cut blocks, in LDS: each workgroup forms it for itself, which is why it takes few steps.
struct Plan {
  int wave_sums[2][8], wave_counts[8][6], wave_rows[8];
  float wave_tiles[8];
  int wave_longest[8];
  int upto[kMaxBlocks];                    // blocks of the sequences up to each
  int q0[kMaxBlocks], nq[kMaxBlocks], len[kMaxBlocks];
  int tiles[kMaxBlocks];
  int16_t begin[kMaxBlocks + 1];           // pieces of the blocks before each
  int16_t seq[kMaxBlocks], in[kMaxBlocks];
  int16_t slot[kMaxBlocks + 1];            // pieces of cut blocks before each
  int16_t cuts[kMaxBlocks + 1];            // cut blocks before each
};

// Sum of v over the threads before this one (THREADS of them); *all: over all of them. A barrier; calls take turns with `sums`.
template <int THREADS>
__device__ int scan_block(int v, int* sums, int* all) {
  const int tid = (int)threadIdx.x, upto = add_up(v);
  if ((tid & 63) == 63) sums[tid >> 6] = upto;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) {
    const int s = sums[i];
    before += i < tid >> 6 ? s : 0;
    total += s;
  }
  *all = total;
  return before + upto - v;
}

template <int THREADS>
__device__ int make_plan(const ChunkArgs& d, int size, int groups, Plan& p) {
  constexpr int kWaves = THREADS / 64;
  const vib3_gqa_chunk& a = d.a;
  const int tid = (int)threadIdx.x, wave = tid >> 6;
  const bool last = (tid & 63) == 63;
  int turn = 0, blocks = 0;  // (no more than kMaxBlocks, unless the offsets decrease somewhere)
  for (int s0 = 0; s0 < a.cache.num_seqs; s0 += THREADS) {
    const int s = s0 + tid;
    const Queries q = queries_of(a, s);  // (without queries past the last sequence)
    const int n = min((int)(((int64_t)q.nq * d.group + size - 1) / size), kMaxBlocks);
    int all;
    const int before = scan_block<THREADS>(n, p.wave_sums[turn ^= 1], &all);
    if (s < a.cache.num_seqs) {
      p.upto[s] = min(blocks + before + n, kMaxBlocks);
      p.q0[s] = q.q0, p.nq[s] = q.nq, p.len[s] = q.len;
    }
    blocks = min(blocks + all, kMaxBlocks);
  }
  __syncthreads();
  float tiles = 0.0f;
  int rows = 0, longest = 0;
  for (int b = tid; b < blocks; b += THREADS) {
    int lo = 0, hi = a.cache.num_seqs - 1;  // the first sequence with upto > b
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (p.upto[mid] > b) hi = mid;
      else lo = mid + 1;
    }
    const int in = b - (lo ? p.upto[lo - 1] : 0);
    p.seq[b] = (int16_t)lo;
    p.in[b] = (int16_t)in;
    const Block bl = block_of(a, Queries{lo, p.q0[lo], p.nq[lo], p.len[lo]}, in, size, d.group);
    p.tiles[b] = bl.tiles;
    tiles += (float)bl.tiles;
    longest = max(longest, bl.tiles);
    rows += min(size, bl.rows - bl.row0);
  }
  tiles = wave_scan(tiles, 0.0f, [](float x, float y) { return x + y; });
  rows = add_up(rows);
  longest = wave_scan(longest, 0, [](int x, int y) { return max(x, y); });
  if (last) p.wave_tiles[wave] = tiles, p.wave_rows[wave] = rows, p.wave_longest[wave] = longest;
  __syncthreads();
  float all_tiles = 0.0f, all_rows = 0.0f;
  longest = 1;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    all_tiles += p.wave_tiles[i];
    all_rows += (float)p.wave_rows[i];
    longest = max(longest, p.wave_longest[i]);
  }
  all_tiles *= (float)a.cache.kv_heads;
  // The length of a piece: whole blocks, an even share of the tiles, or a third more or twice that, where the even share's pieces do not fit
  // the card at a time: whichever takes least, of the longest piece, or of rounds of pieces over the card, and of the parts' time.
  // (An even share is rounded up, above what the sum of tiles lacks: the pieces of cut blocks are fewer than twice the workgroups.)
  const float even = all_tiles / (float)groups * 1.0001f;
  const int length[3] = {(int)fminf(even, 1e9f) + 1, (int)fminf(even * 1.34f, 1e9f) + 1, (int)fminf(even * 2.0f, 1e9f) + 1};
  int count[6] = {};  // pieces, and those of cut blocks
  for (int b = tid; b < blocks; b += THREADS)
#pragma unroll
    for (int k = 0; k < 3; k++) {
      const int n = max((p.tiles[b] + length[k] - 1) / length[k], 1);
      count[k] += n;
      count[3 + k] += n > 1 ? n : 0;
    }
#pragma unroll
  for (int k = 0; k < 6; k++) {
    count[k] = add_up(count[k]);
    if (last) p.wave_counts[wave][k] = count[k];
  }
  __syncthreads();
  auto cost = [&](int len, float pieces) {
    return fmaxf((float)(len + kPieceCost), ceilf(pieces / (float)groups) * (all_tiles / pieces + kPieceCost));
  };
  const float filled = all_rows / ((float)max(blocks, 1) * (float)size);
  int piece = longest;
  float best = cost(piece, fmaxf((float)blocks * (float)a.cache.kv_heads, 1.0f));
#pragma unroll
  for (int k = 0; k < 3; k++) {
    int pieces = 0, slots = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) pieces += p.wave_counts[i][k], slots += p.wave_counts[i][3 + k];
    const float c = cost(length[k], fmaxf((float)pieces * (float)a.cache.kv_heads, 1.0f)) + kJoinCost +
                    kPartsCost * filled * (float)slots * (float)a.cache.kv_heads / (float)groups;
    if (slots > 0 && c < best) best = c, piece = length[k];
  }
  uint32_t at = 0;  // pieces (of a key/value head fewer than 2^11), above them those of cut blocks (as many), and the cut blocks
  for (int b0 = 0; b0 < blocks; b0 += THREADS) {
    const int b = b0 + tid;
    uint32_t n = 0;
    if (b < blocks) {
      n = (uint32_t)max((p.tiles[b] + piece - 1) / piece, 1);
      if (n > 1) n += n << 11 | 1u << 22;
    }
    int all;
    const uint32_t before = at + (uint32_t)scan_block<THREADS>((int)n, p.wave_sums[turn ^= 1], &all);
    if (b < blocks) p.begin[b] = (int16_t)(before & 2047), p.slot[b] = (int16_t)(before >> 11 & 2047), p.cuts[b] = (int16_t)(before >> 22);
    at += (uint32_t)all;
  }
  if (tid == 0) p.begin[blocks] = (int16_t)(at & 2047), p.slot[blocks] = (int16_t)(at >> 11 & 2047), p.cuts[blocks] = (int16_t)(at >> 22);
  __syncthreads();
  return blocks;
}

template <int DT, int D, int WAVES, int NB, bool CUT, bool WHOLE>
__global__ __launch_bounds__(WAVES * 64, D == 64 ? 4 : 1) void k_gqa_tiles(ChunkArgs d) {
  constexpr int C = D / 8;                    // 16-byte chunks of a row
  constexpr int KS = D / 16;                  // k steps of the scores
  constexpr int VB = D / 32;                  // 32-column blocks of the sums
  constexpr int kRows = WAVES * 32 * NB;      // of a block
  constexpr int kPer = 64 / C;                // tokens of one load instruction of a wave
  constexpr int kLoads = kTile / kPer / WAVES;  // load instructions of a wave for a tile's keys
  // Scores a tile ahead of their softmax, and keys two ahead. A head of 256 has no registers for that; one of 64 does without, and four
  // waves fit on a SIMD instead of two (12288 tokens of 64 heads over 8: 1.78 -> 1.49 ms).
  constexpr bool kAhead = D == 128;
  __shared__ __align__(1024) uint8_t ktile[2][kTile * D * 2];
  __shared__ __align__(1024) uint8_t vtile[2][kTile * D * 2];
  __shared__ int odd_values;                  // whether values were cleared
  __shared__ std::conditional_t<CUT, Plan, int> plan;

  const vib3_gqa_chunk& a = d.a;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const float scale = exponent_scale(a.scale);
  const uint32_t flip = sign_flip(a.scale);
  const uint64_t zero = (uint64_t)zero_token;
  if (tid == 0) odd_values = 0;
  __syncthreads();  // any wave may set it, in the first tile already

  // One block's tiles t0..t1 - 1 of key/value head g: its sums go to the output, or as a part to a slot of the workspace.
  auto attend = [&](const Block& bl, int g, int t0, int t1, int slot) {
    const int group = d.group;
    // this lane's rows: their positions (-1: none) and the first tokens of their windows
    int pos[NB], start[NB];
    int64_t q_at[NB], o_at[NB];
#pragma unroll
    for (int n = 0; n < NB; n++) {
      const int r = bl.row0 + (wave * NB + n) * 32 + col, rr = min(r, bl.rows - 1), qi = rr / group;
      const int64_t t = bl.q.q0 + qi, h = g * group + rr - qi * group;
      q_at[n] = t * a.q_token_stride + h * a.q_head_stride;
      o_at[n] = t * a.out_token_stride + h * a.out_head_stride;
      pos[n] = r < bl.rows ? max(bl.q.len - bl.q.nq + qi, -1) : -1;
      start[n] = pos[n] >= 0 ? window_start(pos[n], a.window) : 0;
    }
    // the wave's first and last position (of its rows that there are): tiles that all of them see whole, or none sees
    const int w_row = bl.row0 + wave * NB * 32;
    const bool any_rows = w_row < bl.rows;
    const int w_low = bl.q.len - bl.q.nq + w_row / group;
    const int w_high = any_rows ? bl.q.len - bl.q.nq + (min(w_row + NB * 32, bl.rows) - 1) / group : -1;
    const int low_start = window_start(max(w_low, 0), a.window), high_start = window_start(max(w_high, 0), a.window);
    const int block_start = window_start(max(bl.high, 0), a.window);

    // queries: the B operand, this lane's row at k = 16 s + 8 half
    s16x8 q[NB][KS];
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int s = 0; s < KS; s++) {
        uint4 v = *(const uint4*)((const uint16_t*)a.q + q_at[n] + 16 * s + 8 * half);
        v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
        q[n][s] = __builtin_bit_cast(s16x8, v);
      }
    VIB3_WAIT_VM(0);  // here, once: a wait inside the loop would drain the tiles' loads

    // Page numbers of a tile's tokens, a token a lane, or with whole groups of kPer tokens on a page a group a lane; then their places as
    // offsets from the pools' start in bytes (-1: not there).
    // (With selects, not branches: registers are short here, and the compiler has put a copy that it needed for that at the end
    // of a divergent branch in front of the instruction that brings the other lanes back, which lost their values.)
    constexpr int kStep = WHOLE ? kPer : 1, kGroups = kTile / kStep;
    const int32_t* table = a.cache.block_table + (size_t)bl.q.seq * a.cache.max_pages;
    const int64_t head_at = (int64_t)g * a.cache.head_stride;
    const int first_token = lane % kGroups * kStep;
    const int turn_page = kTile / a.cache.page_size, turn_rest = kTile - turn_page * a.cache.page_size;
    int page = 0, rest = 0, page_no = -1, in_page = -1;  // page and rest: of tile `asked`
    auto find = [&](int t) {  // by division, where a stretch of tiles begins
      const int j = bl.token(t) + first_token;
      page = j / a.cache.page_size;
      rest = j - page * a.cache.page_size;
    };
    auto ask = [&](int t) {
      const bool ok = (t < t1) & (bl.token(t) + first_token < bl.q.len);
      in_page = ok ? rest : -1;
      page_no = table[ok ? page : 0];  // (a block with tiles has a first token, and its page an entry)
      // the next tile's
      if (t + 1 == bl.skip) {
        find(t + 1);
      } else {
        rest += turn_rest;
        page += turn_page;
        const bool over = rest >= a.cache.page_size;
        rest -= over ? a.cache.page_size : 0;
        page += over ? 1 : 0;
      }
    };
    struct Place {
      uint32_t lo, hi;
    };
    auto place = [&]() -> Place {
      const bool ok = (in_page >= 0) & ((unsigned)page_no < (unsigned)a.cache.num_pages);
      const int64_t at = 2 * ((int64_t)page_no * a.cache.page_stride + (int64_t)in_page * a.cache.token_stride + head_at);
      const uint32_t none = ok ? 0 : ~0u;
      return Place{(uint32_t)at | none, (uint32_t)((uint64_t)at >> 32) | none};
    };
    // The tokens of a tile that are there.
    auto seen_of = [&](int t, const Place& p) -> uint64_t {
      if constexpr (!WHOLE) return __ballot((int)p.hi >= 0);
      const uint64_t groups = __ballot((int)p.hi >= 0);
      if (groups == ~0ull && bl.token(t) + kTile <= bl.q.len) return ~0ull;
      return __ballot((groups >> (lane / kStep) & 1) != 0 && bl.token(t) + lane < bl.q.len);
    };
    // Chunk `lane % C ^ swizzle(row)` of this lane's token of each of the wave's load instructions. Of a whole group the first token's address is
    // the same for all lanes, and what a lane adds to it the same for all groups (of every second one, for the keys of a head of 256).
    auto load = [&](const void* pool, uint8_t* dst, const Place& at, const uint32_t (&lane_at)[2], auto swizzle) {
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int run = i * WAVES + wave, row = run * kPer + lane / C;
        if constexpr (WHOLE) {
          const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)at.lo, run), hi = (uint32_t)__builtin_amdgcn_readlane((int)at.hi, run);
          const bool none = (int32_t)hi < 0;
          const uint64_t p = none ? zero : (uint64_t)pool + ((uint64_t)hi << 32 | lo);
          load_group_to_lds16((const void*)p, none ? (uint32_t)(lane % C) * 16 : lane_at[D == 256 ? i & 1 : 0], (lds_u8*)dst + run * 1024);
        } else {
          const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * row, (int)at.lo), hi = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * row, (int)at.hi);
          const uint64_t p = (int32_t)hi < 0 ? zero : (uint64_t)pool + ((uint64_t)hi << 32 | lo);
          load_to_lds16((const void*)(p + (((lane % C) ^ swizzle(row)) * 16)), (lds_u8*)dst + run * 1024);
        }
      }
    };
    auto key_of = [](int r) { return key_swizzle<C>(r); };
    auto value_of = [](int r) { return value_swizzle<C>(r); };
    uint32_t key_at[2], value_at[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int row = (i * WAVES + wave) * kPer + lane / C;
      const uint32_t token = (uint32_t)(lane / C) * (uint32_t)a.cache.token_stride * 2;
      key_at[i] = token + ((lane % C) ^ key_of(row)) * 16;
      value_at[i] = token + ((lane % C) ^ value_of(row)) * 16;
    }
    auto load_keys = [&](int t, const Place& p) { load(a.cache.keys, ktile[t & 1], p, key_at, key_of); };
    auto load_values = [&](int t, const Place& p) { load(a.cache.values, vtile[t & 1], p, value_at, value_of); };
    // A masked place has probability 0, and 0 times an infinity or a NaN is NaN: in tiles with masked places the values that
    // this wave has loaded are cleared of those, and whether there were any is noted.
    auto is_masked = [&](int base) { return !(base + kTile - 1 <= bl.low && (base >= block_start || base + kTile <= a.sinks)); };
    auto clear_values = [&](int t) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        uint4* at = (uint4*)(vtile[t & 1] + (i * WAVES + wave) * 1024 + lane * 16);
        // (of a whole group the tokens past the last one are what lies in its page)
        if (WHOLE && bl.token(t) + (i * WAVES + wave) * kPer + lane / C >= bl.q.len) *at = make_uint4(0, 0, 0, 0);
        const uint4 v = *at, w = make_uint4(finite_only<DT>(v.x), finite_only<DT>(v.y), finite_only<DT>(v.z), finite_only<DT>(v.w));
        if (v.x != w.x || v.y != w.y || v.z != w.z || v.w != w.w) {
          *at = w;
          odd = true;
        }
      }
      if (__any(odd) && lane == 0) odd_values = 1;
    };

    // S^T of a tile: two blocks of 32 tokens
    auto form_scores = [&](int t, f32x16 (*s)[NB]) {
      const lds_u8* k = (lds_u8*)ktile[t & 1] + col * D * 2;
      const int k0 = fresh((half ^ key_swizzle<C>(col)) * 16);
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int n = 0; n < NB; n++) s[b][n] = f32x16{};
#pragma unroll
      for (int i = 0; i < KS; i++)
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const s16x8 key = lds_read16(k + b * 32 * D * 2 + (k0 ^ 32 * i));
#pragma unroll
          for (int n = 0; n < NB; n++) s[b][n] = mma_wide<DT>(key, q[n][i], s[b][n]);
        }
    };

    f32x16 o[NB][VB] = {};
    float m[NB], l[NB];  // running maximum (of unscaled scores) and this lane's part of the sum
#pragma unroll
    for (int n = 0; n < NB; n++) m[n] = -__builtin_huge_valf(), l[n] = 0.0f;
    f32x16 s[2][NB];
    uint64_t seen = 0, seen1 = 0;  // the tokens of this tile and the next that are there
    Place p1{};                    // of the next tile
    if (t0 < t1) {
      find(t0);
      ask(t0);
      Place p0 = place();
      seen = seen_of(t0, p0);
      load_keys(t0, p0);
      ask(t0 + 1);
      if constexpr (kAhead) {
        wait_lds_loads();
        __syncthreads();
        load_values(t0, p0);
        p1 = place();
        seen1 = seen_of(t0 + 1, p1);
        load_keys(t0 + 1, p1);
        ask(t0 + 2);
        form_scores(t0, s);
      } else {
        load_values(t0, p0);
      }
    }
    // this lane's place in a transposing read: row 4 half + (lane % 16) / 4, columns 16 ((lane / 16) % 2) + 4 (lane % 4)
    const int vrow = 4 * half + ((lane & 15) >> 2);
    const int vchunk = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    // One tile: its scores in s, the next one's into s_next.
    auto step = [&](int t, f32x16 (*s)[NB], f32x16 (*s_next)[NB]) {
      wait_lds_loads();
      page_no = fresh(page_no);  // has landed too: no wait for it after the loads below
      const int base = bl.token(t);
      if (is_masked(base)) clear_values(t);
      __syncthreads();  // values t and keys t (or t + 1) are in LDS; everyone is done with those before
      // (loads past the last tile are of zeros)
      const uint64_t mine = seen;
      if constexpr (kAhead) {
        load_values(t + 1, p1);
        seen = seen1;
        p1 = place();
        seen1 = seen_of(t + 2, p1);
        load_keys(t + 2, p1);
        ask(t + 3);
        form_scores(t + 1, s_next);  // past the last tile: of whatever lies there, and not used
      } else {
        p1 = place();
        seen = seen_of(t + 1, p1);
        load_keys(t + 1, p1);
        load_values(t + 1, p1);
        ask(t + 2);
        form_scores(t, s);
      }
      if (base > w_high || (base + kTile <= low_start && base >= a.sinks)) return;  // no row of the wave sees any of it
      if (!(base + kTile - 1 <= w_low && (base >= high_start || base + kTile <= a.sinks) && mine == ~0ull)) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const uint32_t there = (uint32_t)(mine >> (32 * b)) >> (4 * half);
          const int j0 = base + 32 * b + 4 * fresh(half);
#pragma unroll
          for (int n = 0; n < NB; n++) {
            const int last = pos[n] - j0, from = start[n] - j0, sinks = a.sinks - j0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const int k = 8 * (i >> 2) + (i & 3);
              const bool hidden = ((there >> k & 1) == 0) | (k > last) | ((k < from) & (k >= sinks));
              s[b][n][i] = hidden ? -__builtin_huge_valf() : s[b][n][i];
            }
          }
        }
      }

      uint32_t p[NB][16];
#pragma unroll
      for (int n = 0; n < NB; n++) {
        float top = s[0][n][0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, s[0][n][i]);
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, s[1][n][i]);
        top = pair_max(top);
        // The reference value of a row's exponentials follows its maximum only where that grew by more than kLag. (Each row by
        // itself: what others of the wave see does not change its result.)
        const bool grown = (top - m[n]) * scale > kLag<DT> || (m[n] == -__builtin_huge_valf() && top > m[n]);
        if (__any(grown)) {
          const float f = grown ? __builtin_amdgcn_exp2f((m[n] - top) * scale) : 1.0f;
          m[n] = grown ? top : m[n];
          l[n] *= f;
#pragma unroll
          for (int c = 0; c < VB; c++) o[n][c] *= f;
        }
        float ref = m[n] == -__builtin_huge_valf() ? 0.0f : m[n] * scale;
        const bool far = __builtin_fabsf(ref) > kFarExponent;
        if (__any(far)) {
          const float off = far ? m[n] : 0.0f;
          ref = far ? 0.0f : ref;
#pragma unroll
          for (int b = 0; b < 2; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) s[b][n][i] -= off;
        }
        ref -= kProbShift<DT>;
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][n][i], scale, -ref));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][n][i + 1], scale, -ref));
            l[n] += e0 + e1;
            // rounded for the matrix cores; the sum l takes them unrounded. (The remainder as a second operand takes 44 % more: 12288 tokens
            // 1284 -> 1851 us. Without it the result is off by 0.0022 in bf16 and 0.00026 in f16, rounded once by 0.0016 and 0.00021.)
            p[n][8 * b + (i >> 1)] = pack2<DT>(e0, e1);
          }
      }
      lds_u8* const v = (lds_u8*)vtile[t & 1] + vrow * D * 2 + 8 * (lane & 1);
      const int v0 = fresh((vchunk ^ value_swizzle<C>(vrow)) * 16);  // 16 and 8 rows further the swizzle is the same
      // V^T for 32 columns and 16 tokens
      auto values = [&](int k, int c) {
        return join(lds_read_tr(v + 16 * k * D * 2 + (v0 ^ 64 * c)), lds_read_tr(v + (16 * k + 8) * D * 2 + (v0 ^ 64 * c)));
      };
      auto probs = [&](int n, int k) {
        return __builtin_bit_cast(s16x8, make_uint4(p[n][4 * k], p[n][4 * k + 1], p[n][4 * k + 2], p[n][4 * k + 3]));
      };
#pragma unroll
      for (int k = 0; k < kTile / 16; k++)
#pragma unroll
        for (int c = 0; c < VB; c++) {
          const s16x8 x = values(k, c);
#pragma unroll
          for (int n = 0; n < NB; n++) o[n][c] = mma_wide<DT>(x, probs(n, k), o[n][c]);
        }
    };
    if constexpr (kAhead) {  // the two sets of scores in turns
      f32x16 other[2][NB];
      for (int t = t0; t < t1; t += 2) {
        step(t, s, other);
        if (t + 1 < t1) step(t + 1, other, s);
      }
    } else {
      for (int t = t0; t < t1; t++) step(t, s, s);
    }
    wait_lds_loads();  // those past the last tile too: they must not land after the workgroup has ended
    __syncthreads();   // odd_values is whole
    // What is not finite, for the queries that see it: a value that was cleared is missing, and one whose probability is 0 in the
    // 16-bit type only (f16, below 2^-36 of the largest) made a NaN of what is an infinity. Such values are looked for in memory, in
    // masked tiles or, for a sum that is NaN, in all, and count by their probability in f32. (Scores are formed again from memory
    // too, so that the ordinary path holds nothing for this one.)
    float odd_sum[8] = {};  // NaN where a sum of this lane is not finite
#pragma unroll
    for (int n = 0; n < NB; n++)
#pragma unroll
      for (int c = 0; c < VB; c++)
#pragma unroll
        for (int i = 0; i < 16; i++) odd_sum[i % 8] = __builtin_fmaf(o[n][c][i], 0.0f, odd_sum[i % 8]);
#pragma unroll
    for (int i = 1; i < 8; i++) odd_sum[0] += odd_sum[i];
    if (__builtin_amdgcn_readfirstlane(odd_values) || __any(odd_sum[0] != odd_sum[0])) {
      bool open = false, number[NB], zero_sum[NB];  // whether a NaN has to be explained; whether the probabilities' sum is no NaN, and 0
#pragma unroll
      for (int n = 0; n < NB; n++) {
        const float sum = pair_sum(l[n]);
        number[n] = sum == sum;  // (a sum of probabilities that is NaN makes all of the row NaN)
        zero_sum[n] = m[n] == -__builtin_huge_valf() && sum == 0.0f;
#pragma unroll
        for (int c = 0; c < VB; c++)
#pragma unroll
          for (int i = 0; i < 16; i++) open |= number[n] & (o[n][c][i] != o[n][c][i]);
      }
      bool search = __any(open);
      const int lane_now = fresh(lane), half_now = lane_now >> 5;  // (the loop above has its own)
      constexpr uint16_t kFraction = DT == VIB3_DT_F16 ? 0x3ff : 0x7f;
      // a bit for each of the lane's sums: what an infinity of either sign and what a NaN is added to
      uint32_t above[NB][(VB + 1) / 2] = {}, below[NB][(VB + 1) / 2] = {}, none[NB][(VB + 1) / 2] = {};
#pragma unroll 1
      for (int t = t0; t < t1; t++) {
        const int base = bl.token(t);
        if (base > w_high || (base + kTile <= low_start && base >= a.sinks) || !(search || is_masked(base))) continue;
        bool found = false;
#pragma unroll 1
        for (int j0 = base; j0 < base + kTile; j0 += kPer) {
          const int jl = j0 + lane_now / C;
          const int64_t at = jl < bl.q.len ? gqa_token(a.cache, bl.q.seq, jl) : -1;
          const uint4 w = *(const uint4*)(at < 0 ? (const uint16_t*)zero : (const uint16_t*)a.cache.values + at + head_at + lane_now % C * 8);
          uint64_t hits = __ballot(!all_finite<DT>(w));
          found |= hits != 0;
          while (hits) {
            const int in = (__ffsll((unsigned long long)hits) - 1) / C, j = j0 + in;
            hits &= ~(((1ull << C) - 1) << (in * C));
            const int64_t token = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)((uint64_t)at >> 32), in * C) << 32 |
                                            (uint32_t)__builtin_amdgcn_readlane((int)at, in * C));
            const uint16_t* key = (const uint16_t*)a.cache.keys + token + head_at;
            const uint16_t* value = (const uint16_t*)a.cache.values + token + head_at;
#pragma unroll
            for (int n = 0; n < NB; n++) {
              float score = 0.0f;
#pragma unroll 4
              for (int c = 0; c < C; c += 2) {  // the other chunks are the pair's other lane's
                float x[8], y[8];
                unpack8<DT>(*(const uint4*)((const uint16_t*)a.q + q_at[n] + 8 * (c + half_now)), x);
                unpack8<DT>(*(const uint4*)(key + 8 * (c + half_now)), y);
#pragma unroll
                for (int i = 0; i < 8; i++) score = __builtin_fmaf(x[i], y[i], score);
              }
              score = a.scale < 0.0f ? -pair_sum(score) : pair_sum(score);
              const float e = __builtin_amdgcn_exp2f((score - (m[n] == -__builtin_huge_valf() ? 0.0f : m[n])) * scale);
              const bool sees = (j <= pos[n]) & ((j >= start[n]) | (j < a.sinks));
#pragma unroll
              for (int c = 0; c < VB; c++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                  const uint16_t y = value[32 * c + 8 * (i >> 2) + 4 * half_now + (i & 3)];
                  const bool odd = sees & (finite_only<DT>(y) != y), nan = (e == 0.0f) | ((y & kFraction) != 0), minus = (y & 0x8000) != 0;
                  const uint32_t bit = 1u << (c % 2 * 16 + i);
                  none[n][c / 2] |= odd & nan ? bit : 0;
                  above[n][c / 2] |= odd & !nan & !minus ? bit : 0;
                  below[n][c / 2] |= odd & !nan & minus ? bit : 0;
                }
            }
          }
        }
        if (search && found) {  // until each NaN has its reason
          open = false;
#pragma unroll
          for (int n = 0; n < NB; n++)
#pragma unroll
            for (int c = 0; c < VB; c++)
#pragma unroll
              for (int i = 0; i < 16; i++)
                open |= number[n] && o[n][c][i] != o[n][c][i] && !((none[n][c / 2] | (above[n][c / 2] & below[n][c / 2])) >> (c % 2 * 16 + i) & 1);
          search = __any(open);
        }
      }
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int c = 0; c < VB; c++)
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const uint32_t bit = 1u << (c % 2 * 16 + i);
            const bool up = above[n][c / 2] & bit, down = below[n][c / 2] & bit, nan = (none[n][c / 2] & bit) || (up && down);
            const float odd = nan ? __builtin_nanf("") : up ? __builtin_huge_valf() : -__builtin_huge_valf(), sum = o[n][c][i];
            o[n][c][i] = zero_sum[n] ? 0.0f : !(nan | up | down) ? sum : sum != sum ? odd : sum + odd;
          }
    }

    if (slot >= 0) {
      float* part = d.w.part + (size_t)slot * kRows * D;
#pragma unroll
      for (int n = 0; n < NB; n++) {
        if (w_row + n * 32 >= bl.rows) continue;  // no rows: nobody joins them
        const int row = (wave * NB + n) * 32 + col;
        const float sum = pair_sum(l[n]);
        if (half == 0) d.w.stat[(size_t)slot * kRows + row] = make_float2(m[n], sum);
#pragma unroll
        for (int c = 0; c < VB; c++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            *(float4*)(part + ((((wave * NB + n) * VB + c) * 4 + i) * 64 + lane) * 4) =
                make_float4(o[n][c][4 * i], o[n][c][4 * i + 1], o[n][c][4 * i + 2], o[n][c][4 * i + 3]);
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < NB; n++) {
      const float sum = pair_sum(l[n]), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const bool there = bl.row0 + (wave * NB + n) * 32 + col < bl.rows;
      uint16_t* out = (uint16_t*)a.out + o_at[n];
#pragma unroll
      for (int c = 0; c < VB; c++)
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
          // columns 8 (i / 4) + 4 half + 0..3 and 8 further: the pair of lanes trades halves, so that each has 8 neighbouring ones
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 2; j++) {
            const auto x = __builtin_amdgcn_permlane32_swap(pack2<DT>(o[n][c][i + 2 * j] * inv, o[n][c][i + 2 * j + 1] * inv),
                                                            pack2<DT>(o[n][c][i + 4 + 2 * j] * inv, o[n][c][i + 5 + 2 * j] * inv), false, false);
            w[j] = x[0];
            w[2 + j] = x[1];
          }
          if (there) *(uint4*)(out + 32 * c + 2 * i + 8 * half) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
  };

  if constexpr (!CUT) {
    const unsigned item = wide_block();
    const int g = (int)(item % (unsigned)a.cache.kv_heads);
    Block bl;
    if (!find_block(a, (int)(item / (unsigned)a.cache.kv_heads), kRows, d.group, &bl)) return;
    attend(bl, g, 0, bl.tiles, -1);
  } else {
    const int blocks = __builtin_amdgcn_readfirstlane(make_plan<WAVES * 64>(d, kRows, card_groups(D), plan));
    const int slots = __builtin_amdgcn_readfirstlane((int)plan.slot[blocks]);
    if (blockIdx.x == 0) {
      if (tid == 0) d.w.head[0] = plan.cuts[blocks], d.w.head[1] = slots;
      for (int b = tid; b < blocks; b += WAVES * 64) {
        const int s = plan.seq[b], pieces = plan.slot[b + 1] - plan.slot[b];
        if (pieces > 0) d.w.join[plan.cuts[b]] = JoinBlock{plan.q0[s], plan.nq[s] * d.group, plan.in[b] * kRows, pieces, plan.slot[b], {}};
      }
    }
    // the last pieces first: those of a sequence's last queries
    const int g = (int)(blockIdx.x % (unsigned)a.cache.kv_heads);
    const int at = __builtin_amdgcn_readfirstlane((int)plan.begin[blocks]) - 1 - (int)(blockIdx.x / (unsigned)a.cache.kv_heads);
    if (at < 0) return;
    int b = 0;
    for (int hi = blocks - 1; b < hi;) {  // the last block that begins at or before `at` (each has a piece)
      const int mid = (b + hi + 1) / 2;
      if (__builtin_amdgcn_readfirstlane((int)plan.begin[mid]) <= at) b = mid;
      else hi = mid - 1;
    }
    const int begin = __builtin_amdgcn_readfirstlane((int)plan.begin[b]), n = __builtin_amdgcn_readfirstlane((int)plan.begin[b + 1]) - begin, i = at - begin;
    const int s = __builtin_amdgcn_readfirstlane((int)plan.seq[b]);
    const Queries q{s, __builtin_amdgcn_readfirstlane(plan.q0[s]), __builtin_amdgcn_readfirstlane(plan.nq[s]), __builtin_amdgcn_readfirstlane(plan.len[s])};
    const Block bl = block_of(a, q, __builtin_amdgcn_readfirstlane((int)plan.in[b]), kRows, d.group);
    const int each = bl.tiles / n, over = bl.tiles - each * n;
    attend(bl, g, each * i + min(i, over), each * (i + 1) + min(i + 1, over),
           n == 1 ? -1 : g * slots + __builtin_amdgcn_readfirstlane((int)plan.slot[b]) + i);
  }
}

// Joins the parts of 32 rows of a block that was cut: a wave for each 32 columns.
template <int DT, int D>
__global__ __launch_bounds__(D * 2) void k_gqa_join_tiles(ChunkArgs d, int size) {
  constexpr int VB = D / 32;
  const vib3_gqa_chunk& a = d.a;
  const int lane = (int)threadIdx.x & 63, c = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int subs = size / 32, sub = (int)blockIdx.x % subs, item = (int)blockIdx.x / subs;
  const int b = item / a.cache.kv_heads, g = item - b * a.cache.kv_heads;  // (b is less than the workgroups on the card)
  const JoinBlock k = d.w.join[b];
  const int row0 = k.row0 + sub * 32;
  if (b >= d.w.head[0] || row0 >= k.rows) return;
  const size_t first = (size_t)g * d.w.head[1] + k.slot;
  const float scale = exponent_scale(a.scale);
  float m = -__builtin_huge_valf(), l = 0.0f;
  for (int j = 0; j < k.pieces; j++) m = fmaxf(m, d.w.stat[(first + j) * size + sub * 32 + col].x);
  const float ref = m == -__builtin_huge_valf() ? 0.0f : m;
  float o[16] = {};
#pragma unroll 2
  for (int j = 0; j < k.pieces; j++) {
    const float2 st = d.w.stat[(first + j) * size + sub * 32 + col];
    const float f = __builtin_amdgcn_exp2f((st.x - ref) * scale);
    const float4* p = (const float4*)(d.w.part + (first + j) * size * D) + ((sub * VB + c) * 4) * 64 + lane;
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = p[i * 64];
    l += f * st.y;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      o[4 * i] += f * v[i].x;
      o[4 * i + 1] += f * v[i].y;
      o[4 * i + 2] += f * v[i].z;
      o[4 * i + 3] += f * v[i].w;
    }
  }
  const int r = row0 + col;
  if (r >= k.rows) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int qi = r / d.group;
  uint16_t* out = (uint16_t*)a.out + (int64_t)(k.q0 + qi) * a.out_token_stride + (int64_t)(g * d.group + r - qi * d.group) * a.out_head_stride;
#pragma unroll
  for (int i = 0; i < 4; i++)
    *(uint2*)(out + 32 * c + 8 * i + 4 * half) =
        make_uint2(pack2<DT>(o[4 * i] * inv, o[4 * i + 1] * inv), pack2<DT>(o[4 * i + 2] * inv, o[4 * i + 3] * inv));
}

// Waves and row blocks of a wave: as their registers leave room for.
template <int D>
struct Shape {
  static constexpr int waves = D == 256 ? 4 : 8, blocks = 1, rows = waves * 32 * blocks;
};

inline int block_rows(int dim) { return dim == 64 ? Shape<64>::rows : dim == 128 ? Shape<128>::rows : Shape<256>::rows; }

template <int DT, int D, bool WHOLE>
int launch_chunk(const ChunkArgs& d, hipStream_t st) {
  using S = Shape<D>;
  const vib3_gqa_chunk& a = d.a;
  // Sequences' blocks number at most this many (each ends in one that is not full, and has a query)
  const int64_t seqs = a.cache.num_seqs < a.q_tokens ? a.cache.num_seqs : a.q_tokens;
  const int64_t blocks = ((int64_t)a.q_tokens * d.group + (S::rows - 1) * seqs) / S::rows, items = blocks * a.cache.kv_heads;
  if (items > 0x7fffffff) return VIB3_ERR_BAD_COUNT;
  constexpr int kGroups = card_groups(D);
  // Whole blocks save the plan and the second launch, but the card waits for a long one beside short ones, and the host does not know the
  // lengths. So: whole from four blocks a place on the card, and from two where none can see more than 96 tiles. Measured with 32 heads
  // over 8 of 128, us whole / cut:
  //   one prompt   80 / 88 (2048 tokens, one block a place: cut, for what may lie beside it), 185 / 200 (4096, two), 363 / 377 (6144, three
  //                of 96 tiles), 463 / 477 (7168, 3.5 of 112 tiles), 590 / 603 (8192, four)
  //   16 tokens after 6000 (94 tiles) beside prompts of 200   145 / 98 (24 of them, three blocks a place), 156 / 172 (48, six)
  //   the same after 30000                                    673 / 125 and 675 / 200: the 96 keeps the first of them cut, the last is not
  int64_t longest = (int64_t)a.cache.max_pages * a.cache.page_size;
  if (a.window > 0 && (int64_t)a.window + a.sinks + S::rows / d.group < longest) longest = (int64_t)a.window + a.sinks + S::rows / d.group;
  if (items >= (longest <= 96 * kTile ? 2 : 4) * kGroups || blocks > kMaxBlocks || a.cache.num_seqs > kMaxBlocks) {
    hipLaunchKernelGGL((k_gqa_tiles<DT, D, S::waves, S::blocks, false, WHOLE>), wide_grid(items), dim3(S::waves * 64), 0, st, d);
  } else {  // (pieces of at least an even share: no more than blocks and shares)
    hipLaunchKernelGGL((k_gqa_tiles<DT, D, S::waves, S::blocks, true, WHOLE>), dim3((unsigned)items + kGroups), dim3(S::waves * 64), 0, st, d);
    hipLaunchKernelGGL((k_gqa_join_tiles<DT, D>), dim3((unsigned)(items < kGroups ? items : kGroups) * (S::rows / 32)), dim3(D * 2), 0, st, d, S::rows);
  }
  VIB3_RETURN_LAUNCH();
}

template <int DT>
int launch_chunk_dt(const ChunkArgs& d, hipStream_t st) {
  const vib3_gqa_cache& c = d.a.cache;
  // whole groups of tokens on a page, and their distance in 32 bits
  if (c.page_size % 8 == 0 && c.token_stride < (1 << 27))
    return c.dim == 64 ? launch_chunk<DT, 64, true>(d, st) : c.dim == 128 ? launch_chunk<DT, 128, true>(d, st) : launch_chunk<DT, 256, true>(d, st);
  return c.dim == 64 ? launch_chunk<DT, 64, false>(d, st) : c.dim == 128 ? launch_chunk<DT, 128, false>(d, st) : launch_chunk<DT, 256, false>(d, st);
}

}  // namespace
}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_gqa_chunk_workspace_bytes(const vib3_gqa_chunk* args) {
  if (!args || check_gqa_cache(args->cache) || args->q_tokens < 0 || !gqa_heads(args->heads, args->cache.kv_heads)) return 0;
  return chunk_ws(block_rows(args->cache.dim), args->cache.dim, nullptr, nullptr);
}

extern "C" int vib3_launch_gqa_chunk(const vib3_gqa_chunk* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_gqa_chunk& a = *args;
  if (const int rc = check_gqa_cache(a.cache)) return rc;
  if (!__builtin_isfinite(a.scale)) return VIB3_ERR_UNSUPPORTED;
  if (!gqa_heads(a.heads, a.cache.kv_heads) || a.q_tokens < 0 || a.window < 0 || a.sinks < 0) return VIB3_ERR_BAD_COUNT;
  if ((int64_t)a.q_tokens * a.heads > 0x7fffffff - 256) return VIB3_ERR_BAD_COUNT;  // so that the end of the last block is an int
  if (a.q_tokens == 0 || a.cache.num_seqs == 0) return 0;
  if (!a.cu_q || !a.lens || !mla_aligned(a.q) || !mla_aligned(a.out) || !mla_stride(a.q_token_stride) || !mla_stride(a.q_head_stride) ||
      !mla_stride(a.out_token_stride) || !mla_stride(a.out_head_stride) || !a.workspace || ((uintptr_t)a.workspace & 255))
    return VIB3_ERR_BAD_POINTER;
  ChunkArgs d;
  d.a = a;
  d.group = a.heads / a.cache.kv_heads;
  if (a.workspace_bytes < chunk_ws(block_rows(a.cache.dim), a.cache.dim, &d.w, a.workspace)) return VIB3_ERR_WORKSPACE;
  return a.cache.dtype == VIB3_DT_F16 ? launch_chunk_dt<VIB3_DT_F16>(d, (hipStream_t)stream)
                                      : launch_chunk_dt<VIB3_DT_BF16>(d, (hipStream_t)stream);
}
