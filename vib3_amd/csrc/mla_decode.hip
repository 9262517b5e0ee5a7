// mla_decode.hip — attention of single query tokens over the paged latent cache, absorbed form.
//
// Per row and head: ql = q_nope . W_uk, scores of every visible cached row against [ql | q_rope], softmax, the
// weighted sum of the latents, out = W_uv . that. All heads share the cached rows, so a row of 1152 bytes
// serves 64 heads x 2176 flops: at 64 heads the cache read and the matrix cores are of one order, and the read bounds.
// Three launches:
//   k_mla_absorb   ql for all rows, on the matrix cores; one more workgroup plans the next launch
//   k_mla_attend   the attention in the latent space, over equal shares of all rows' cached tokens
//   k_mla_finish   rows that several workgroups shared are joined, and W_uv applied
// At 64 heads of 128 x 512, bf16, the launches' own times: one row of 777 tokens 5 + 14 + 8 us; one of 131072 5 + 45 + 16;
// 96 rows of 2048 to 12288 (654 MB) 12 + 140 to 159 + 20.
//
// The plan: tokens are taken 32 at a time (a unit), heads in groups of up to 64. All units of all items
// (row, head group) in order, with kItemCost units' time in front of each item for taking it up and storing its sums, are
// cut into kShares equal runs, one workgroup each, whatever the rows' lengths: a long row is shared by many workgroups, a run
// covers many short rows (without the fixed time 41 rows of 1 to 4100 tokens took 28 us, with it 19). Nothing on the host
// depends on the lengths, so a captured launch follows them.
#include <type_traits>

#include "mla.h"

namespace vib3 {

constexpr int kMlaMaxRows = 65536;
constexpr int kUnit = 32;      // cached tokens of one step
constexpr int kShares = 256;   // workgroups of the attention launch, one per CU (its LDS tiles fill one)
constexpr int kItemCost = 3;   // an item's fixed time, in units

struct Item {
  int64_t begin;      // where the item begins, in units and fixed times of the items before
  int32_t len, seq;   // visible tokens of its row, and their sequence
};

__host__ __device__ inline int64_t unit_count(int64_t len) { return (len + kUnit - 1) / kUnit; }

struct Share {        // what a workgroup starts with
  int64_t total;      // its units
  int32_t item, seq, len, unit, left;  // the first item, its units before the share and in it
};

// Device workspace. Slot w of the parts holds that of the item that share w starts with (where it does not cover all of it), slot
// kShares + w that of the item it ends in, if that is another one. A slot is followed by 2 KB, so that one head's parts, which
// one workgroup joins, do not all lie in the same memory channels.
struct DecodeWs {
  int64_t* head;      // length of a share, in units and fixed times
  Item* items;        // [items + 1]
  Share* shares;      // [kShares]
  uint16_t* ql;       // [rows][heads][2][rank] latent queries: rounded to 16 bits, and what the rounding left
  float* ol;          // [rows][padded heads][rank] weighted latent of items that one share covers
  float* part;        // [2 kShares][heads of a group][rank] (and the gap) unnormalised sums
  float2* stat;       // [heads of a group][2 kShares] reference value (of unscaled scores) and sum
};

__host__ __device__ inline int head_groups(int heads) { return (heads + 63) / 64; }
__host__ __device__ inline int head_blocks(int heads) { return heads <= 16 ? 1 : heads <= 32 ? 2 : 4; }  // of 16, a group's
// Heads that a row of weighted latents and a slot of parts have room for: whole blocks, so that nothing is cut off in storing.
__host__ __device__ inline int padded_heads(int heads) { return heads <= 64 ? head_blocks(heads) * 16 : 128; }
__host__ __device__ inline int group_heads(int heads) { return head_blocks(heads) * 16; }
constexpr int kSlotGap = 512;  // floats

inline size_t decode_ws(const vib3_mla_decode& a, DecodeWs* w, void* base) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return (uint8_t*)base + p;
  };
  const size_t row = (size_t)a.heads * a.cache.rank;
  DecodeWs r;
  r.head = (int64_t*)take(16);
  r.items = (Item*)take(sizeof(Item) * ((size_t)a.rows * head_groups(a.heads) + 1));
  r.shares = (Share*)take(sizeof(Share) * kShares);
  r.ql = (uint16_t*)take(a.kv_b ? 4 * row * a.rows : 0);
  r.ol = (float*)take(4 * (size_t)padded_heads(a.heads) * a.cache.rank * a.rows);
  r.part = (float*)take(4 * ((size_t)group_heads(a.heads) * a.cache.rank + kSlotGap) * 2 * kShares);
  r.stat = (float2*)take(8 * (size_t)group_heads(a.heads) * 2 * kShares);
  if (w) *w = r;
  return at;
}

struct DecodeArgs {
  vib3_mla_decode a;
  DecodeWs w;
};

// Visible cached tokens of row r and its sequence.
__device__ __forceinline__ int row_len(const vib3_mla_decode& a, int r, int* seq) {
  const int s = a.seqs ? a.seqs[r] : r;
  *seq = s;
  return (unsigned)s < (unsigned)a.cache.num_seqs ? clamp_len(a.cache, a.lens[r]) : 0;
}

// ------------------------------------------------------------------------- the plan

// One workgroup of 256: where the items begin, the share length, and what each share starts with. An item without tokens has
// no extent; of any other, the units come after the fixed time, so that a share that ends within that has none of them.
__device__ void make_plan(const vib3_mla_decode& a, const DecodeWs& w) {
  constexpr int kLocal = 1024;  // with more items the search below goes through memory
  __shared__ int64_t wave_total[4];
  __shared__ int64_t begins[kLocal + 1];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int groups = head_groups(a.heads), items = a.rows * groups;
  int64_t before = 0;
  for (int x0 = 0; x0 < items; x0 += 256) {
    const int x = x0 + tid;
    int seq = 0;
    const int len = x < items ? row_len(a, x / groups, &seq) : 0;
    const int64_t n = len > 0 ? unit_count(len) + kItemCost : 0;
    int64_t sum = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    if (lane == 63) wave_total[tid >> 6] = sum;
    __syncthreads();
    int64_t base = before;
    for (int i = 0; i < 4; i++) {
      if (i < (tid >> 6)) base += wave_total[i];
      before += wave_total[i];
    }
    if (x < items) {
      w.items[x] = Item{base + sum - n, len, seq};
      if (x < kLocal) begins[x] = base + sum - n;
    }
    __syncthreads();
  }
  const int64_t per = max((int64_t)1, (before + kShares - 1) / kShares);
  if (tid == 0) {
    w.items[items] = Item{before, 0, 0};
    if (items <= kLocal) begins[items] = before;
    w.head[0] = per;
  }
  __syncthreads();
  static_assert(kShares == 256, "a thread per share");
  const int64_t from = tid * per, to = min(from + per, before);
  Share sh{};
  if (from < before) {
    auto begin = [&](int x) { return items <= kLocal ? begins[x] : w.items[x].begin; };
    int lo = 0, hi = items;  // the last item that begins at or before the share
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (begin(mid) <= from) lo = mid;
      else hi = mid;
    }
    const Item it = w.items[lo];
    const int64_t first = max((int64_t)0, from - it.begin - kItemCost);
    sh.item = lo;
    sh.seq = it.seq;
    sh.len = it.len;
    sh.unit = (int32_t)first;
    sh.left = (int32_t)max((int64_t)0, min(to - it.begin - kItemCost, unit_count(it.len)) - first);
    sh.total = sh.left;
    for (int x = lo + 1; x < items && begin(x) < to; x++)  // the units of the items that begin in the share
      sh.total += max((int64_t)0, min(to, begin(x + 1)) - begin(x) - kItemCost);
  }
  w.shares[tid] = sh;
}

__global__ __launch_bounds__(256) void k_mla_plan(DecodeArgs d) { make_plan(d.a, d.w); }

// ------------------------------------------------------------------------- ql = q_nope . W_uk

constexpr int kAbsorbCols = 128;
constexpr int kAbsorbRows = 64;

// A workgroup takes 128 latent columns of one head for 64 rows, 16 rows a wave: that part of W_uk goes to LDS while each wave loads
// its queries, and is multiplied as (W_uk^T) . (q^T). W_uk lies with the latent columns contiguous, so its operand is read
// transposed. LDS rows are 256 bytes; 16-byte chunk c of row n lies at c ^ swizzle(n), which spreads a transposing read over the
// banks. Bound by the read of W_uk (8.4 MB for 64 heads of 128 x 512), and below some 16 rows by its latency.
__device__ __forceinline__ int absorb_swizzle(int n) { return ((n & 3) << 2) ^ (((n >> 3) & 1) << 1); }

template <int DT>
__global__ __launch_bounds__(256) void k_mla_absorb(DecodeArgs d, int col_blocks) {
  const vib3_mla_decode& a = d.a;
  extern __shared__ __align__(16) uint8_t tile[];  // [nope][kAbsorbCols]
  if (blockIdx.x == 0) {  // first: the next launch waits for it
    if (blockIdx.y == 0) make_plan(a, d.w);
    return;
  }
  const int h = (int)(blockIdx.x - 1) / col_blocks, c0 = ((int)(blockIdx.x - 1) % col_blocks) * kAbsorbCols;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rank = a.cache.rank;
  const uint16_t* w = (const uint16_t*)a.kv_b + (size_t)h * (a.nope + a.v_dim) * rank + c0;
  for (int i = wave; i < a.nope / 4; i += 4) {  // four rows of W_uk at a time
    const int n = 4 * i + (lane >> 4), c = (lane & 15) ^ absorb_swizzle(n);
    load_to_lds16(w + (size_t)n * rank + 8 * c, (lds_u8*)tile + i * 1024);
  }
  const int row = lane & 15, g = lane >> 4;
  const int r = (int)blockIdx.y * kAbsorbRows + wave * 16 + row;
  const uint16_t* q = (const uint16_t*)a.q_nope + (int64_t)min(r, a.rows - 1) * a.q_nope_row_stride + (int64_t)h * a.q_nope_head_stride + 8 * g;
  s16x8 b[8];
#pragma unroll
  for (int k = 0; k < 8; k++) b[k] = k * 32 < a.nope ? *(const s16x8*)(q + k * 32) : s16x8{};
  // this lane's element of a transposing read: row 8 g + row / 4 (+ 4), columns 16 blk + 4 (row % 4)
  const int n0 = 8 * g + (row >> 2);
  wait_lds_loads();
  __syncthreads();
  if ((int)blockIdx.y * kAbsorbRows + wave * 16 >= a.rows) return;
  f32x4 acc[8] = {};
#pragma unroll
  for (int k = 0; k < 8; k++) {
    if (k * 32 >= a.nope) break;
    const int na = k * 32 + n0, nb = na + 4;
    lds_u8* t = (lds_u8*)tile + na * 256 + 8 * (row & 1);
#pragma unroll
    for (int blk = 0; blk < 8; blk++) {
      const int c = blk * 2 + ((row & 3) >> 1);
      acc[blk] = mma32<DT>(join(lds_read_tr(t + (c ^ absorb_swizzle(na)) * 16), lds_read_tr(t + 1024 + (c ^ absorb_swizzle(nb)) * 16)),
                           b[k], acc[blk]);
    }
  }
  if (r < a.rows) {
    uint16_t* o = d.w.ql + ((size_t)r * a.heads + h) * 2 * rank + c0 + 4 * g;
    // A rounding of the latent query alone would double the result's error (0.0034 against 0.0017 relative in bf16, together
    // with one of the weighted latent); the remainder costs products, but no further reads of the cached rows.
#pragma unroll
    for (int blk = 0; blk < 8; blk++) {
      const Halves x = split2<DT>(acc[blk][0], acc[blk][1]), y = split2<DT>(acc[blk][2], acc[blk][3]);
      *(uint2*)(o + 16 * blk) = make_uint2(x.hi, y.hi);
      *(uint2*)(o + rank + 16 * blk) = make_uint2(x.lo, y.lo);
    }
  }
}

// ------------------------------------------------------------------------- attention in the latent space

// What masked tokens read instead of the cache: their probability is 0, and 0 times whatever lies there must be 0.
__device__ const uint4 zero_row[(512 + 64) / 8] = {};

// A workgroup takes HB blocks of 16 heads (1, 2 or 4; more than 64 heads are groups of 64, planned like rows of their own)
// with eight waves, one of either kind on each SIMD, that work on neighbouring units of 32 tokens between the same two barriers:
//   waves 0-3  form the scores and probabilities of unit k, 16 heads each. S^T = K . Q^T: a lane holds one head's scores of 4
//              tokens per 16, so that the running maximum and sum stay within the wave; the probabilities go to LDS.
//   waves 4-7  add to the sums O^T = C^T . P^T of all heads for unit k - 1, a quarter of the latent's columns each (C^T by
//              transposing reads), and load unit k + 2.
// With one barrier a unit, and each SIMD with vector work of one wave next to products of the other, 96 rows of 64 heads
// took 133 us; all eight waves going through the same phases, with three barriers, 163. The latent queries' second summand
// (below) made it 140 to 159: 4.0 to 4.5 TB/s, of the 6.0 that reading alone reaches. Bound by both: a unit's rows come at that rate
// in 1.6 us, and its reads from LDS (each row once per 16 heads for the scores, and once for the sums) fill some 1400 cycles of
// the 2 us that it takes, the products 1100.
//
// Rows go from the pages straight to LDS (16 bytes a lane) into a ring of four units, two in use and two in flight (74 KB a CU,
// 19 MB over the chip); the stream runs on from one item of the share to the next. The page numbers travel the same way, three
// units ahead of the rows' loads, so that no load is ever waited for but in the order of the ring (one count, kLoads a unit).
// The latent parts of the rows and the rotary parts lie apart, so that one load instruction covers whole rows. Chunk c (16 bytes)
// of a latent part lies at c ^ row_swizzle(row): the rows' stride is a multiple of all 64 banks, and so the 16 rows of a score
// operand, and the 8 rows of half a transposing read, fall into different banks; a rotary part has 128 bytes whatever its
// width, chunk c at c ^ (row / 2) % 8.
__device__ __forceinline__ int row_swizzle(int row) { return ((row & 3) << 1) | (((row >> 3) & 1) << 3) | ((row >> 2) & 1); }

template <typename T>
__device__ __forceinline__ T ld_const(const T* p) {  // wave-uniform address: a scalar load
  return *(const __attribute__((address_space(4))) T*)p;
}

__device__ __forceinline__ const uint8_t* lane_ptr(uint64_t p, int lane) {  // a lane's pointer, wave-uniform
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)p, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(p >> 32), lane);
  return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// The items of a share one after the other: units of the current one and the length of its row.
struct Walk {
  const Item* items;
  int64_t left;   // units of the share after the current item
  int item, unit, units, len;
  __device__ __forceinline__ explicit Walk(const DecodeWs& w, const Share* s)
      : items(w.items), left(ld_const(&s->total) - ld_const(&s->left)), item(ld_const(&s->item)), unit(ld_const(&s->unit)),
        units(ld_const(&s->left)), len(ld_const(&s->len)) {}
  __device__ __forceinline__ int next() const {  // (only where left > 0)
    int x = item;
    do x++;
    while (ld_const(&items[x].len) == 0);
    return x;
  }
  __device__ __forceinline__ bool step() {
    if (left == 0) return false;
    item = next();
    len = ld_const(&items[item].len);
    unit = 0;
    units = (int)min((int64_t)((len + kUnit - 1) / kUnit), left);
    left -= units;
    return true;
  }
};

template <int DT, int R, int P, int HB>
__global__ __launch_bounds__(512, 2) void k_mla_attend(DecodeArgs d) {
  constexpr int kRing = 4;
  constexpr int kTpw = kUnit / 4;                      // rows that one of the four loading waves loads: 8, eight lanes for each
  constexpr int RC = R / 8, PC = P / 8;                // 16-byte chunks of the two parts of a row
  constexpr int kPer = 64 / RC;                        // latent parts of one load instruction: 1 or 2
  constexpr int kLoads = kTpw / kPer + 2;              // a wave's load instructions per unit: latents, rotary parts, page numbers
  constexpr int CB = R / 16 / 4;                       // 16-column blocks of a wave's sums
  static_assert(CB == kTpw / kPer, "a load instruction goes with each of them");
  __shared__ __align__(1024) uint8_t lat[kRing][kUnit * R * 2];
  __shared__ __align__(1024) uint8_t rot[kRing][kUnit * 128];
  __shared__ __align__(16) uint8_t prob[2][HB * 16 * kUnit * 2];  // [head][token], chunk c of a row at c ^ (head / 4) % 4
  __shared__ float fade[2][HB * 16];                   // factor of a head's earlier sums
  __shared__ float2 stats[2][HB * 16];                 // at the end of an item: a head's maximum and sum
  __shared__ __align__(16) float seen[kRing][kUnit];   // 1: the token is seen
  __shared__ __align__(16) int32_t page_no[kRing][4][kTpw];  // of the rows a wave loads
  __shared__ __align__(16) int32_t place[kRing][4][kTpw];    // their places in the pages, -1: not seen

  const vib3_mla_decode& a = d.a;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = head_groups(a.heads);
  const Share* sh = d.w.shares + blockIdx.x;
  if (ld_const(&sh->total) == 0) return;
  Walk at(d.w, sh);

  if (wave < 4) {
    if (wave >= HB) {
      for (int64_t k = ld_const(&sh->total); k >= 0; k--) __syncthreads();
      return;
    }
    const int g = lane >> 4, col = lane & 15, head_in_group = wave * 16 + col;
    const float scale = exponent_scale(a.scale), sign = a.scale < 0.0f ? -1.0f : 1.0f;
    // queries: the B operand, this lane's head at k = 32 s + 8 g; the latent part in two summands where
    // it was formed by W_uk
    constexpr int KS = (R + P) / 32;
    s16x8 q[KS], q_low[R / 32];
    auto load_q = [&](int x) {
      const int r = x / groups;
      const int64_t h = min((x - r * groups) * 64 + head_in_group, a.heads - 1);
      const uint16_t* ql = a.kv_b ? d.w.ql + ((size_t)r * a.heads + h) * 2 * R
                                  : (const uint16_t*)a.q_nope + r * a.q_nope_row_stride + h * a.q_nope_head_stride;
      const uint16_t* qr = (const uint16_t*)a.q_rope + r * a.q_rope_row_stride + h * a.q_rope_head_stride;
#pragma unroll
      for (int s = 0; s < KS; s++) q[s] = *(const s16x8*)(s < R / 32 ? ql + 32 * s + 8 * g : qr + 32 * (s - R / 32) + 8 * g);
      if (a.kv_b) {
#pragma unroll
        for (int s = 0; s < R / 32; s++) q_low[s] = *(const s16x8*)(ql + R + 32 * s + 8 * g);
      }
    };
    // this lane's row of a 16-token block; 16 rows further the swizzles are the same
    const int k0 = (g ^ row_swizzle(col)) * 16, r0 = (g ^ ((col >> 1) & 7)) * 16;
    load_q(at.item);
    int k = 0;  // unit of the share
    do {
      float m = -__builtin_huge_valf(), l = 0.0f;  // of this lane's head (unscaled scores); l over this lane's own tokens
      for (int i = 0; i < at.units; i++, k++) {
        __syncthreads();  // unit k is in LDS; the probabilities of unit k - 2 are done with
        const lds_u8* t = (lds_u8*)lat[k % kRing] + col * R * 2;
        const lds_u8* u = (lds_u8*)rot[k % kRing] + col * 128;
        f32x4 s[2] = {};
        auto latent_scores = [&](auto summands) {  // chunk (4 c + g) ^ row_swizzle(col), a constant and two bits away from that of c = 0
#pragma unroll
          for (int c = 0; c < R / 32; c++)
#pragma unroll
            for (int b = 0; b < 2; b++) {
              const s16x8 key = lds_read16(t + b * 32 * R + (k0 ^ c % 4 * 64) + c / 4 * 256);
              s[b] = mma32<DT>(key, q[c], s[b]);
              if (decltype(summands)::value == 2) s[b] = mma32<DT>(key, q_low[c], s[b]);
            }
        };
        // (queries that are latent already have no second summand, and its zeros would make NaN of an infinite latent)
        if (a.kv_b) latent_scores(std::integral_constant<int, 2>{});
        else latent_scores(std::integral_constant<int, 1>{});
#pragma unroll
        for (int c = 0; c < P / 32; c++)
#pragma unroll
          for (int b = 0; b < 2; b++) s[b] = mma32<DT>(lds_read16(u + b * 16 * 128 + (r0 ^ 64 * c)), q[R / 32 + c], s[b]);
        if (i + 1 == at.units && at.left > 0) load_q(at.next());  // on its way during what follows
        float top = -__builtin_huge_valf();
#pragma unroll
        for (int b = 0; b < 2; b++) {
          const float4 v = *(const float4*)&seen[k % kRing][b * 16 + 4 * g];
          const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; j++) {
            s[b][j] = vv[j] != 0.0f ? s[b][j] * sign : -__builtin_huge_valf();
            top = fmaxf(top, s[b][j]);
          }
        }
        top = max_over_rows(top);
        // The reference value of a head's exponentials follows its maximum only where that grew by more than kLag.
        const bool grown = (top - m) * scale > kLag<DT> || (m == -__builtin_huge_valf() && top > m);
        const float f = grown ? __builtin_amdgcn_exp2f((m - top) * scale) : 1.0f;
        m = grown ? top : m;
        l *= f;
        float base = m == -__builtin_huge_valf() ? 0.0f : m * scale;
        const bool far = __builtin_fabsf(base) > kFarExponent;
        if (__any(far)) {
          const float off = far ? m : 0.0f;
          base = far ? 0.0f : base;
#pragma unroll
          for (int b = 0; b < 2; b++) s[b] -= off;
        }
        base -= kProbShift<DT>;
        if (g == 0) fade[k & 1][head_in_group] = f;
#pragma unroll
        for (int b = 0; b < 2; b++) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; j++) e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][j], scale, -base));
          l += (e[0] + e[1]) + (e[2] + e[3]);
          // Rounded for the matrix cores; the sum l takes them unrounded. (A remainder as a second summand takes 8 KB more, of
          // which the ring leaves 5. Without it the result is off by 0.0017 to 0.0021 in bf16, a single rounding by 0.0017.)
          lds_write8((lds_u8*)prob[k & 1] + head_in_group * (kUnit * 2) + ((2 * b + (g >> 1)) ^ (col >> 2)) * 16 + 8 * (g & 1),
                     pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3]));
        }
      }
      const float sum = sum_over_rows(l);
      if (g == 0) stats[(k - 1) & 1][head_in_group] = make_float2(m, sum);
    } while (at.step());
    __syncthreads();
    return;
  }

  const int pw = wave - 4;
  // The stream of page numbers: a lane holds the token, page and place in the page of row lane % 8 of its wave's next rows.
  const int page_size = a.cache.page_size, page_step = kUnit / page_size, off_step = kUnit % page_size;
  const int my_row = pw * kTpw + (lane & 7);
  Walk ahead = at;
  int s_left = at.units;
  const int32_t* s_table = a.cache.block_table + (size_t)ld_const(&sh->seq) * a.cache.max_pages;
  int s_token = at.unit * kUnit + my_row;
  int s_page = s_token / page_size, s_off = s_token - s_page * page_size;
  // The next unit's page numbers into ring place k % kRing.
  auto look_up = [&](int k) {
    if (s_left == 0 && ahead.step()) {
      s_left = ahead.units;
      s_table = a.cache.block_table + (size_t)ld_const(&ahead.items[ahead.item].seq) * a.cache.max_pages;
      s_token = my_row;
      s_page = s_token / page_size;
      s_off = s_token - s_page * page_size;
    }
    const bool ok = s_left > 0 && s_token < ahead.len;
    const int32_t* p = ok ? s_table + s_page : (const int32_t*)zero_row;
    if (lane < kTpw) {
      place[k % kRing][pw][lane] = ok ? s_off : -1;
      load_to_lds4(p, (lds_u8*)page_no[k % kRing][pw]);
    }
    if (s_left > 0) {
      s_left--;
      s_token += kUnit;
      s_off += off_step;
      s_page += page_step;
      if (s_off >= page_size) {
        s_off -= page_size;
        s_page++;
      }
    }
  };
  // The addresses of unit k's rows, eight lanes for each (a row of zeros for those not seen, and once the stream is through).
  uint64_t row = 0;
  bool row_seen = false;
  auto aim = [&](int k) {
    const int id = page_no[k % kRing][pw][lane >> 3], off = place[k % kRing][pw][lane >> 3];
    row_seen = off >= 0 && (unsigned)id < (unsigned)a.cache.num_pages;
    row = row_seen ? (uint64_t)(uintptr_t)((const uint16_t*)a.cache.pool + (int64_t)id * a.cache.page_stride +
                                           (int64_t)off * a.cache.row_stride)
                   : (uint64_t)(uintptr_t)zero_row;
  };
  // One of the loads of the unit aimed at into ring place k % kRing: latent parts i * kPer on, or at the end the rotary parts.
  constexpr int kIssues = kTpw / kPer + 1;
  auto issue = [&](int k, int i) {
    const int slot = k % kRing;
    if (i < kIssues - 1) {
      const int t = i * kPer + (kPer == 2 ? lane >> 5 : 0);
      const uint8_t* p = lane_ptr(row, 8 * i * kPer);
      if (kPer == 2) {
        const uint8_t* p1 = lane_ptr(row, 8 * i * kPer + 8);
        p = lane >= 32 ? p1 : p;
      }
      load_to_lds16(p + ((fresh(lane) & (RC - 1)) ^ row_swizzle(pw * kTpw + t)) * 16, (lds_u8*)lat[slot] + (pw * kTpw + i * kPer) * R * 2);
    } else {
      const int ln = fresh(lane);
      const int c = (ln & 7) ^ ((ln >> 4) & 3) ^ (pw & 1) * 4;  // (row / 2) % 8 of row pw * 8 + lane / 8
      if (PC == 8 || c < PC) load_to_lds16((const uint8_t*)(uintptr_t)row + R * 2 + c * 16, (lds_u8*)rot[slot] + pw * kTpw * 128);
      if ((ln & 7) == 0) seen[slot][pw * kTpw + (ln >> 3)] = row_seen ? 1.0f : 0.0f;
    }
  };
  auto issue_all = [&](int k) {
#pragma unroll
    for (int i = 0; i < kIssues; i++) issue(k, i);
  };
  // Unit k's rows, and the page numbers of unit k + 3, have landed for this wave once no more than the next unit's loads are out.
  auto landed = [&] { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory"); };

  look_up(0);
  look_up(1);
  look_up(2);
  wait_lds_loads();
  aim(0);
  issue_all(0);
  look_up(3);
  aim(1);
  issue_all(1);
  look_up(4);
  aim(2);
  landed();
  __syncthreads();
  issue_all(2);
  look_up(5);
  aim(3);
  int k = 1;
  do {
    f32x4 o[HB][CB] = {};
    const bool starts_share = k == 1;
    for (int i = 0; i < at.units; i++, k++) {
      landed();
      __syncthreads();  // unit k and the probabilities of unit k - 1 are there; unit k - 2 is done with
      const int ln = fresh(lane), g = ln >> 4, col = ln & 15;
      // rows vrow and vrow + 4, chunk ch ^ vf of column block c: ch = 2 (pw CB + c) + (col % 4) / 2, and vf ^ 1 in the second row
      const int vrow = 8 * g + (col >> 2), vf = row_swizzle(vrow);
      lds_u8* t = (lds_u8*)lat[(k - 1) % kRing] + vrow * R * 2 + 8 * (col & 1) + pw * 2 * CB / 16 * 256;
      const int v0 = ((pw * 2 * CB % 16 + ((col & 3) >> 1)) ^ vf) * 16;
      auto latents = [&](int c) { return join(lds_read_tr(t + (v0 ^ 32 * c)), lds_read_tr(t + 8 * R + (v0 ^ 32 * c ^ 16))); };
      s16x8 pb[HB], av[CB];
      float f[HB];
      bool changed = false;
#pragma unroll
      for (int h = 0; h < HB; h++) f[h] = fade[(k - 1) & 1][h * 16 + col];
#pragma unroll
      for (int h = 0; h < HB; h++) pb[h] = lds_read16((lds_u8*)prob[(k - 1) & 1] + (h * 16 + col) * (kUnit * 2) + (g ^ (col >> 2)) * 16);
      av[0] = latents(0);
      av[1] = latents(1);
#pragma unroll
      for (int h = 0; h < HB; h++) changed |= f[h] != 1.0f;
      if (__any(changed)) {
#pragma unroll
        for (int h = 0; h < HB; h++)
#pragma unroll
          for (int c = 0; c < CB; c++) o[h][c] *= f[h];
      }
      // the products, with the loads of unit k + 2 spread among them
#pragma unroll
      for (int c = 0; c < CB; c++) {
        issue(k + 2, c);
        if (c + 2 < CB) av[c + 2] = latents(c + 2);
#pragma unroll
        for (int h = 0; h < HB; h++) o[h][c] = mma32<DT>(av[c], pb[h], o[h][c]);
      }
      issue(k + 2, CB);
      look_up(k + 5);
      aim(k + 3);
    }
    const int r = at.item / groups, h0 = (at.item - r * groups) * 64;
    const int col = fresh(lane) & 15, c0 = pw * CB * 16 + 4 * (fresh(lane) >> 4);
    const float2* st = stats[k & 1];  // of unit k - 2, the item's last
    if (at.unit == 0 && at.units == (at.len + kUnit - 1) / kUnit) {
      float* out = d.w.ol + ((size_t)r * padded_heads(a.heads) + h0 + col) * R + c0;
#pragma unroll
      for (int h = 0; h < HB; h++) {
        const float sum = st[h * 16 + col].y;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int c = 0; c < CB; c++)
          *(float4*)(out + h * 16 * R + 16 * c) = make_float4(o[h][c][0] * inv, o[h][c][1] * inv, o[h][c][2] * inv, o[h][c][3] * inv);
      }
    } else {
      const size_t slot = blockIdx.x + (starts_share ? 0 : kShares);
      float* out = d.w.part + slot * (HB * 16 * R + kSlotGap) + col * R + c0;
#pragma unroll
      for (int h = 0; h < HB; h++)
#pragma unroll
        for (int c = 0; c < CB; c++) *(float4*)(out + h * 16 * R + 16 * c) = make_float4(o[h][c][0], o[h][c][1], o[h][c][2], o[h][c][3]);
      if (pw == 0 && lane < HB * 16) d.w.stat[lane * (2 * kShares) + slot] = st[lane];
    }
  } while (at.step());
  wait_lds_loads();  // those of the stream's empty end: not into LDS that is no longer this workgroup's
}

// ------------------------------------------------------------------------- joined rows and W_uv

// A workgroup takes up to 16 rows of one head. Its 16 waves are dealt over the rows: a wave, or where there are fewer rows
// several, joins a row's parts. Their statistics and the first parts' sums are read at the same time (a part's place does not
// depend on its weight). The rows' weighted latents go to LDS in two 16-bit summands (a rounding alone would show in the result, see
// k_mla_absorb), and v_dim / 16 waves multiply them by 16 rows of W_uv each. Without W_uv the weighted latents are the result.
// Bound by latency: the plan, the parts, W_uv, one after the other; 64 registers a lane let two workgroups share a CU, so that
// up to 512 run at once. 8 us for one short row of 64 heads, 16 where 256 parts (34 MB) are joined, 20 for 96 rows.
template <int DT, int R>
__global__ __launch_bounds__(1024, 8) void k_mla_finish(DecodeArgs d) {
  const vib3_mla_decode& a = d.a;
  constexpr int kStride = R + 8;  // 16 bytes more: rows start in different banks
  constexpr int kCols = R / 64;   // columns of a lane
  constexpr int kAhead = 4;       // parts in flight
  __shared__ __align__(16) uint16_t lat[16 * kStride];
  __shared__ __align__(16) float sums[16][R];
  // weights of the parts of a wave's row; later the weighted latents' remainders
  __shared__ __align__(16) uint8_t both[16 * (kStride * 2 > kShares * 4 ? kStride * 2 : kShares * 4)];
  float(*const weight)[kShares] = (float(*)[kShares])both;
  uint16_t* const lat_low = (uint16_t*)both;
  const int h = (int)blockIdx.x, r0 = (int)blockIdx.y * 16;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = min(16, a.rows - r0);
  const int teams = rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows;  // rows joined at a time
  const int per_row = 16 / teams, i = wave / per_row, mate = wave % per_row;
  {
    const int r = r0 + i, x = r * head_groups(a.heads) + h / 64;
    float o[kCols] = {};
    const int64_t per = ld_const(d.w.head);
    const int64_t lo = i < rows ? ld_const(&d.w.items[x].begin) : 0, hi = i < rows ? ld_const(&d.w.items[x + 1].begin) : 0;
    if (hi > lo) {
      const int w0 = (int)((lo + kItemCost) / per), parts = (int)((hi - 1) / per) - w0 + 1;
      if (parts == 1) {
        if (mate == 0) {
          const float* p = d.w.ol + ((size_t)r * padded_heads(a.heads) + h) * R + lane * kCols;
#pragma unroll
          for (int c = 0; c < kCols; c += 4) *(float4*)(o + c) = *(const float4*)(p + c);
        }
      } else {
        // part j: slot w0 + j, but the first one kShares + w0 where its share began with another item
        const bool late = w0 * per < lo;
        const int hg = group_heads(a.heads), hh = h % 64;
        auto slot = [&](int j) { return (size_t)(w0 + j + (j == 0 && late ? kShares : 0)); };
        float2 st[kShares / 64];  // lane l: parts l, l + 64, ... (asked for first: loads come back in order)
#pragma unroll
        for (int k = 0; k < kShares / 64; k++) {
          st[k] = make_float2(-__builtin_huge_valf(), 0.0f);
          if (lane + 64 * k < parts) st[k] = d.w.stat[hh * (2 * kShares) + slot(lane + 64 * k)];
        }
        // kAhead parts at a time, without a branch around a load (past the end: the last one again, with weight 0)
        float4 v[kAhead][kCols / 4];
        auto fetch = [&](int j0) {
#pragma unroll
          for (int k = 0; k < kAhead; k++) {
            const float* p = d.w.part + slot(min(j0 + k * per_row, parts - 1)) * (hg * R + kSlotGap) + hh * R + lane * kCols;
#pragma unroll
            for (int c = 0; c < kCols / 4; c++) v[k][c] = *(const float4*)(p + 4 * c);
          }
        };
        fetch(mate);
        float m = fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x)), l = 0.0f;
#pragma unroll
        for (int s = 1; s < 64; s *= 2) m = fmaxf(m, __shfl_xor(m, s));
        const float base = m == -__builtin_huge_valf() ? 0.0f : m, scale = exponent_scale(a.scale);
#pragma unroll
        for (int k = 0; k < kShares / 64; k++) {
          st[k].x = __builtin_amdgcn_exp2f((st[k].x - base) * scale);
          l += st[k].x * st[k].y;
        }
        l = wave_sum(l);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int k = 0; k < kShares / 64; k++) weight[wave][lane + 64 * k] = st[k].x * inv;
        for (int j0 = mate;;) {
#pragma unroll
          for (int k = 0; k < kAhead; k++) {
            const int j = j0 + k * per_row;
            const float f = j < parts ? weight[wave][j] : 0.0f;
            if (f == 0.0f) continue;  // (a weight of 0 says nothing about what lies there)
#pragma unroll
            for (int c = 0; c < kCols / 4; c++) {
              o[4 * c] += f * v[k][c].x;
              o[4 * c + 1] += f * v[k][c].y;
              o[4 * c + 2] += f * v[k][c].z;
              o[4 * c + 3] += f * v[k][c].w;
            }
          }
          j0 += kAhead * per_row;
          if (j0 >= parts) break;
          fetch(j0);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kCols; c += 4) *(float4*)&sums[wave][lane * kCols + c] = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
  }
  // half of the W_uv rows of this wave meanwhile
  const int g = lane >> 4, col = lane & 15;
  const bool product = a.kv_b && wave * 16 < a.v_dim;
  const uint16_t* wv = (const uint16_t*)a.kv_b + ((size_t)h * (a.nope + a.v_dim) + a.nope + wave * 16 + col) * R + 8 * g;
  s16x8 first[R / 64];
#pragma unroll
  for (int k = 0; k < R / 64; k++) first[k] = product ? *(const s16x8*)(wv + k * 32) : s16x8{};
  __syncthreads();
  for (int at = tid; at < rows * R; at += 1024) {
    const int k = at / R, c = at % R;
    float v = 0.0f;
    for (int s = 0; s < per_row; s++) v += sums[k * per_row + s][c];
    if (a.kv_b) {
      const Halves x = split2<DT>(v, 0.0f);
      lat[k * kStride + c] = (uint16_t)x.hi;
      lat_low[k * kStride + c] = (uint16_t)x.lo;
    } else
      ((uint16_t*)a.out)[(int64_t)(r0 + k) * a.out_row_stride + (int64_t)h * a.out_head_stride + c] = from_f32<DT>(v);
  }
  if (!a.kv_b) return;
  __syncthreads();
  if (!product) return;
  const int row = min(col, rows - 1);
  f32x4 acc = {};
  // rows of W_uv times the rows' latents: a lane ends with 4 outputs of one row
#pragma unroll
  for (int k = 0; k < R / 32; k++) {
    const s16x8 w = k < R / 64 ? first[k] : *(const s16x8*)(wv + k * 32);
    acc = mma32<DT>(w, *(const s16x8*)(lat + row * kStride + k * 32 + 8 * g), acc);
    acc = mma32<DT>(w, *(const s16x8*)(lat_low + row * kStride + k * 32 + 8 * g), acc);
  }
  if (col < rows)
    *(uint2*)((uint16_t*)a.out + (int64_t)(r0 + col) * a.out_row_stride + (int64_t)h * a.out_head_stride + wave * 16 + 4 * g) =
        make_uint2(pack2<DT>(acc[0], acc[1]), pack2<DT>(acc[2], acc[3]));
}

template <int DT, int R, int P>
int launch_decode(const DecodeArgs& d, hipStream_t st) {
  const vib3_mla_decode& a = d.a;
  if (a.kv_b) {
    const int col_blocks = R / kAbsorbCols;
    hipLaunchKernelGGL(k_mla_absorb<DT>, dim3((unsigned)(a.heads * col_blocks + 1), (unsigned)((a.rows + kAbsorbRows - 1) / kAbsorbRows)), dim3(256),
                       (unsigned)(a.nope * kAbsorbCols * 2), st, d, col_blocks);
  } else {
    hipLaunchKernelGGL(k_mla_plan, dim3(1), dim3(256), 0, st, d);
  }
  if (a.heads <= 16)
    hipLaunchKernelGGL((k_mla_attend<DT, R, P, 1>), dim3(kShares), dim3(512), 0, st, d);
  else if (a.heads <= 32)
    hipLaunchKernelGGL((k_mla_attend<DT, R, P, 2>), dim3(kShares), dim3(512), 0, st, d);
  else
    hipLaunchKernelGGL((k_mla_attend<DT, R, P, 4>), dim3(kShares), dim3(512), 0, st, d);
  hipLaunchKernelGGL((k_mla_finish<DT, R>), dim3((unsigned)a.heads, (unsigned)((a.rows + 15) / 16)), dim3(1024), 0, st, d);
  VIB3_RETURN_LAUNCH();
}

template <int DT>
int launch_decode_dt(const DecodeArgs& d, hipStream_t st) {
  if (d.a.cache.rank == 512)
    return d.a.cache.rope == 64 ? launch_decode<DT, 512, 64>(d, st) : launch_decode<DT, 512, 32>(d, st);
  return d.a.cache.rope == 64 ? launch_decode<DT, 256, 64>(d, st) : launch_decode<DT, 256, 32>(d, st);
}

bool decode_counts(const vib3_mla_decode& a) {
  return a.rows >= 0 && a.rows <= kMlaMaxRows && a.heads >= 1 && a.heads <= 128;
}

}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_mla_decode_workspace_bytes(const vib3_mla_decode* args) {
  if (!args || !decode_counts(*args) || (args->cache.rank != 256 && args->cache.rank != 512)) return 0;
  vib3_mla_decode a = *args;
  a.kv_b = &a;  // the larger of the two forms
  return decode_ws(a, nullptr, nullptr);
}

extern "C" int vib3_launch_mla_decode(const vib3_mla_decode* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_mla_decode& a = *args;
  if (const int rc = check_cache(a.cache)) return rc;
  if (!decode_counts(a)) return VIB3_ERR_BAD_COUNT;
  if (!__builtin_isfinite(a.scale)) return VIB3_ERR_UNSUPPORTED;
  if (a.kv_b && (a.nope < 32 || a.nope > 256 || a.nope % 32 || a.v_dim < 32 || a.v_dim > 256 || a.v_dim % 32))
    return VIB3_ERR_UNSUPPORTED;
  if (a.rows == 0) return 0;
  if (!a.lens || !mla_aligned(a.q_nope) || !mla_aligned(a.q_rope) || !mla_aligned(a.out) ||
      (a.kv_b && !mla_aligned(a.kv_b)) || !mla_stride(a.q_nope_row_stride) || !mla_stride(a.q_nope_head_stride) ||
      !mla_stride(a.q_rope_row_stride) || !mla_stride(a.q_rope_head_stride) || !mla_stride(a.out_row_stride) ||
      !mla_stride(a.out_head_stride) || !a.workspace || ((uintptr_t)a.workspace & 255))
    return VIB3_ERR_BAD_POINTER;
  if (a.workspace_bytes < vib3_mla_decode_workspace_bytes(args)) return VIB3_ERR_WORKSPACE;
  DecodeArgs d;
  d.a = a;
  decode_ws(a, &d.w, a.workspace);
  return a.cache.dtype == VIB3_DT_F16 ? launch_decode_dt<VIB3_DT_F16>(d, (hipStream_t)stream)
                                      : launch_decode_dt<VIB3_DT_BF16>(d, (hipStream_t)stream);
}
