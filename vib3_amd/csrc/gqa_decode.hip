// gqa_decode.hip — attention of single query tokens over the paged key/value cache.
//
// Bound by the bytes of the cache: a key and a value of dim 16-bit elements serve heads / kv_heads queries, 4 flops a byte and query.
// Two launches:
//   k_gqa_attend   the attention, over equal shares of all rows' visible tokens
//   k_gqa_join     rows that several shares were needed for, and those in which something is NaN once more
//
// The shares: tokens are taken 32 at a time, 64 for heads of 64 (a unit). All units of all rows in order, with kRowCost units' time in front of each row
// for taking it up and storing its sums, are cut into equal runs, whatever the rows' lengths. A run is walked by one wave per
// key/value head (and per 16 heads of its group), all by themselves: there is no barrier after the plan, which every workgroup
// forms anew from the lengths (a scan of an int a row). Nothing on the host depends on the lengths, so a captured launch follows
// them.
//
// A wave holds the keys of a unit as it gets them from memory, as the matrix cores' A operand (S^T = K . Q^T, the group's heads are
// the columns), so that a lane has the scores of 8 of 32 tokens and one head; packed in pairs of 16 bits they are, as they stand, the B
// operand of O^T = V^T . P^T (the tokens' order along k is free as long as V^T is read in the same one). Values pass through the
// wave's own rows of LDS, from where transposing reads take V^T. The next unit's keys and values are on their way
// meanwhile, and the page numbers of the one after that.
//
// Measured (attention + joining): 61 rows of 300 to 50000 tokens, 32 heads over 8 of 128: 430 + 7 us, 5.8 TB/s (a kernel that only reads gets
// 6.0); one row of 901 tokens 9 + 5, launches and dependent reads (length, page number, tokens; place, parts). 97 rows of 64 heads over 8 of 64
// with a window of 4096: 55 + 6; with 32 tokens a step and 16 waves 59 + 6, which spilled registers. Equal shares against a workgroup
// per row and head: 440 us against 56 ms for the 61 rows. Groups above 16 heads are streamed once for each 16: the 61 rows with 16, 32 and
// 48 heads over one of 128 (312 MB, 52 us at 6.0 TB/s) 80, 101 and 138 us.
#include <type_traits>

#include "gqa.h"
#include "scan.h"

namespace vib3 {
namespace {  // the names below are this file's: other files have a decode_ws or a launch_decode_dt of their own

constexpr int kGqaMaxRows = 65536;
constexpr int kRowCost = 2;   // a row's fixed time, in units
constexpr int kWorkgroups = 256;

// Tokens of one step, and waves of a workgroup: as many as their registers leave room for.
__host__ __device__ constexpr int unit_tokens(int dim) { return dim == 64 ? 64 : 32; }
__host__ __device__ constexpr int attend_waves(int dim) { return dim == 256 ? 4 : 8; }

// What a wave takes of the heads: 16 of a group at most.
struct Heads {
  int group, cols, parts, units;  // heads a key/value head, columns of a wave, waves a group, waves a run
};
__host__ __device__ inline Heads split_heads(int heads, int kv_heads) {
  Heads h;
  h.group = heads / kv_heads;
  h.cols = h.group < 16 ? h.group : 16;
  h.parts = (h.group + 15) / 16;
  h.units = kv_heads * h.parts;
  return h;
}

// Runs: a wave for each (run, unit of heads), at most kWorkgroups workgroups of them (or one run).
__host__ __device__ inline int run_count(const Heads& h, int dim) {
  const int n = kWorkgroups * attend_waves(dim) / h.units;
  return n < 1 ? 1 : n;
}

// Device workspace. Slot w of the parts (w = run * units + unit of heads) holds that of the row that the run starts with (where it
// does not cover all of it), slot runs * units + w that of the row it ends in, if that is another one.
struct DecodeWs {
  int64_t* head;    // length of a run, in units and fixed times
  int64_t* begin;   // [rows + 1] where the rows begin
  float* part;      // [2][runs][units][cols][dim] unnormalised sums
  float2* stat;     // [2][runs][units][cols] reference value (of unscaled scores) and sum
};

inline size_t decode_ws(const vib3_gqa_decode& a, DecodeWs* w, void* base) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return (uint8_t*)base + p;
  };
  const Heads h = split_heads(a.heads, a.cache.kv_heads);
  const size_t slots = 2 * (size_t)run_count(h, a.cache.dim) * h.units;
  DecodeWs r;
  r.head = (int64_t*)take(8);
  r.begin = (int64_t*)take(8 * ((size_t)a.rows + 1));
  r.part = (float*)take(4 * slots * h.cols * a.cache.dim);
  r.stat = (float2*)take(8 * slots * h.cols);
  if (w) *w = r;
  return at;
}

struct DecodeArgs {
  vib3_gqa_decode a;
  DecodeWs w;
  Heads h;
  int runs;
};

// a / b (exact below 2^42 where it is below 2^11: the quotient's distance from the next integer is more than its rounding).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) { return (int64_t)((double)a / (double)b); }

// What the query of a row sees, in units: `skip` units from the first token on (those with sinks), then from unit `first` to the end.
template <int UNIT>
struct Seen {
  int seq, len, start;        // visible are the tokens from start and the first sinks, to len
  int skip, first, units;
  __device__ __forceinline__ int token(int u) const { return (u < skip ? u : first + u - skip) * UNIT; }
};

template <int UNIT>
__device__ __forceinline__ Seen<UNIT> row_seen(const vib3_gqa_decode& a, int r) {
  Seen<UNIT> s;
  s.seq = a.seqs ? a.seqs[r] : r;
  s.len = (unsigned)s.seq < (unsigned)a.cache.num_seqs ? gqa_len(a.cache, a.lens[r]) : 0;
  s.start = s.len > 0 ? window_start(s.len - 1, a.window) : 0;
  s.first = s.start / UNIT;
  s.skip = min((min(a.sinks, s.start) + UNIT - 1) / UNIT, s.first);
  s.units = (s.len + UNIT - 1) / UNIT - s.first + s.skip;
  return s;
}

// A row's extent in the order of all: a row that sees nothing has none.
template <int UNIT>
__device__ __forceinline__ int64_t row_extent(const vib3_gqa_decode& a, int r) {
  const int n = r < a.rows ? row_seen<UNIT>(a, r).units : 0;
  return n > 0 ? n + kRowCost : 0;
}

// Sum over the lanes up to this one (of values from 0 to 2^40).
__device__ __forceinline__ int64_t scan64(int64_t v) {
  return ((int64_t)add_up((int)(v >> 16)) << 16) + add_up((int)(v & 0xffff));
}

// v of lane i (the same in all lanes), as a value that is known to be uniform.
__device__ __forceinline__ int64_t uniform64(int64_t v, int i) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, i);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), i);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// 16 bytes of global memory, and an int that is the same in all lanes and not written while the kernel runs.
__device__ __forceinline__ s16x8 ld_global16(uint64_t p) { return *(const __attribute__((address_space(1))) s16x8*)p; }
__device__ __forceinline__ int ld_global4(const int32_t* p) { return *(const __attribute__((address_space(1))) int32_t*)(uint64_t)p; }

// What tokens that are not seen are read from.
__device__ const uint4 zero_token[256 / 8] = {};

// Two probabilities as pairs of 16-bit elements: cut off (towards 0), and what that left, rounded (in bf16 off by at most 2^-15 of the
// number, in f16 by 2^-21 of it or 2^-25). No remainder is negative, and in bf16 none is 0, so that an infinity times both stays one;
// in f16 the smallest number is too large for that, and the NaN is looked into where rows are joined.
template <int DT>
__device__ __forceinline__ Halves cut2(float a, float b) {
  if (DT == VIB3_DT_F16) {
    const auto hi = __builtin_amdgcn_cvt_pkrtz(a, b);
    return Halves{__builtin_bit_cast(uint32_t, hi), pack2<DT>(a - (float)hi[0], b - (float)hi[1])};
  }
  const uint32_t u = __float_as_uint(a) & 0xffff0000u, w = __float_as_uint(b) & 0xffff0000u;
  return Halves{u >> 16 | w, pack2<DT>(fmaxf(a - __uint_as_float(u), 0x1p-120f), fmaxf(b - __uint_as_float(w), 0x1p-120f))};
}

template <int DT, int D>
__global__ __launch_bounds__(attend_waves(D) * 64) void k_gqa_attend(DecodeArgs d) {
  constexpr int WAVES = attend_waves(D);
  constexpr int KS = D / 32;  // k steps of the scores
  constexpr int VB = D / 16;  // 16-row blocks of the sums
  constexpr int UNIT = unit_tokens(D), TB = UNIT / 16;  // 16-token blocks of a step
  __shared__ __align__(1024) uint8_t vtile[WAVES][UNIT * D * 2];
  __shared__ int64_t group_sum[kGqaMaxRows / 64];
  const vib3_gqa_decode& a = d.a;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // the plan: extents of 64 rows at a time, then their sum and where this wave's run begins
  const int row_groups = (a.rows + 63) / 64;
  for (int k = wave; k < row_groups; k += WAVES) {
    const int64_t n = scan64(row_extent<UNIT>(a, 64 * k + lane));
    if (lane == 63) group_sum[k] = n;
  }
  __syncthreads();
  const bool planner = blockIdx.x + 1 == gridDim.x;  // writes down the rows' places, for the rows' joining
  int64_t all = 0;
  for (int k = 0; k < row_groups; k += 64) {
    const int64_t n = k + lane < row_groups ? group_sum[k + lane] : 0, upto = scan64(n) + all;
    if (planner)
      for (int i = wave; i < 64 && k + i < row_groups; i += WAVES) {
        const int r = 64 * (k + i) + lane;
        const int64_t x = row_extent<UNIT>(a, r), at = uniform64(upto - n, i) + scan64(x) - x;
        if (r < a.rows) d.w.begin[r] = at;
      }
    all = uniform64(upto, 63);
  }
  const int64_t per = max((int64_t)1, quotient(all + d.runs - 1, d.runs));
  if (planner) {
    if (tid == 0) {
      d.w.begin[a.rows] = all;
      *d.w.head = per;
    }
    return;
  }
  const int worker = (int)blockIdx.x * WAVES + wave;
  const int run = worker / d.h.units, hu = worker - run * d.h.units;
  const int64_t from = run * per, to = min(from + per, all);
  if (run >= d.runs || from >= all) return;
  int row = 0;
  int64_t begin = 0;
  for (int k = 0; k < row_groups; k += 64) {
    const int64_t n = k + lane < row_groups ? group_sum[k + lane] : 0, upto = scan64(n) + begin;
    const uint64_t hit = __ballot(from < upto);
    if (hit) {
      const int i = __ffsll((unsigned long long)hit) - 1;
      begin = uniform64(upto - n, i);
      const int64_t x = row_extent<UNIT>(a, 64 * (k + i) + lane), end = scan64(x) + begin;
      const int j = __ffsll((unsigned long long)__ballot(from < end)) - 1;
      begin = uniform64(end - x, j);
      row = 64 * (k + i) + j;
      break;
    }
    begin = uniform64(upto, 63);
  }

  const int g = lane >> 4, col = lane & 15;
  const int kv_head = hu / d.h.parts, head0 = kv_head * d.h.group + (hu - kv_head * d.h.parts) * 16;
  const int cols = min(16, (kv_head + 1) * d.h.group - head0);
  const float scale = exponent_scale(a.scale);
  const uint32_t flip = sign_flip(a.scale);
  const uint64_t kbase = (uint64_t)a.cache.keys + 2 * (kv_head * a.cache.head_stride + 8 * g);
  const uint64_t vbase = (uint64_t)a.cache.values + 2 * (kv_head * a.cache.head_stride + 8 * g);
  const uint64_t zbase = (uint64_t)zero_token + 16 * g;

  // The stream of units, two steps ahead of the products: page numbers, then addresses and loads.
  Seen<UNIT> ahead = row_seen<UNIT>(a, row);  // the row of the unit that page numbers are asked for next
  int ahead_row = row;
  int64_t ahead_begin = begin;
  int ahead_u = (int)max((int64_t)0, from - begin - kRowCost);
  int ahead_end = (int)min((int64_t)ahead.units, to - begin - kRowCost);
  int page_no[TB], place[TB];  // of this lane's tokens; place -1: not seen
  bool more = true;          // whether the unit that was asked for is one of the run
  auto ask = [&] {
    while (ahead_u >= ahead_end) {  // the next row
      ahead_begin += ahead.units > 0 ? ahead.units + kRowCost : 0;
      ahead_row++;
      if (ahead_begin + kRowCost >= to) {
        more = false;
#pragma unroll
        for (int b = 0; b < TB; b++) place[b] = -1;
        return;
      }
      ahead = row_seen<UNIT>(a, ahead_row);
      ahead_u = 0;
      ahead_end = (int)min((int64_t)ahead.units, to - ahead_begin - kRowCost);
    }
    const int t0 = ahead.token(ahead_u) + col;
    const int32_t* table = a.cache.block_table + (size_t)ahead.seq * a.cache.max_pages;
#pragma unroll
    for (int b = 0; b < TB; b++) {
      const int t = t0 + 16 * b;
      const bool ok = t < ahead.len && (t >= ahead.start || t < a.sinks);
      const int page = ok ? t / a.cache.page_size : 0;  // (by multiplication heads of 64 and 128 gain 0.5 %, those of 256 lose 5)
      place[b] = ok ? t - page * a.cache.page_size : -1;
      page_no[b] = ld_global4(table + page);
    }
    ahead_u++;
  };
  using Mask = std::conditional_t<TB == 4, uint64_t, uint32_t>;
  // Loads of the unit that was asked for: this lane's chunks g + 4 c of its two tokens. Returns the mask of the tokens that are seen.
  auto load = [&](s16x8 (*k)[KS], s16x8 (*v)[KS]) -> Mask {
    Mask mask = 0;
#pragma unroll
    for (int b = 0; b < TB; b++) {
      const bool ok = place[b] >= 0 && (unsigned)page_no[b] < (unsigned)a.cache.num_pages;
      mask |= (Mask)(__ballot(ok) & 0xffff) << (16 * b);
      const uint64_t at = 2 * ((int64_t)page_no[b] * a.cache.page_stride + (int64_t)place[b] * a.cache.token_stride);
      const uint64_t ka = ok ? kbase + at : zbase, va = ok ? vbase + at : zbase;
#pragma unroll
      for (int c = 0; c < KS; c++) k[b][c] = ld_global16(ka + 64 * c);
#pragma unroll
      for (int c = 0; c < KS; c++) v[b][c] = ld_global16(va + 64 * c);
    }
    return mask;
  };

  // 16-byte chunk c of row r of the values lies at c ^ swizzle(r): a transposing read takes 32 bytes of each of 8 rows
  auto swizzle = [](int r) { return D == 64 ? (r & 6) : (r & 7) * 2; };
  lds_u8* const tile = (lds_u8*)vtile[wave];
  lds_u8* const put = tile + col * D * 2;
  const int put0 = (g ^ swizzle(col)) * 16;
  const int vrow = 4 * g + (col >> 2);
  lds_u8* const get = tile + vrow * D * 2 + 8 * (col & 1);
  const int get0 = (((col & 3) >> 1) ^ swizzle(vrow)) * 16;

  Seen<UNIT> at = ahead;
  int u = ahead_u, end = ahead_end;
  ask();
  if (!more) return;
  s16x8 k[2][TB][KS], v[2][TB][KS];
  Mask mask[2];
  mask[0] = load(k[0], v[0]);
  ask();
  bool first_row = true;
  // (a run may begin within a row's fixed time or end there: rows without units of the run are stepped over, as in ask())
  while (true) {
    while (u >= end) {
      begin += at.units > 0 ? at.units + kRowCost : 0;
      row++;
      first_row = false;
      if (begin + kRowCost >= to) return;
      at = row_seen<UNIT>(a, row);
      u = 0;
      end = (int)min((int64_t)at.units, to - begin - kRowCost);
    }
    const bool whole = u == 0 && end == at.units;
    s16x8 q[KS];
    {
      const uint64_t p = (uint64_t)a.q + 2 * (row * a.q_row_stride + (head0 + min(col, cols - 1)) * a.q_head_stride + 8 * g);
#pragma unroll
      for (int c = 0; c < KS; c++) {
        uint4 w = __builtin_bit_cast(uint4, ld_global16(p + 64 * c));
        w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
        q[c] = __builtin_bit_cast(s16x8, w);
      }
    }
    f32x4 o[VB] = {};
    float m = -__builtin_huge_valf(), l = 0.0f;  // of this lane's head (unscaled scores); l over this lane's own tokens
    auto step = [&](s16x8 (*kc)[KS], s16x8 (*vc)[KS], Mask seen, s16x8 (*kn)[KS], s16x8 (*vn)[KS], Mask* next) {
      if (more) {
        *next = load(kn, vn);
        ask();
      }
      f32x4 s[TB] = {};
#pragma unroll
      for (int c = 0; c < KS; c++)
#pragma unroll
        for (int b = 0; b < TB; b++) s[b] = mma32<DT>(kc[b][c], q[c], s[b]);
#pragma unroll
      for (int b = 0; b < TB; b++)
#pragma unroll
        for (int c = 0; c < KS; c++) *(__attribute__((address_space(3))) s16x8*)(put + 16 * b * D * 2 + (put0 ^ 64 * c)) = vc[b][c];
      if (seen != (Mask)~(Mask)0) {
#pragma unroll
        for (int b = 0; b < TB; b++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (!(seen >> (16 * b + 4 * g + i) & 1)) s[b][i] = -__builtin_huge_valf();
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < TB; b++) top = fmaxf(top, fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])));
      top = max_over_rows(top);
      // The reference value of a head's exponentials follows its maximum only where that grew by more than kLag.
      const bool grown = (top - m) * scale > kLag<DT> || (m == -__builtin_huge_valf() && top > m);
      if (__any(grown)) {
        const float f = grown ? __builtin_amdgcn_exp2f((m - top) * scale) : 1.0f;
        m = grown ? top : m;
        l *= f;
#pragma unroll
        for (int b = 0; b < VB; b++) o[b] *= f;
      }
      float base = m == -__builtin_huge_valf() ? 0.0f : m * scale;
      const bool far = __builtin_fabsf(base) > kFarExponent;
      if (__any(far)) {
        const float off = far ? m : 0.0f;
        base = far ? 0.0f : base;
#pragma unroll
        for (int b = 0; b < TB; b++) s[b] -= off;
      }
      base -= kProbShift<DT>;
      uint32_t p[2 * TB], r[2 * TB];
#pragma unroll
      for (int b = 0; b < TB; b++) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], scale, -base));
        l += (e[0] + e[1]) + (e[2] + e[3]);
        // In two summands: as one rounded number a result is off by 0.0023 in bf16 (root mean square over the 61 rows), so by 0.0017, as a
        // result that is rounded once. The second product costs at most 1 % (the 61 rows 438.4 -> 439.5 us), as the cache is waited for.
        const Halves first = cut2<DT>(e[0], e[1]), second = cut2<DT>(e[2], e[3]);
        p[2 * b] = first.hi, p[2 * b + 1] = second.hi;
        r[2 * b] = first.lo, r[2 * b + 1] = second.lo;
      }
#pragma unroll
      for (int t = 0; t < TB; t += 2) {
        const s16x8 prob = __builtin_bit_cast(s16x8, make_uint4(p[2 * t], p[2 * t + 1], p[2 * t + 2], p[2 * t + 3]));
        const s16x8 rest = __builtin_bit_cast(s16x8, make_uint4(r[2 * t], r[2 * t + 1], r[2 * t + 2], r[2 * t + 3]));
        lds_u8* const x = get + 16 * t * D * 2;
#pragma unroll
        for (int b = 0; b < VB; b++) {
          const s16x8 value = join(lds_read_tr(x + (get0 ^ 32 * b)), lds_read_tr(x + 16 * D * 2 + (get0 ^ 32 * b)));
          o[b] = mma32<DT>(value, prob, o[b]);
          o[b] = mma32<DT>(value, rest, o[b]);
        }
      }
    };
    for (; u < end; u++) {
      step(k[0], v[0], mask[0], k[1], v[1], &mask[1]);
#pragma unroll
      for (int b = 0; b < TB; b++)
#pragma unroll
        for (int c = 0; c < KS; c++) {
          k[0][b][c] = k[1][b][c];
          v[0][b][c] = v[1][b][c];
        }
      mask[0] = mask[1];
    }
    const float sum = sum_over_rows(l);
    if (whole) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint16_t* to_out = (uint16_t*)a.out + (int64_t)row * a.out_row_stride + (int64_t)(head0 + col) * a.out_head_stride + 4 * g;
      if (col < cols) {
#pragma unroll
        for (int b = 0; b < VB; b++)
          *(uint2*)(to_out + 16 * b) = make_uint2(pack2<DT>(o[b][0] * inv, o[b][1] * inv), pack2<DT>(o[b][2] * inv, o[b][3] * inv));
      }
    } else if (col < cols) {
      const size_t slot = (size_t)worker + (first_row ? 0 : (size_t)d.runs * d.h.units);
      float* part = d.w.part + (slot * d.h.cols + col) * D + 4 * g;
#pragma unroll
      for (int b = 0; b < VB; b++) *(float4*)(part + 16 * b) = make_float4(o[b][0], o[b][1], o[b][2], o[b][3]);
      if (g == 0) d.w.stat[slot * d.h.cols + col] = make_float2(m, sum);
    }
  }
}

// ------------------------------------------------------------------------- joined rows

// What values hold that is not finite, in the 8 elements of a chunk (packed as they are): `up` and `down` are 0 where there was an
// infinity of that sign, `nan` is not 0 where there was a NaN. top: what such an element's magnitude begins with.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <int DT>
struct Odd {
  static constexpr uint16_t top = DT == VIB3_DT_F16 ? 0x7c00 : 0x7f80;
  u16x2 up[4], down[4], nan[4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 4; i++) up[i] = down[i] = u16x2{0xffff, 0xffff}, nan[i] = u16x2{0, 0};
  }
  // A value whose probability is 0 or not: 0 times an infinity is NaN.
  __device__ __forceinline__ void add(uint4 v, bool zero) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const uint16_t most = zero ? top - 1 : top, off = zero ? 0xffff : 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const u16x2 x = __builtin_bit_cast(u16x2, w[i]), size = x & (uint16_t)0x7fff;
      up[i] = __builtin_elementwise_min(up[i], (x ^ top) | off);
      down[i] = __builtin_elementwise_min(down[i], (x ^ (uint16_t)(top | 0x8000)) | off);
      nan[i] = __builtin_elementwise_max(nan[i], __builtin_elementwise_max(size, u16x2{most, most}) - most);
    }
  }
  // Bit i for an infinity above 0 in element i, bit 8 + i for one below, bit 16 + i for a NaN.
  __device__ __forceinline__ uint32_t bits() const {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) b |= ((up[i / 2][i % 2] ? 0 : 1u) | (down[i / 2][i % 2] ? 0 : 1u << 8) | (nan[i / 2][i % 2] ? 1u << 16 : 0)) << i;
    return b;
  }
};

template <int DT>
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  if constexpr (DT == VIB3_DT_F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b), c, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
}

// Result y (E columns a lane) of a row and head in which something is NaN, as the formula gives it in f32: an infinite value whose
// probability is 0 in the 16-bit type only (f16, below 2^-36 of the largest) made a NaN of what is an infinity. By one wave, from
// memory, kPer tokens at a time and D / 8 lanes a token: the largest score, the smallest one of a token whose value is not finite, and
// what such values hold; if that one's probability is 0 (in f32), once more, by each one's. It ends early where values are NaN.
template <int DT, int D>
__device__ __forceinline__ void count_infinities(const vib3_gqa_decode& a, int r, int h, int64_t head_at, float (&y)[D / 64]) {
  constexpr int C = D / 8, kPer = 64 / C, E = D / 64, kAhead = 2;
  const int lane = lane_id();
  const Seen<1> row = row_seen<1>(a, r);
  const int sinks = min(a.sinks, row.start);
  const int tokens = sinks + row.len - row.start;  // that the row sees
  const auto place = [&](int i) -> int64_t {  // the newest come first: of a sequence that has become NaN they are
    const int j = tokens - 1 - i;
    return j < 0 ? -1 : gqa_token(a.cache, row.seq, j < sinks ? j : row.start + j - sinks);
  };
  const auto chunk = [&](const void* pool, int64_t at) {
    return *(const uint4*)(at < 0 ? (const uint16_t*)zero_token : (const uint16_t*)pool + at + head_at + lane % C * 8);
  };
  const uint32_t flip = sign_flip(a.scale);
  const uint4 q = *(const uint4*)((const uint16_t*)a.q + (int64_t)r * a.q_row_stride + (int64_t)h * a.q_head_stride + lane % C * 8);
  const auto score = [&](uint4 key) {
    float s = dot2<DT>(q.x ^ flip, key.x, dot2<DT>(q.y ^ flip, key.y, dot2<DT>(q.z ^ flip, key.z, dot2<DT>(q.w ^ flip, key.w, 0.0f))));
    auto more = [&](int moved) { s += __int_as_float(moved); };  // over the token's lanes
    more(__builtin_amdgcn_update_dpp(0, __float_as_int(s), 0xb1, 0xf, 0xf, false));
    more(__builtin_amdgcn_update_dpp(0, __float_as_int(s), 0x4e, 0xf, 0xf, false));
    more(__builtin_amdgcn_update_dpp(0, __float_as_int(s), 0x141, 0xf, 0xf, false));
    if (C > 8) more(__builtin_amdgcn_update_dpp(0, __float_as_int(s), 0x140, 0xf, 0xf, false));
    if (C > 16) s += __shfl_xor(s, 16);
    return s;
  };
  // f(whether there is a token, its score, this lane's chunk of its value), until `done` after a group of them
  const auto walk = [&](auto f, auto done) {
    int64_t next[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; k++) next[k] = place(k * kPer + lane / C);
#pragma unroll 1
    for (int i0 = 0; i0 < tokens; i0 += kAhead * kPer) {
      bool there[kAhead];
      uint4 key[kAhead], v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; k++) there[k] = next[k] >= 0, key[k] = chunk(a.cache.keys, next[k]), v[k] = chunk(a.cache.values, next[k]);
#pragma unroll
      for (int k = 0; k < kAhead; k++) next[k] = place(i0 + (kAhead + k) * kPer + lane / C);
#pragma unroll
      for (int k = 0; k < kAhead; k++) f(there[k], score(key[k]), v[k]);
      if (done()) return;
    }
  };
  // what the values hold in this lane's E columns (as Odd::bits)
  Odd<DT> odd;
  odd.clear();
  const auto mine = [&] {
    uint32_t all = odd.bits();
#pragma unroll
    for (int d = C; d < 64; d *= 2) all |= (uint32_t)__shfl_xor((int)all, d);
    return (uint32_t)__shfl((int)all, lane * E / 8) >> (lane * E % 8);
  };
  float top = -__builtin_huge_valf(), low = __builtin_huge_valf();
  bool none = false;  // whether a score is no number
  bool settled = false;
  walk(
      [&](bool there, float s, uint4 v) {
        top = there ? fmaxf(top, s) : top;
        none |= there & (s != s);
        low = all_finite<DT>(v) ? low : fminf(low, s);
        odd.add(v, false);
      },
      [&] {
        if (__any(none)) return true;
        bool open = false;  // a value that is NaN is so with any probability
#pragma unroll
        for (int i = 0; i < 4; i++) open |= __builtin_bit_cast(uint32_t, odd.nan[i]) != 0;
        if (!__any(open) || !__any(top > -__builtin_huge_valf())) return false;
        const uint32_t has = mine();
        open = false;
#pragma unroll
        for (int e = 0; e < E; e++) open |= y[e] != y[e] && !(has >> (16 + e) & 1);
        return settled = !__any(open);
      });
  if (settled) return;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d)), low = fminf(low, __shfl_xor(low, d));
  if (__any(none) || top == -__builtin_huge_valf() || top == __builtin_huge_valf()) {
    // (scores that are all -infinity give nothing a probability)
    const float all = !__any(none) && top < 0.0f ? 0.0f : __builtin_nanf("");
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = all;
    return;
  }
  const float scale = exponent_scale(a.scale);
  if (__builtin_amdgcn_exp2f((low - top) * scale) == 0.0f) {
    odd.clear();
    walk([&](bool, float s, uint4 v) { odd.add(v, __builtin_amdgcn_exp2f((s - top) * scale) == 0.0f); }, [] { return false; });
  }
  const uint32_t has = mine();
#pragma unroll
  for (int e = 0; e < E; e++) {
    const bool up = has >> e & 1, down = has >> (8 + e) & 1, nan = (has >> (16 + e) & 1) || (up && down);
    const float x = nan ? __builtin_nanf("") : up ? __builtin_huge_valf() : -__builtin_huge_valf();
    y[e] = y[e] != y[e] && (nan | up | down) ? x : y[e];
  }
}

// `team` waves (1, 2, 4, 8 or 16) of a workgroup of WAVES join the parts of one (row, head); rows that see nothing become zero. Rows of
// one share, which wrote them, are looked at too: what is NaN is formed again.
template <int DT, int D, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void k_gqa_join(DecodeArgs d, int team) {
  constexpr int E = D / 64;  // columns of a lane
  constexpr int kAhead = 4;  // parts in flight
  __shared__ float sums[WAVES][D];
  __shared__ float tops[WAVES], totals[WAVES];
  const vib3_gqa_decode& a = d.a;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int x = (int)wide_block() * (WAVES / team) + wave / team;
  const int mate = wave % team;
  const int r = x / a.heads, h = x - r * a.heads;
  int parts = 1;
  float m = -__builtin_huge_valf(), l = 0.0f, o[E] = {};
  if (r < a.rows) {
    const int64_t per = *d.w.head, lo = d.w.begin[r], hi = d.w.begin[r + 1];
    const int w0 = (int)quotient(lo + kRowCost, per);
    parts = hi > lo ? (int)quotient(hi - 1, per) - w0 + 1 : 0;
    if (parts > 1) {
      const int kv_head = h / d.h.group, in_group = h - kv_head * d.h.group;
      const int hu = kv_head * d.h.parts + in_group / 16, col = in_group % 16;
      // part j: that of run w0 + j, in the second slot for the first one where that run began with another row
      const bool late = w0 * per < lo;
      auto slot = [&](int j) {
        return ((size_t)(w0 + j) * d.h.units + hu + (j == 0 && late ? (size_t)d.runs * d.h.units : 0)) * d.h.cols + col;
      };
      const float scale = exponent_scale(a.scale);
      for (int j0 = mate; j0 < parts; j0 += kAhead * team) {
        float2 st[kAhead];
        float v[kAhead][E];
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
          const size_t s = slot(min(j0 + k * team, parts - 1));
          st[k] = d.w.stat[s];
          const float* p = d.w.part + s * D + lane * E;
#pragma unroll
          for (int e = 0; e < E; e++) v[k][e] = p[e];
          if (j0 + k * team >= parts) {
            st[k] = make_float2(-__builtin_huge_valf(), 0.0f);
#pragma unroll
            for (int e = 0; e < E; e++) v[k][e] = 0.0f;
          }
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kAhead; k++) top = fmaxf(top, st[k].x);
        const float ref = top == -__builtin_huge_valf() ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f((m - ref) * scale);
        m = top;
        l *= f;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= f;
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
          const float w = __builtin_amdgcn_exp2f((st[k].x - ref) * scale);
          l += w * st[k].y;
#pragma unroll
          for (int e = 0; e < E; e++) o[e] += w * v[k][e];
        }
      }
    }
  }
  if (team > 1) {
#pragma unroll
    for (int e = 0; e < E; e++) sums[wave][lane * E + e] = o[e];
    if (lane == 0) tops[wave] = m, totals[wave] = l;
    __syncthreads();
    if (mate == 0 && parts > 1) {
      const float scale = exponent_scale(a.scale);
      float top = m;
      for (int w = 1; w < team; w++) top = fmaxf(top, tops[wave + w]);
      const float ref = top == -__builtin_huge_valf() ? 0.0f : top;
      l = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e++) o[e] = 0.0f;
      for (int w = 0; w < team; w++) {
        const float f = __builtin_amdgcn_exp2f((tops[wave + w] - ref) * scale);
        l += f * totals[wave + w];
#pragma unroll
        for (int e = 0; e < E; e++) o[e] += f * sums[wave + w][lane * E + e];
      }
    }
  }
  if (r >= a.rows || mate) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + (int64_t)r * a.out_row_stride + (int64_t)h * a.out_head_stride + lane * E;
  float y[E];
  bool nan = false;
#pragma unroll
  for (int e = 0; e < E; e++) {
    y[e] = parts == 1 ? to_f32<DT>(out[e]) : o[e] * inv;
    nan |= y[e] != y[e];
  }
  const bool again = __any(nan) && l == l;  // (a sum of probabilities that is NaN makes all of the row NaN)
  if (__builtin_expect(again, false)) count_infinities<DT, D>(a, r, h, h / d.h.group * a.cache.head_stride, y);
  if (parts == 1 && !again) return;
#pragma unroll
  for (int e = 0; e < E; e++) out[e] = from_f32<DT>(y[e]);
}

template <int DT, int D>
int launch_decode(const DecodeArgs& d, hipStream_t st) {
  const int workers = d.runs * d.h.units;
  const int blocks = (workers + attend_waves(D) - 1) / attend_waves(D) + 1;  // and the planner
  hipLaunchKernelGGL((k_gqa_attend<DT, D>), dim3((unsigned)blocks), dim3(attend_waves(D) * 64), 0, st, d);
  const int64_t items = (int64_t)d.a.rows * d.a.heads;
  int team = 16;
  while (team > 1 && items * team > 8192) team /= 2;  // 16 waves a CU twice over
  if (team > 4) hipLaunchKernelGGL((k_gqa_join<DT, D, 16>), wide_grid((items * team + 15) / 16), dim3(1024), 0, st, d, team);
  else hipLaunchKernelGGL((k_gqa_join<DT, D, 4>), wide_grid((items * team + 3) / 4), dim3(256), 0, st, d, team);
  VIB3_RETURN_LAUNCH();
}

template <int DT>
int launch_decode_dt(const DecodeArgs& d, hipStream_t st) {
  const int dim = d.a.cache.dim;
  return dim == 64 ? launch_decode<DT, 64>(d, st) : dim == 128 ? launch_decode<DT, 128>(d, st) : launch_decode<DT, 256>(d, st);
}

}  // namespace
}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_gqa_decode_workspace_bytes(const vib3_gqa_decode* args) {
  if (!args || check_gqa_cache(args->cache) || args->rows < 0 || args->rows > kGqaMaxRows ||
      !gqa_heads(args->heads, args->cache.kv_heads))
    return 0;
  return decode_ws(*args, nullptr, nullptr);
}

extern "C" int vib3_launch_gqa_decode(const vib3_gqa_decode* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_gqa_decode& a = *args;
  if (const int rc = check_gqa_cache(a.cache)) return rc;
  if (!__builtin_isfinite(a.scale)) return VIB3_ERR_UNSUPPORTED;
  if (a.rows < 0 || a.rows > kGqaMaxRows || !gqa_heads(a.heads, a.cache.kv_heads) || a.window < 0 || a.sinks < 0)
    return VIB3_ERR_BAD_COUNT;
  if (a.rows == 0) return 0;
  if (!a.lens || !mla_aligned(a.q) || !mla_aligned(a.out) || !mla_stride(a.q_row_stride) || !mla_stride(a.q_head_stride) ||
      !mla_stride(a.out_row_stride) || !mla_stride(a.out_head_stride) || !a.workspace || ((uintptr_t)a.workspace & 255))
    return VIB3_ERR_BAD_POINTER;
  DecodeArgs d;
  d.a = a;
  if (a.workspace_bytes < decode_ws(a, &d.w, a.workspace)) return VIB3_ERR_WORKSPACE;
  d.h = split_heads(a.heads, a.cache.kv_heads);
  d.runs = run_count(d.h, a.cache.dim);
  return a.cache.dtype == VIB3_DT_F16 ? launch_decode_dt<VIB3_DT_F16>(d, (hipStream_t)stream)
                                      : launch_decode_dt<VIB3_DT_BF16>(d, (hipStream_t)stream);
}
