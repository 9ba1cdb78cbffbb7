// How the attention over paged caches deals out its work, and what its kernels have in common whatever the pages hold: entries, shares and items
// (paged_attn.hip says what these are), a lane's column, the sums of a column, results and their joining.
#pragma once

#include <algorithm>

#include "mfma_common.hpp"
#include "paged_common.hpp"

namespace segpt {
namespace {

// Division by a number the host knows, for 0 <= n < 2^31: a product's upper half (the quotient's own sequence takes 25 dependent instructions,
// and an item's place in the work takes seven of them)
struct Divisor {
  int32_t d;
  uint32_t mul, shift;
  __host__ void set(int32_t by) {
    int bits = 1;
    while ((int64_t{1} << bits) < by) ++bits;
    d = by;
    mul = (uint32_t)((uint64_t{1} << (31 + bits)) / (uint32_t)by + 1);
    shift = (uint32_t)bits - 1;
  }
  __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift); }
};
// the same by a number of the device's own, that all lanes have
struct DeviceDivisor {
  int32_t d;
  double inverse;
  __device__ __forceinline__ explicit DeviceDivisor(int by) : d(by) {
    const double x = by, r = __builtin_amdgcn_rcp(x), r1 = fma(fma(-x, r, 1.0), r, r);
    inverse = fma(fma(-x, r1, 1.0), r1, r1);
  }
  __device__ __forceinline__ int of(int n) const { return (int)((n + 0.5) * inverse); }  // exact: the half keeps the quotient off the whole numbers
};

struct PagedArgs {
  segpt_paged_params p;
  Divisor rep, hkv, each;         // H / Hkv, Hkv, rows_each
  int32_t entries, shared;        // shared: 1 if entry 0 is the prefix
  int32_t rows_each, log_page, capacity;
  int32_t target;                 // workgroups of four waves there are to be
  int32_t min_few, min_many;      // shortest shares, in blocks of 32 keys
  int32_t n_many, n_few;          // items there may be of either kind
  int32_t n_joins;                // tiles and kv heads whose partial results there may be to join; kJoinColumns: groups of columns of a kv head
  int32_t joined;                 // kJoinColumns: columns of a group, a power of two up to kMany
  int32_t n_slots;                // partial results there is room for, 32 columns each
  size_t planned_bytes;           // of upto
  int32_t* lens;                  // blocks of a share (few, many) and tiles and kv heads to join, left for the merge
  int32_t* upto;                  // more than kKept * 64 entries: their running sums, [4][entries] in the order of Counts; else NULL
  float* part;                    // [n_slots][32][D]
  float2* stat;                   // [n_slots][32]
};

constexpr int kBlock = 32;          // keys of a score tile
#ifndef SEGPT_FEW_COLUMNS
#define SEGPT_FEW_COLUMNS 32
#endif
constexpr int kFew = SEGPT_FEW_COLUMNS, kMany = 128;  // columns of a tile; kFew: up to 32, set where another number suits the kernels
constexpr int kMostFew = 32;                          // an entry of more columns has tiles of kMany
// What a workgroup of the merge has: by tiles, some of the columns there may be of a tile, whether there are so many or not; by columns, `a.joined` of
// those that there are.  The latter for new callers: the order of a column's sums follows from the number of its units, and what was there keeps its own.
#ifdef SEGPT_JOIN_COLUMNS
constexpr bool kJoinColumns = true;
#else
constexpr bool kJoinColumns = false;
#endif
constexpr float kLazy = 8.f;        // the reference is raised where a score exceeds it by 2^8: probabilities stay below 2^8

// ---- the plan, computed by every wave for itself or, for many entries, by paged_plan_kernel
struct Entry {
  int first, n, len;   // rows, keys
  int tiles, blocks;
  bool many;
  bool broken;         // a length no sequence can have: every row of the entry is NaN
};
// what an entry's numbers are made of: loads alone, so that several entries' are on their way together
struct Raw {
  int r0, r1, len;
};
__device__ __forceinline__ Raw raw_at(const PagedArgs& a, int e) {
  const segpt_paged_params& p = a.p;
  const int b = min(max(e - a.shared, 0), p.B - 1);
  if (p.seq_start) return {p.seq_start[b], p.seq_start[b + 1], p.kv_len[b]};
  return {b * a.rows_each, (b + 1) * a.rows_each, p.kv_len[b]};
}
__device__ __forceinline__ Entry entry_of(const PagedArgs& a, int e, int rep, const Raw& raw) {
  const segpt_paged_params& p = a.p;
  int r0 = min(max(raw.r0, 0), p.T), r1 = min(max(raw.r1, 0), p.T), len = min(max(raw.len, 0), a.capacity);
  bool broken = raw.len < 0 || raw.len > a.capacity;
  if (a.shared && e == 0) {  // the prefix, with the rows of the whole batch
    r0 = p.seq_start ? min(max(p.seq_start[0], 0), p.T) : 0;
    r1 = p.seq_start ? min(max(p.seq_start[p.B], 0), p.T) : p.T;
    len = p.prefix_len;
    broken = false;
  }
  Entry x;
  x.first = r0;
  x.n = e < a.entries ? max(r1 - r0, 0) : 0;
  x.len = len;
  const int cols = x.n * rep;
  x.many = cols > kMostFew;
  x.tiles = x.many ? (cols + kMany - 1) / kMany : (cols + kFew - 1) / kFew;
  x.blocks = (x.len + kBlock - 1) / kBlock;
  x.broken = broken;
  return x;
}
__device__ __forceinline__ Entry entry_at(const PagedArgs& a, int e, int rep) { return entry_of(a, e, rep, raw_at(a, e)); }
// inclusive running sum over the lanes of a wave
template <typename T>
__device__ __forceinline__ T lane_prefix_sum(T v) {
  auto step = [](T x, auto ctrl, auto rows) {
    const int t = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    return x + __builtin_bit_cast(T, t);
  };
  v = step(v, IC<0x111>{}, IC<0xf>{});
  v = step(v, IC<0x112>{}, IC<0xf>{});
  v = step(v, IC<0x114>{}, IC<0xf>{});
  v = step(v, IC<0x118>{}, IC<0xf>{});
  v = step(v, IC<0x142>{}, IC<0xa>{});
  return step(v, IC<0x143>{}, IC<0xc>{});
}
template <typename T>
__device__ __forceinline__ T lane_value(T v, int lane) {
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
struct Shares {
  int few, many;  // blocks of a share
  double per_few, per_many;  // 1 / that
};
// Shares of an entry, its blocks over the share's, rounded up; one also of no keys: it writes what such rows get.  A division by a number
// that all lanes have: in fp64 it is exact (blocks < 2^26; the half keeps the quotient off the whole numbers) and a tenth of the instructions.
__device__ __forceinline__ int shares_of(const Entry& x, Shares s) {
  const int few = max((int)(((double)x.blocks + (s.few - 0.5)) * s.per_few), 1), many = max((int)(((double)x.blocks + (s.many - 0.5)) * s.per_many), 1);
  return x.many ? many : few;
}
// The entries a wave (the plan's kernel: its workgroup) keeps in registers, one a lane and turn, all of them loaded at once (one after the other,
// 129 entries cost a launch of 47 us 8).
constexpr int kKept = 4;
struct Entries {
  Entry e[kKept];
};
template <int LANES>
__device__ __forceinline__ Entries load_entries(const PagedArgs& a, int lane, int rep) {
  Raw raw[kKept] = {};
#pragma unroll
  for (int u = 0; u < kKept; ++u)
    if (LANES * u < a.entries) raw[u] = raw_at(a, LANES * u + lane);
  Entries x = {};
#pragma unroll
  for (int u = 0; u < kKept; ++u)
    if (LANES * u < a.entries) x.e[u] = entry_of(a, LANES * u + lane, rep, raw[u]);
  return x;
}
__device__ __forceinline__ Entries kept_entries(const PagedArgs& a, int lane, int rep) {
  if (a.upto) return {};
  return load_entries<64>(a, lane, rep);
}
__device__ __forceinline__ Shares shares_from(int few, int many) { return {few, many, DeviceDivisor(few).inverse, DeviceDivisor(many).inverse}; }
// Blocks of a share, such that the workgroups are resident at once if the tiles alone are not too many for that: the mean first, then longer
// ones until the begun ones fit too (one workgroup too many is a round of its own).  A block of many columns keeps a workgroup as long as the
// memory does that of few columns, in a quarter of the workgroup each: a wave's share is a quarter as long.  sum(of): of() over all entries
// and kv heads, in floats: it may round, but to the same value in every wave.
template <typename F>
__device__ __forceinline__ Shares share_blocks(const PagedArgs& a, F sum) {
  auto room = [](const Entry& x) { return (float)x.tiles * (x.many ? 1.f : 0.25f); };  // workgroups of a share of each tile
  const float target = (float)a.target, per = __builtin_amdgcn_rcpf(target);
  float len = sum([](const Entry& x) { return (float)x.tiles * (float)x.blocks; }) * per;
  const bool fits = sum(room) < target;
  for (int i = 0;; ++i) {
    const Shares s = shares_from(max((int)fminf(ceilf(0.25f * len), 1e9f), a.min_few), max((int)fminf(ceilf(len), 1e9f), a.min_many));
    if (!fits || i == 2) return s;
    const float groups = sum([&](const Entry& x) { return room(x) * (float)shares_of(x, s); });
    if (groups <= target) return s;
    len *= fmaxf(groups * per, 1.03f);
  }
}
__device__ __forceinline__ Shares share_blocks(const PagedArgs& a, const Entries& kept) {
  if (a.upto) return shares_from(a.lens[0], a.lens[1]);
  return share_blocks(a, [&](auto of) {
    float v = 0.f;
#pragma unroll
    for (int u = 0; u < kKept; ++u)
      if (64 * u < a.entries) v += of(kept.e[u]);
    return lane_value(lane_prefix_sum(v), 63) * (float)a.p.Hkv;
  });
}
// What an entry adds to the running sums: items of either kind, tiles and kv heads whose partial results are to be joined, partial results
enum Find { kFindFew, kFindMany, kFindJoin, kSlots, kFindFirst };
struct Counts {
  int of[4];  // by Find
  int shares;
};
__device__ __forceinline__ Counts counts_of(const PagedArgs& a, int e, const Entry& x, const Shares& share) {
  const int shares = shares_of(x, share), items = x.tiles * shares * a.p.Hkv;
  const bool partial = a.shared || shares > 1;
  const int joined = x.many ? a.joined : min(a.joined, kFew), joins = kJoinColumns ? (x.n * a.rep.d + joined - 1) >> __builtin_ctz(joined) : x.tiles;
  return {{x.many ? 0 : items, x.many ? items : 0, partial && e >= a.shared ? joins * a.p.Hkv : 0, partial ? items * (x.many ? kMany / 32 : 1) : 0}, shares};
}
// an entry as the whole wave sees it
struct Found {
  int entry;          // -1: none
  int first, n, len, blocks;
  int shares, base;   // shares of its keys; number of its first item of its kind (or tile to be joined); none: how many there are
  int slot;           // of its first partial result (entries whose tiles leave any)
  bool many, broken;
};
// The entry of an item of its kind, or of a tile and kv head whose partial results are to be joined, by number; or the first entry.  With the sums of
// paged_plan_kernel: 64 of them are looked at a time (three loads one after the other for 2^18 entries).
template <Find F>
__device__ __forceinline__ Found search_entry(const PagedArgs& a, int lane, int rep, const Shares& share, int which) {
  Found found{-1, 0, 0, 0, 0, 0, 0, 0, false, false};
  const int32_t* upto = a.upto + (int64_t)(F == kFindFirst ? kSlots : F) * a.entries;
  int e = 0;
  if (F != kFindFirst) {
    const int all = upto[a.entries - 1];
    if (which >= all) {
      found.base = all;
      return found;
    }
    for (int n = a.entries, step = n; step > 1;) {  // the first of e .. e + n - 1 whose sum is above `which`
      step = (n + 63) >> 6;
      const uint64_t above = __builtin_amdgcn_ballot_w64(upto[e + min((lane + 1) * step, n) - 1] > which);
      if (!above) return found;  // row ranges that overlap, their sum beyond 32 bits
      const int l = __builtin_ctzll(above);
      e += l * step;
      n = min(step, n - l * step);
    }
  }
  const Entry x = entry_at(a, e, rep);
  const Counts c = counts_of(a, e, x, share);
  const int base = F == kFindFirst || e == 0 ? 0 : upto[e - 1];
  if (F != kFindFirst && (uint32_t)(which - base) >= (uint32_t)c.of[F]) return found;
  return {e, x.first, x.n, x.len, x.blocks, c.shares, base, e == 0 ? 0 : a.upto[(int64_t)kSlots * a.entries + e - 1], x.many, x.broken};
}
template <Find F>
__device__ __forceinline__ Found find_entry(const PagedArgs& a, int lane, int rep, const Shares& share, const Entries& kept, int which) {
  if (a.upto) return search_entry<F>(a, lane, rep, share, which);
  int base = 0, slot = 0;
  Found found{-1, 0, 0, 0, 0, 0, 0, 0, false, false};
  auto look = [&](int e0, const Entry& x) {  // true: it is among these 64
    const Counts c = counts_of(a, e0 + lane, x, share);
    const int slots = c.of[kSlots], slots_upto = slot + lane_prefix_sum(slots);
    const int mine_n = F == kFindFirst ? 0 : c.of[F == kFindFirst ? 0 : F];
    const int upto = F == kFindFirst ? 0 : base + lane_prefix_sum(mine_n);
    const uint64_t hits = F == kFindFirst ? 1 : __builtin_amdgcn_ballot_w64(which >= upto - mine_n && which < upto);
    if (hits) {
      const int l = __builtin_ctzll(hits);
      found = Found{e0 + l, lane_value(x.first, l), lane_value(x.n, l), lane_value(x.len, l), lane_value(x.blocks, l), lane_value(c.shares, l),
                    lane_value(upto - mine_n, l), lane_value(slots_upto - slots, l), lane_value((int)x.many, l) != 0, lane_value((int)x.broken, l) != 0};
      return true;
    }
    base = lane_value(upto, 63);
    slot = lane_value(slots_upto, 63);
    return false;
  };
#pragma unroll
  for (int u = 0; u < kKept; ++u)
    if (64 * u < a.entries && look(64 * u, kept.e[u])) return found;
  found.base = base;
  return found;
}
// The plan of more than kKept * 64 entries, by one workgroup: lengths of the shares and running sums.  Formed by every wave for itself, an entry's
// numbers are read by all of them, several times over, and the time grows with the square of the entries.  Single tokens, 18 / 6 heads of 64, us, by
// every wave and here: 300 sequences 132, 134; 1000 200, 197; 4000 586, 244.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedArgs a) {
  constexpr int kWaves = kPlanThreads / 64;
  __shared__ float sums[kWaves];
  __shared__ int counts[4][kWaves];
  const int tid = threadIdx.x, wave = tid >> 6, rep = a.rep.d;
  const Entries kept = load_entries<kPlanThreads>(a, tid, rep);
  const Shares share = share_blocks(a, [&](auto of) {
    float v = 0.f;
#pragma unroll
    for (int u = 0; u < kKept; ++u)
      if (kPlanThreads * u < a.entries) v += of(kept.e[u]);
    for (int e = kPlanThreads * kKept; e < a.entries; e += kPlanThreads) v += of(entry_at(a, e + tid, rep));
    v = lane_prefix_sum(v);
    __syncthreads();  // the sums before have been read
    if ((tid & 63) == 63) sums[wave] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += sums[w];
    return v * (float)a.p.Hkv;
  });
  int before[4] = {0, 0, 0, 0};
  auto add = [&](int e, const Entry& x) {
    const Counts c = counts_of(a, e, x, share);
    int own[4];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      own[k] = lane_prefix_sum(c.of[k]);
      if ((tid & 63) == 63) counts[k][wave] = own[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      int upto = before[k] + own[k];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int n = counts[k][w];
        before[k] += n;
        upto += w < wave ? n : 0;
      }
      if (e < a.entries) a.upto[(int64_t)k * a.entries + e] = upto;
    }
  };
#pragma unroll
  for (int u = 0; u < kKept; ++u)
    if (kPlanThreads * u < a.entries) add(kPlanThreads * u + tid, kept.e[u]);
  for (int e = kPlanThreads * kKept; e < a.entries; e += kPlanThreads) add(e + tid, entry_at(a, e + tid, rep));
  if (tid == 0) { a.lens[0] = share.few; a.lens[1] = share.many; a.lens[2] = before[kFindJoin]; }
}

// A pair of values in two bf16 parts each.  The first is cut off, a little below the value in size and never the value itself, so that the second has
// the same sign and is not zero: the products of both with an infinity are that infinity, not NaN.  The second is at most 2^-7 + 2^-9 of the
// value and exact in fp32; what its rounding leaves out is less than 2^-14 of the value.
__device__ __forceinline__ void two_parts(float a, float b, uint32_t& first, uint32_t& second) {
  constexpr float kBelow = 1.f - 0x1p-9f;
  const uint32_t x = __float_as_uint(a * kBelow) & 0xffff0000u, y = __float_as_uint(b * kBelow) & 0xffff0000u;
  first = x >> 16 | y;
  second = pack_bf16x2(a - __uint_as_float(x), b - __uint_as_float(y));
}

template <typename E, int D>
__device__ __forceinline__ float gate_factor(const segpt_paged_params& p, E z) {
  float x;
  if constexpr (sizeof(E) == 2) x = bf16_to_f32(z); else x = z;
  return p.gate_scale / (1.0f + __expf(-x));
}
template <typename E, int D>
__device__ __forceinline__ float gate_factor(const segpt_paged_params& p, int t, int h) { return gate_factor<E, D>(p, row_of<E>(p.gate, t, h)[0]); }

// ---- an item
struct Item {
  Found x;
  int g, part, tile, cols;
  int k0, nk;        // its keys: k0 .. k0 + nk - 1
  int past;          // row i of a sequence sees its keys up to past + i; the prefix's all rows see, but for those that stand in it
  int slot;
  bool prefix, direct, valid;
  const int* ids;    // page numbers
};
template <bool MANY>
__device__ __forceinline__ Item locate(const PagedArgs& a, int lane, int rep, const Shares& share, const Entries& mine, int number) {
  constexpr int COLS = MANY ? kMany : kFew, SLOTS = MANY ? kMany / 32 : 1;
  Item it;
  it.x = find_entry<MANY ? kFindMany : kFindFew>(a, lane, rep, share, mine, number);
  const Found& x = it.x;
  it.valid = x.entry >= 0;
  if (!it.valid) return it;
  it.cols = x.n * rep;
  const int n_tiles = (it.cols + COLS - 1) / COLS, local = number - x.base;
  const DeviceDivisor shares(x.shares);
  const int per_head = a.hkv.of(local), from_last = shares.of(per_head);
  it.g = local - per_head * a.p.Hkv;
  it.part = per_head - from_last * x.shares;
  it.tile = n_tiles - 1 - from_last;  // the last tiles see the most keys: they start first
  it.prefix = a.shared && x.entry == 0;
  it.direct = !a.shared && x.shares == 1;
  it.slot = x.slot + ((it.tile * x.shares + it.part) * a.p.Hkv + it.g) * SLOTS;
  // row ranges that overlap may add up to more than 32 bits hold: nothing is written outside the scratch
  it.valid = it.tile >= 0 && (it.direct || (it.slot >= 0 && it.slot <= a.n_slots - SLOTS));
  it.past = x.len - x.n;
  const int per = shares.of(x.blocks + x.shares - 1) * kBlock;  // shares as even as whole blocks allow
  const int last_col = min(it.cols, (it.tile + 1) * COLS) - 1, sees = it.prefix ? x.len : min(x.len, it.past + a.rep.of(last_col) + 1);
  it.k0 = it.part * per;
  it.nk = max(min(sees, it.k0 + per) - it.k0, 0);
  it.ids = it.prefix ? a.p.prefix_table : a.p.block_table + (int64_t)(x.entry - a.shared) * a.p.table_stride;
  return it;
}
// what scales component d of every query: asked for, and worked out
struct Gain {
  float q, k;
};
__device__ __forceinline__ Gain fetch_gain(const segpt_paged_params& p, int d) {
  const float* gk = p.g_k ? p.g_k : p.g_q;
  return {p.g_q[p.gq_numel == 1 ? 0 : d], gk[p.gk_numel > 1 ? d : 0]};
}
__device__ __forceinline__ float scale_of(const segpt_paged_params& p, const Gain& g) { return g.q * (p.g_k ? g.k : 1.f) * p.sm_scale * kLog2e; }

// ---- a lane's column, and what it sees of the item's keys (counted from k0 on)
struct Column {
  int t, h;      // row and head
  bool live;
  int lim;       // last key of the lane's row
  int all, any;  // last key that all columns of the wave see, that any of them sees
};
// q: where the query's row goes; Q::kCols = 2^Q::kLogCols columns stand side by side in a wave
template <typename E, int D, typename Q>
__device__ __forceinline__ Column column_of(const PagedArgs& a, const Item& it, int rep, int wave_col, int lane, Q& q) {
  const segpt_paged_params& p = a.p;
  Column c;
  const bool works = wave_col < it.cols;
  const int col = wave_col + (lane & (Q::kCols - 1)), safe = min(col, it.cols - 1), i = a.rep.of(safe);
  c.live = col < it.cols;
  c.t = it.x.first + i;
  c.h = it.g * rep + safe - i * rep;
  int own = it.past + i;  // position among the sequence's own keys: negative where it stands in the prefix
  if (it.prefix) {        // the row's own sequence says where it stands
    int b = 0, f = 0, n = 0;
    if (p.seq_start) {
      for (int lo = 0, hi = p.B - 1; lo <= hi;) {  // last sequence that starts at or before the row
        const int m = (lo + hi) >> 1;
        if (p.seq_start[m] <= c.t) { b = m; lo = m + 1; } else hi = m - 1;
      }
    } else {
      b = a.each.of(c.t);
    }
    sequence_rows(p, a.rows_each, b, &f, &n);
    own = (int)max(min((int64_t)p.kv_len[b] - n + (c.t - f), (int64_t)a.capacity - 1), -1 - (int64_t)p.prefix_len);  // whatever the length says
  }
  const int64_t pos = max((int64_t)p.prefix_len + own, (int64_t)0);
  q.fetch(p, row_of<E>(p.q, c.t, c.h), (p.rope_pos0 + pos) * (D / 2), lane >> Q::kLogCols);
  c.lim = min((it.prefix ? p.prefix_len : 0) + own - it.k0, it.nk - 1);
  if (it.prefix) {
    const bool cut = __builtin_amdgcn_ballot_w64(c.live && c.lim < it.nk - 1) != 0;  // rows that stand in the prefix
    c.all = !works || cut ? -1 : it.nk - 1;
    c.any = works ? it.nk - 1 : -1;
  } else {
    c.all = works ? min(it.past + a.rep.of(wave_col) - it.k0, it.nk - 1) : -1;
    c.any = works ? min(it.past + a.rep.of(min(wave_col + Q::kCols - 1, it.cols - 1)) - it.k0, it.nk - 1) : -1;
  }
  return c;
}

// Sums of a column.  Scores come out of the product less the reference already: it is the C operand of their first instruction.
template <int MB>
struct State {
  f32x16 o[MB], less;  // less: the reference's negative, in every register
  float m, limit;      // reference (log2 units); a score may exceed it by `limit` before it is raised: -inf as long as no key has been seen
  float l[2];          // of this lane's half of the keys
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) o[mb] = splat16(0.f);
    less = splat16(0.f);
    m = 0.f;
    limit = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  __device__ __forceinline__ float reference() const { return limit == -INFINITY ? -INFINITY : m; }
  // raises the reference where scores of N blocks exceed it
  template <int N>
  __device__ __forceinline__ void raise(f32x16 (&s)[N]) {
    float mx[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      mx[n] = s[n][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx[n] = fmaxf(mx[n], s[n][r]);
    }
#pragma unroll
    for (int n = 1; n < N; ++n) mx[0] = fmaxf(mx[0], mx[n]);
    const float top = half_max(mx[0]);
    if (__builtin_amdgcn_ballot_w64(top > limit) != 0) {
      const float up = top > limit ? top : 0.f, corr = limit == -INFINITY ? 1.f : fast_exp2(-up);  // nothing to scale before the first key
      m += up;
      if (top > limit) limit = kLazy;
      less = splat16(-m);
      l[0] *= corr;
      l[1] *= corr;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[mb][r] *= corr;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[n][r] -= up;
    }
  }
  template <int N>
  static __device__ __forceinline__ void exponentials(f32x16 (&s)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = fast_exp2(s[n][r]);
  }
};
__device__ __forceinline__ void hide_unseen(f32x16& s, int seen, int hh) {  // register r holds key 4 hh + c_r, c_r = 8 (r / 4) + r % 4
  const int t = seen - 4 * hh;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (8 * (r >> 2) + (r & 3) > t) s[r] = -INFINITY;
}

// What an item leaves: y where it is its tile's only one, else a partial result
template <typename E, int D, typename S>
__device__ __forceinline__ void store_result(const PagedArgs& a, const Item& it, const Column& c, S& st, bool bad, int slot_col, int hh) {
  const segpt_paged_params& p = a.p;
  constexpr int MB = D / 32;
  float l = half_sum(st.l[0] + st.l[1]), m = st.reference();
  if (bad) { l = __builtin_nanf(""); m = 0.f; }
  if (!c.live) return;
  if (!it.direct) {
    const int64_t at = (int64_t)it.slot * 32 + slot_col;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(a.part + at * D + 32 * mb + 8 * q + 4 * hh) =
            make_float4(st.o[mb][4 * q], st.o[mb][4 * q + 1], st.o[mb][4 * q + 2], st.o[mb][4 * q + 3]);
    if (hh == 0) a.stat[at] = make_float2(m, l);
    return;
  }
  float f = l == 0.f ? 0.f : 1.0f / l;
  if (p.lse && hh == 0) p.lse[(int64_t)c.t * p.H + c.h] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
  if (p.gate.ptr) f *= gate_factor<E, D>(p, c.t, c.h);
  E* out = row_of<E>(p.o, c.t, c.h);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float y[4] = {st.o[mb][4 * q] * f, st.o[mb][4 * q + 1] * f, st.o[mb][4 * q + 2] * f, st.o[mb][4 * q + 3] * f};
      E* at = out + 32 * mb + 8 * q + 4 * hh;
      if constexpr (sizeof(E) == 2) *reinterpret_cast<u32x2*>(at) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      else store16(at, y);
    }
}

// Rows before the first sequence and behind the last, by the last workgroups of the launch, which mostly have no item
template <typename E>
__device__ __forceinline__ void clear_rest(const PagedArgs& a, int tid, int threads, int D) {
  constexpr int kBy = 64;
  const segpt_paged_params& p = a.p;
  const int by = min(kBy, (int)gridDim.x), from = (int)blockIdx.x - ((int)gridDim.x - by);
  if (!p.seq_start || !(p.flags & SEGPT_FLAG_ZERO_REST) || from < 0) return;
  int head, f, n;
  sequence_rows(p, 0, 0, &head, &n);
  sequence_rows(p, 0, p.B - 1, &f, &n);
  const int tail = max(f + n, head);
  for (int i = from; i < head + p.T - tail; i += by) {
    const int t = i < head ? i : i - head + tail;
    for (int x = tid; x < p.H * D; x += threads) row_of<E>(p.o, t, x / D)[x % D] = 0;
    for (int h = tid; p.lse && h < p.H; h += threads) p.lse[(int64_t)t * p.H + h] = -INFINITY;
  }
}

// What the merge goes by, from the last workgroup, which mostly has no item, where no plan was made before
__device__ __forceinline__ void leave_plan(const PagedArgs& a, int lane, int rep, const Shares& share, const Entries& mine) {
  if (a.upto || blockIdx.x != gridDim.x - 1) return;
  const int joins = find_entry<kFindJoin>(a, lane, rep, share, mine, INT32_MAX).base;
  if (threadIdx.x == 0) { a.lens[0] = share.few; a.lens[1] = share.many; a.lens[2] = joins; }
}

// Joins the partial results of `per_sub` columns of a tile: its sequence's shares and, behind them, the prefix's.  A unit of D / 4 lanes holds a
// row; as many units stand side by side over the shares of a column as leave each one batch of kBatch that is requested together, and
// their sums meet in LDS.  Fixed order: deterministic.  4.9 us for one token of 18 heads (launch and two round trips), 5.9 for 32 of them, 12 for
// 128 tokens of 16 heads of 128 behind a prefix (25 MB).
// By columns (kJoinColumns): 223 rows of 16 heads of 128 behind 5001 keys 16.2 -> 9.5 us, 2891 rows of fp32, 8 / 4 heads of 64, 11.4 -> 7.4; single tokens as before.
constexpr int kMergeThreads = 256, kMergeGroups = 2048;
template <typename E, int D>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_kernel(PagedArgs a, int subs, int per_sub) {
  const segpt_paged_params& p = a.p;
  constexpr int LPR = D / 4, kUnits = kMergeThreads / LPR, kBatch = 4;
  __shared__ float4 sums[kMergeThreads];
  __shared__ float2 stats[kUnits];
  const int tid = threadIdx.x, lane = tid & 63, unit = tid / LPR, c = tid % LPR;
  const int rep = a.rep.d;
  const int few = a.lens[0], many = a.lens[1], joins = a.lens[2];
  const Entries mine = kept_entries(a, lane, rep);
  const int which = kJoinColumns ? blockIdx.x : blockIdx.x / subs, sub = blockIdx.x - which * subs;
  if (which >= joins) return;
  const Shares share = shares_from(few, many);
  const Found own = find_entry<kFindJoin>(a, lane, rep, share, mine, which);
  if (own.entry < 0) return;
  const int number = a.hkv.of(which - own.base), g = which - own.base - number * p.Hkv, cols = own.n * rep, tile_cols = own.many ? kMany : kFew;
  if (kJoinColumns) per_sub = min(per_sub, tile_cols);
  const int tile = kJoinColumns ? number * per_sub / tile_cols : number, from = kJoinColumns ? number * per_sub - tile * tile_cols : sub * per_sub;
  Found pre{-1, 0, 0, 0, 0, 0, 0, 0, false, false};
  if (a.shared) pre = find_entry<kFindFirst>(a, lane, rep, share, mine, 0);
  const int pre_cols = pre.many ? kMany : kFew;
  const int n = own.shares + pre.shares;
  int step = min(per_sub, kUnits);  // columns at a time
  while (step > 1 && kUnits / step * kBatch < n) step >>= 1;
  const int wide = kUnits / step;  // units of a column
  for (int c0 = from; c0 < min(from + per_sub, tile_cols); c0 += step) {  // the same for all threads
    if (tile * tile_cols + c0 >= cols) return;
    const int col = tile * tile_cols + min(c0 + unit % step, tile_cols - 1);
    const bool live = col < cols && c0 + unit % step < min(from + per_sub, tile_cols);
    const int i = a.rep.of(min(col, cols - 1)), t = own.first + i, h = g * rep + (min(col, cols - 1) - i * rep);
    const int pcol = (t - pre.first) * rep + h - g * rep, ptile = pcol / pre_cols;
    auto place = [&](int s) {  // row of share s among all partial results; none: there is no room for it
      const bool is_own = s < own.shares;
      const Found& x = is_own ? own : pre;
      const int slot = x.slot + (((is_own ? tile : ptile) * x.shares + (is_own ? s : s - own.shares)) * p.Hkv + g) * (x.many ? kMany / 32 : 1);
      return slot < a.n_slots - (x.many ? kMany / 32 - 1 : 0) ? (int64_t)slot * 32 + (is_own ? col - tile * tile_cols : pcol - ptile * pre_cols) : (int64_t)-1;
    };
    E gate{};  // on its way while the results are joined
    if (p.gate.ptr) gate = row_of<E>(p.gate, t, h)[0];
    float m = -INFINITY, l = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live)
      for (int s0 = unit / step; s0 < n; s0 += kBatch * wide) {
        float2 x[kBatch];
        float4 o[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int64_t at = place(min(s0 + u * wide, n - 1));
          x[u] = at < 0 ? make_float2(0.f, __builtin_nanf("")) : a.stat[at];
          o[u] = *reinterpret_cast<const float4*>(a.part + max(at, (int64_t)0) * D + 4 * c);
          if (s0 + u * wide >= n) x[u] = make_float2(-INFINITY, 0.f);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) top = fmaxf(top, x[u].x);
        const float ref = top == -INFINITY ? 0.f : top, w0 = fast_exp2(m - ref);
        m = top;
        l *= w0;
        y.x *= w0; y.y *= w0; y.z *= w0; y.w *= w0;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (x[u].y == 0.f) continue;  // saw no key
          const float w = fast_exp2(x[u].x - ref);
          l += w * x[u].y;
          y.x += w * o[u].x; y.y += w * o[u].y; y.z += w * o[u].z; y.w += w * o[u].w;
        }
      }
    auto take_in = [&](float2 x, float4 o) {  // another unit's sums of the column
      const float top = fmaxf(m, x.x), ref = top == -INFINITY ? 0.f : top, w0 = fast_exp2(m - ref), w1 = fast_exp2(x.x - ref);
      m = top;
      l = l * w0 + x.y * w1;
      y.x = y.x * w0 + o.x * w1; y.y = y.y * w0 + o.y * w1; y.z = y.z * w0 + o.z * w1; y.w = y.w * w0 + o.w * w1;
    };
    // the units of a wave first, then the waves
    for (int o = step * LPR; o < 64; o <<= 1)
      take_in(make_float2(__shfl_xor(m, o, 64), __shfl_xor(l, o, 64)), make_float4(__shfl_xor(y.x, o, 64), __shfl_xor(y.y, o, 64), __shfl_xor(y.z, o, 64), __shfl_xor(y.w, o, 64)));
    if (wide > 1) {
      __syncthreads();  // the round before has been read
      sums[tid] = y;
      if (c == 0) stats[unit] = make_float2(m, l);
      __syncthreads();
      if (unit >= step) continue;
      const int far = max(step, 64 / LPR);  // units from one wave's sums to the next one's
#pragma unroll
      for (int w = 1; w < 4; ++w)
        if (unit + w * far < kUnits) take_in(stats[unit + w * far], sums[w * far * LPR + tid]);
    }
    if (!live) continue;
    if (own.broken) l = __builtin_nanf("");
    float f = l == 0.f ? 0.f : 1.0f / l;
    if (p.lse && c == 0) p.lse[(int64_t)t * p.H + h] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
    if (p.gate.ptr) f *= gate_factor<E, D>(p, gate);
    E* out = row_of<E>(p.o, t, h) + 4 * c;
    const float v[4] = {y.x * f, y.y * f, y.z * f, y.w * f};
    if constexpr (sizeof(E) == 2) *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    else store16(out, v);
  }
}

// ---- host side
bool all_few(const segpt_paged_params& p) {  // known on the host
  return !p.prefix_table && !p.seq_start && (int64_t)p.H / p.Hkv * (p.T / p.B) <= kMostFew;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// fills the plan for as many workgroups of four waves as there are to be; returns the scratch bytes
size_t plan(const segpt_paged_params& p, PagedArgs& a, int target) {
  const int rep = p.H / p.Hkv;
  a.rep.set(rep);
  a.hkv.set(p.Hkv);
  a.shared = p.prefix_table ? 1 : 0;
  a.entries = p.B + a.shared;
  a.rows_each = p.seq_start ? 0 : p.T / p.B;
  a.each.set(p.seq_start ? 1 : a.rows_each);
  a.log_page = __builtin_ctz((unsigned)p.page_size);
  a.capacity = paged_capacity(p);
  a.target = target;
  a.min_few = 2;
  a.min_many = 4;
  // Tiles: whole ones of the columns there are, and one begun an entry (of few columns: one, and another where a tile does not hold them).  Items: a
  // tile's part of what the target stands for, and one begun.
  const int64_t cols = (int64_t)p.T * rep;
  int64_t many = cols / kMany + std::min<int64_t>(p.B, cols / (kMostFew + 1)), few = std::min<int64_t>(p.B, p.T);
  static_assert(kFew <= kMostFew && 2 * kFew >= kMostFew);
  if (kFew < kMostFew) few += std::min<int64_t>(few, cols / (kFew + 1));
  if (!p.seq_start) {
    const int64_t each = cols / p.B;
    many = each > kMostFew ? (each + kMany - 1) / kMany * p.B : 0;
    few = each > kMostFew ? 0 : (each + kFew - 1) / kFew * p.B;
  }
  const int64_t own = many + few, own_many = many;
  if (a.shared && cols > kMostFew) many += (cols + kMany - 1) / kMany;
  else if (a.shared) few += (cols + kFew - 1) / kFew;
  const int64_t slack = 64;  // the sum that gives the length of a share is rounded
  const int64_t n_many = many ? many * p.Hkv + a.target + slack : 0, n_few = few ? few * p.Hkv + 4 * a.target + slack : 0;
  a.n_many = (int32_t)std::min<int64_t>(n_many, INT32_MAX);
  a.n_few = (int32_t)std::min<int64_t>(n_few, INT32_MAX);
  // a tile that leaves partial results has two shares or more, i.e. at most twice its part of the target; beside a prefix all leave them
  const int64_t most = (int64_t)a.target + slack;
  const int64_t slots = kMany / 32 * (a.shared ? n_many : std::min(n_many, 2 * most)) + (a.shared ? n_few : std::min(n_few, 8 * most));
  a.n_slots = (int32_t)std::min<int64_t>(slots, INT32_MAX / 32);
  const int64_t tiles = a.shared ? own * p.Hkv : std::min(own_many * p.Hkv, most) + std::min((own - own_many) * p.Hkv, 4 * most);
  int64_t joins = tiles;
  if (kJoinColumns) {
    // groups of so many columns that the card holds their workgroups at once, if there are not even more of them; what is begun counts as one
    const int64_t each = cols / p.B, many_tiles = a.shared ? own_many * p.Hkv : std::min(own_many * p.Hkv, most);
    for (a.joined = 1;; a.joined *= 2) {
      const int64_t j = a.joined, jf = std::min<int64_t>(j, kFew), own_j = each > kMostFew ? j : jf, begun = std::min<int64_t>(p.B, p.T);
      const int64_t all = p.seq_start ? cols / j + begun + (j > jf ? std::min(begun, cols / (kFew + 1)) : 0) : (each + own_j - 1) / own_j * p.B;
      joins = std::min(all * p.Hkv, many_tiles * (kMany / j) + (tiles - many_tiles) * (kFew / jf));
      if (joins <= kMergeGroups || j == kMany) break;
    }
  }
  a.n_joins = (int32_t)std::min<int64_t>(joins, INT32_MAX);
  a.planned_bytes = a.entries > kKept * 64 ? (size_t)4 * a.entries * sizeof(int32_t) : 0;
  // a launch has fewer than 2^32 threads (the merge: a workgroup a join at least)
  const int64_t most_groups = UINT32_MAX / 256;
  return n_many + (n_few + 3) / 4 > most_groups || joins > most_groups || slots > INT32_MAX / 32 ? SIZE_MAX : 256 + up256(a.planned_bytes) + (size_t)a.n_slots * 32 * (p.D + 2) * sizeof(float);
}

// the call's sizes, its plan and where its scratch lies
int prepare_call(const segpt_paged_params* p, PagedArgs& a, int target) {
  a.p = *p;
  const size_t need = plan(*p, a, target);
  if (need > SIZE_MAX - 256) return SEGPT_E_SHAPE;
  if (!p->workspace || p->workspace_bytes < up256(need)) return SEGPT_E_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(p->workspace) & 255u) return SEGPT_E_ALIGN;
  a.lens = reinterpret_cast<int32_t*>(p->workspace);
  if (a.planned_bytes) a.upto = a.lens + 256 / sizeof(int32_t);
  a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(p->workspace) + 256 + up256(a.planned_bytes));
  a.stat = reinterpret_cast<float2*>(a.part + (size_t)a.n_slots * 32 * p->D);
  return SEGPT_OK;
}

int launch_plan(const PagedArgs& a, hipStream_t st) {
  if (!a.upto) return SEGPT_OK;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
  return (int)hipGetLastError();
}

template <typename E, int D>
int launch_merge(const PagedArgs& a, hipStream_t st) {
  const segpt_paged_params& p = a.p;
  if (kJoinColumns) {
    hipLaunchKernelGGL((paged_merge_kernel<E, D>), dim3((unsigned)a.n_joins), dim3(kMergeThreads), 0, st, a, 1, a.joined);
    return (int)hipGetLastError();
  }
  // a column a workgroup, or so many that there are not more workgroups than the card holds a few times over
  const int64_t all = (int64_t)p.T * (p.H / p.Hkv);
  const bool any_many = p.seq_start ? all > kFew : all / p.B > kFew;
  const int most = any_many ? kMany : kFew, cols = p.seq_start ? most : (int)std::min<int64_t>(most, all / p.B);
  int per_sub = 1;
  while (per_sub < kMany && (int64_t)a.n_joins * ((cols + per_sub - 1) / per_sub) > 4096) per_sub *= 2;
  const int subs = (cols + per_sub - 1) / per_sub;
  hipLaunchKernelGGL((paged_merge_kernel<E, D>), dim3((unsigned)(a.n_joins * subs)), dim3(kMergeThreads), 0, st, a, subs, per_sub);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace segpt
