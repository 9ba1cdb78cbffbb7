// Attention over a paged key/value cache, forward only: ragged rows of B sequences, each against the pages its table names, and, if the
// batch shares one, against the pages of a common prefix.
//
//   y_i = sum_j exp(s_ij - lse_i) v'_j      s_ij = qhat_i . k'_j      qhat = sm_scale rot(q) rsqrt(mean q^2 + eps) g_q g_k
//
// over the prefix's keys and the sequence's keys j <= kv_len - n + i.  The pool's rows are already rotated and normalised, so that what is
// left per key is a product on either side of the softmax.
//
// Work.  The heads of a kv group and the rows of a sequence are the columns n = i * (H / Hkv) + head of one product.  An ENTRY is a set of
// columns that read the same pages: a sequence, or the shared prefix with the rows of the whole batch.  Entries of up to 32 columns (generated
// tokens) are FEW: an item of work is one wave with its own buffers, bound by the memory it reads.  The others are MANY: an item is a
// workgroup of four waves with 32 columns each that share the staged keys, bound by the matrix pipe and the exponentials.  Either way an item
// is (entry, tile of columns, share of its keys, kv head).  Lengths live on the device, so the device deals out the work: the length of a
// share follows from the sum over all entries, such that the items fill the card once, and every workgroup finds its own item in the running
// sum of the entries' items (one load and a few register moves for up to 64 sequences).  Up to 256 entries every wave forms the sums for itself;
// more are summed once, by paged_plan_kernel, and searched.  A tile with one share writes y; others leave (reference m, sum l, products O) in
// fp32, which paged_merge_kernel joins.
//
// Scores are transposed as in the other forward kernels: lane = query column, S^T = K' . Qhat^T, and the probabilities are already the
// B operand of O^T = V'^T . P^T.
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
  int32_t n_joins;                // tiles and kv heads whose partial results there may be to join
  int32_t n_slots;                // partial results there is room for, 32 columns each
  size_t planned_bytes;           // of upto
  int32_t* lens;                  // blocks of a share (few, many) and tiles and kv heads to join, left for the merge
  int32_t* upto;                  // more than kKept * 64 entries: their running sums, [4][entries] in the order of Counts; else NULL
  float* part;                    // [n_slots][32][D]
  float2* stat;                   // [n_slots][32]
};

constexpr int kBlock = 32;          // keys of a score tile
constexpr int kFew = 32, kMany = 128;  // columns of a tile
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
  x.many = cols > kFew;
  x.tiles = x.many ? (cols + kMany - 1) / kMany : cols > 0;
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
  return {{x.many ? 0 : items, x.many ? items : 0, partial && e >= a.shared ? x.tiles * a.p.Hkv : 0, partial ? items * (x.many ? kMany / 32 : 1) : 0}, shares};
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

// ---- tiles: BK rows of D elements, filled by direct global->LDS loads of 1 KB; the 16-byte chunk c of row r lies at chunk c ^ f(r)
template <typename E, int D>
struct Tile {
  static constexpr int kRB = D * (int)sizeof(E), kChunks = kRB / 16, kRowsPerLoad = 1024 / kRB;
  static __device__ __forceinline__ int f(int row) {
    if constexpr (sizeof(E) == 2) return Swz<D>::f(row);
    // fp32: the b128 reads of 16 consecutive rows want 16 different chunks, the b32 reads of two rows four apart opposite halves of the banks
    else if constexpr (D == 32) return (row >> 1) & 7;
    else return (row & 3) | ((row >> 1) & 4) | ((row & 4) << 1);
  }
};
template <typename E, int D>
struct Shape {
  static constexpr int kRB = D * (int)sizeof(E);
  // MANY: keys per staged tile (16 KB with its values, at fp32 head_dim 128 32) and stages of the ring
  static constexpr int kBK = kRB <= 128 ? 64 : 32;
  static constexpr int kTileBytes = kBK * kRB, kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = kRB <= 256 ? 4 : 3;
  static constexpr int kManyTable = 256;  // page numbers held in LDS: a longer share takes its keys in windows
  static constexpr int kManyBytes = kStages * kStageBytes;
  // FEW: one block of keys and one of values a wave
  static constexpr int kFewTable = 64;
  static constexpr int kDepth = kRB <= 128 ? 2 : 1;  // buffers
  static constexpr int kFewBytes = 2 * kBlock * kRB;  // of a buffer
  static constexpr int kOcc = kRB > 256 ? 1 : 2;  // workgroups of four waves per CU
};

// A pair of values in two bf16 parts each.  The first is cut off, a little below the value in size and never the value itself, so that the second has
// the same sign and is not zero: the products of both with an infinity are that infinity, not NaN.  The second is at most 2^-7 + 2^-9 of the
// value and exact in fp32; what its rounding leaves out is less than 2^-14 of the value.
__device__ __forceinline__ void two_parts(float a, float b, uint32_t& first, uint32_t& second) {
  constexpr float kBelow = 1.f - 0x1p-9f;
  const uint32_t x = __float_as_uint(a * kBelow) & 0xffff0000u, y = __float_as_uint(b * kBelow) & 0xffff0000u;
  first = x >> 16 | y;
  second = pack_bf16x2(a - __uint_as_float(x), b - __uint_as_float(y));
}

// Query columns in the B operand's layout, scaled by everything that does not depend on the key (gsm: g_q g_k sm_scale log2 e); D / 2 values
// a lane.  bf16: element 16 ks + 8 hh + t; fp32: chunk 2 c + hh of four.  fetch() asks for the row and its angles, no branch between (without
// a rotation the row's own bytes stand in for the angles and are not used), so that they are on their way with the page numbers; finish()
// makes the operand of them.  (Fetched where they are needed they took 7500 of an item's 25000 cycles: two round trips behind the tiles.)
// bf16 has a second operand, what the first one's rounding left, so that scores are as good as the pool's keys.  With one operand, and probabilities
// rounded once, the error against 64 bits is 2.9e-3 of y, of which 1.7e-3 is y's own rounding: more than one and a half times what it has to be.
// In FEW the further products are hidden (a block's products are 400 cycles of the 4400 that its bytes take).  In MANY they cost what they are: six
// prompts of 333 .. 4096 tokens, 18 / 6 heads of 64, 148 -> 169 us (2.5e-3 -> 2.1e-3), with 16 / 4 of 128 208 -> 257; 512 rows beside 15 tokens 56 -> 62
// (2.9e-3 -> 2.3e-3); 128 tokens behind 16001 keys, 16 / 4 heads of 128, 49 -> 55 (2.9e-3 -> 2.3e-3); 32 behind 8192 20.6 -> 21.0.  The probabilities in
// two parts instead: 188, 268, 67, 54 and 21.4, the same errors.
template <typename E, int D>
struct Query;
template <int D>
struct Query<uint16_t, D> {
  static constexpr int KS = D / 16;
  bf16x8 reg[KS], rest[KS];
  u32x4 raw[KS];
  f32x4 cs[KS], sn[KS];
  __device__ __forceinline__ void fetch(const segpt_paged_params& p, const uint16_t* row, int64_t angle, int hh) {
    const float* c = (p.rope_cos ? p.rope_cos + angle : reinterpret_cast<const float*>(row)) + 8 * hh;
    const float* s = (p.rope_cos ? p.rope_sin + angle : reinterpret_cast<const float*>(row)) + 8 * hh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) raw[ks] = *reinterpret_cast<const u32x4*>(row + 16 * ks + 8 * hh);
#pragma unroll
    for (int i = 0; i < KS; ++i) {  // floats 16 (i / 2) + 8 hh + 4 (i % 2) ..
      cs[i] = *reinterpret_cast<const f32x4*>(c + 16 * (i / 2) + 4 * (i % 2));
      sn[i] = *reinterpret_cast<const f32x4*>(s + 16 * (i / 2) + 4 * (i % 2));
    }
  }
  __device__ __forceinline__ void finish(const segpt_paged_params& p, bool live, int hh, const float* gsm) {
    float x[KS][8];
    unpack_b_layout<KS>(raw, x);
    if (p.rope_cos) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) rope_pair(x[i / 2][4 * (i % 2) + t], x[i / 2 + KS / 2][4 * (i % 2) + t], cs[i][t], sn[i][t]);
    }
    float sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int t = 0; t < 8; ++t) sq[t % 4] += x[ks][t] * x[ks][t];
    const float ss = half_sum((sq[0] + sq[1]) + (sq[2] + sq[3]));
    const float alpha = (p.flags & SEGPT_FLAG_NO_NORM) ? 1.f : __builtin_amdgcn_rsqf(ss * (1.0f / D) + p.eps);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const float4 ga = *reinterpret_cast<const float4*>(gsm + 16 * ks + 8 * hh), gb = *reinterpret_cast<const float4*>(gsm + 16 * ks + 8 * hh + 4);
      const float g[8] = {ga.x, ga.y, ga.z, ga.w, gb.x, gb.y, gb.z, gb.w};
      u32x4 w, r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t first, second;
        two_parts(x[ks][2 * i] * alpha * g[2 * i], x[ks][2 * i + 1] * alpha * g[2 * i + 1], first, second);
        w[i] = live ? first : 0u;
        r[i] = live ? second : 0u;
      }
      reg[ks] = as_bf16x8(w);
      rest[ks] = as_bf16x8(r);
    }
  }
};
template <int D>
struct Query<float, D> {
  static constexpr int C = D / 8;
  float reg[C][4];
  f32x4 cs[C / 2], sn[C / 2];
  __device__ __forceinline__ void fetch(const segpt_paged_params& p, const float* row, int64_t angle, int hh) {
    const float* c = (p.rope_cos ? p.rope_cos + angle : row) + 4 * hh;
    const float* s = (p.rope_cos ? p.rope_sin + angle : row) + 4 * hh;
#pragma unroll
    for (int i = 0; i < C; ++i) load16(row + 8 * i + 4 * hh, reg[i]);
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
      cs[i] = *reinterpret_cast<const f32x4*>(c + 8 * i);
      sn[i] = *reinterpret_cast<const f32x4*>(s + 8 * i);
    }
  }
  __device__ __forceinline__ void finish(const segpt_paged_params& p, bool live, int hh, const float* gsm) {
    if (p.rope_cos) {
#pragma unroll
      for (int c = 0; c < C / 2; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) rope_pair(reg[c][t], reg[c + C / 2][t], cs[c][t], sn[c][t]);
    }
    float sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) sq[t] += reg[c][t] * reg[c][t];
    const float ss = half_sum((sq[0] + sq[1]) + (sq[2] + sq[3]));
    const float alpha = (p.flags & SEGPT_FLAG_NO_NORM) ? 1.f : 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) reg[c][t] = live ? reg[c][t] * alpha * gsm[8 * c + 4 * hh + t] : 0.f;
  }
};

__device__ __forceinline__ float lds_read_f(uint32_t addr) { return *(const __attribute__((address_space(3))) float*)addr; }

template <typename E, int D>
__device__ __forceinline__ float gate_factor(const segpt_paged_params& p, int t, int h) {
  const E z = row_of<E>(p.gate, t, h)[0];
  float x;
  if constexpr (sizeof(E) == 2) x = bf16_to_f32(z); else x = z;
  return p.gate_scale / (1.0f + __expf(-x));
}

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
  constexpr int COLS = MANY ? kMany : kFew;
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
  it.slot = x.slot + ((it.tile * x.shares + it.part) * a.p.Hkv + it.g) * (COLS / 32);
  // row ranges that overlap may add up to more than 32 bits hold: nothing is written outside the scratch
  it.valid = it.tile >= 0 && (it.direct || (it.slot >= 0 && it.slot <= a.n_slots - COLS / 32));
  it.past = x.len - x.n;
  const int per = shares.of(x.blocks + x.shares - 1) * kBlock;  // shares as even as whole blocks allow
  const int last_col = min(it.cols, (it.tile + 1) * COLS) - 1, sees = it.prefix ? x.len : min(x.len, it.past + a.rep.of(last_col) + 1);
  it.k0 = it.part * per;
  it.nk = max(min(sees, it.k0 + per) - it.k0, 0);
  it.ids = it.prefix ? a.p.prefix_table : a.p.block_table + (int64_t)(x.entry - a.shared) * a.p.table_stride;
  return it;
}
// Page numbers of keys w0 .. w0 + wn - 1 into LDS; one that is not in the pool is replaced by page 0: returns whether this wave met one
__device__ __forceinline__ bool stage_table(const PagedArgs& a, const Item& it, int w0, int wn, int* table, int first, int step) {
  const int p0 = w0 >> a.log_page, pages = wn ? ((w0 + wn - 1) >> a.log_page) - p0 + 1 : 0;
  bool bad = false;
  for (int i = first; i < pages; i += step) {
    int id = it.ids[p0 + i];
    if ((uint32_t)id >= (uint32_t)a.p.n_pages) { id = 0; bad = true; }
    table[i] = id;
  }
  return __builtin_amdgcn_ballot_w64(bad) != 0;
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

// Requests of tiles of keys w0 .. w0 + wn - 1.  A load covers kRowsPerLoad rows, at most 8, of one page: its address is a scalar base and
// a lane offset.  LOADS loads a tensor and tile; number ps is load first + ps * step of the tile.  Where the rows of a load begin is worked out
// side by side, a lane a load, for as many tiles as there are lanes (27 of 72 vector instructions a block of MANY, one tile at a time);
// what a lane adds is the same for every whole tile.
template <typename E, int D, int BK, int LOADS>
struct Requests {
  using Z = Tile<E, D>;
  const char *kbase, *vbase;
  int64_t kpage, vpage;
  uint32_t kstep, vstep;
  int w0, wn, log_page, first, step, lane;
  const int* table;
  uint32_t klane[LOADS], vlane[LOADS];
  static constexpr int kAhead = 64 / LOADS;  // tiles worked out at a time
  int64_t kplace, vplace;                    // byte offsets from the head's first row, lane t * LOADS + ps: of load ps of the t-th of these tiles
  __device__ __forceinline__ int first_row(int jt, int ps) const {  // from w0 on; past the last key: the last rows once more
    return min(jt * BK + (ps * step + first) * Z::kRowsPerLoad, (wn - 1) & ~(Z::kRowsPerLoad - 1));
  }
  __device__ __forceinline__ uint32_t chunk(int ps) const {
    return (uint32_t)((lane % Z::kChunks) ^ Z::f((ps * step + first) * Z::kRowsPerLoad + lane / Z::kChunks)) << 4;
  }
  __device__ __forceinline__ void work_out(int jt) {  // tiles jt .. jt + kAhead - 1
    const int key = w0 + first_row(jt + lane / LOADS, lane % LOADS), page = table[(key >> log_page) - (w0 >> log_page)];
    const uint32_t slot = (uint32_t)(key & ((1 << log_page) - 1));
    kplace = page * kpage + (int64_t)((uint64_t)slot * kstep);
    vplace = page * vpage + (int64_t)((uint64_t)slot * vstep);
  }
  static __device__ __forceinline__ const char* at(const char* base, int64_t off, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)off, l), hi = __builtin_amdgcn_readlane((int)(off >> 32), l);
    return base + (int64_t)((uint64_t)hi << 32 | lo);
  }
  // the keys or values of tile jt; the first tile of every kAhead is asked for its keys first
  template <bool VALUES>
  __device__ __forceinline__ void issue(int jt, uint32_t dst) {
    const int l = jt % kAhead * LOADS;
    if (!VALUES && l == 0) work_out(jt);
    if (wn - jt * BK >= BK) {
#pragma unroll
      for (int ps = 0; ps < LOADS; ++ps)
        gload_lds16_so(VALUES ? at(vbase, vplace, l + ps) : at(kbase, kplace, l + ps), VALUES ? vlane[ps] : klane[ps], dst + (ps * step + first) * 1024);
    } else {
#pragma unroll
      for (int ps = 0; ps < LOADS; ++ps) {
        const uint32_t r = min(lane / Z::kChunks, wn - 1 - first_row(jt, ps));
        gload_lds16_so(VALUES ? at(vbase, vplace, l + ps) : at(kbase, kplace, l + ps), r * (VALUES ? vstep : kstep) + chunk(ps), dst + (ps * step + first) * 1024);
      }
    }
  }
};
template <typename E, int D, int BK, int LOADS>
__device__ __forceinline__ Requests<E, D, BK, LOADS> requests(const PagedArgs& a, const Item& it, const int* table, int first, int step, int lane) {
  const segpt_paged_params& p = a.p;
  Requests<E, D, BK, LOADS> r{page_row<E>(p.k_pages, 0, it.g, 0), page_row<E>(p.v_pages, 0, it.g, 0), p.k_pages.stride_b * (int)sizeof(E), p.v_pages.stride_b * (int)sizeof(E),
          (uint32_t)p.k_pages.stride_s * (int)sizeof(E), (uint32_t)p.v_pages.stride_s * (int)sizeof(E), it.k0, 0, a.log_page, first, step, lane, table};
#pragma unroll
  for (int ps = 0; ps < LOADS; ++ps) {
    r.klane[ps] = (uint32_t)(lane / Tile<E, D>::kChunks) * r.kstep + r.chunk(ps);
    r.vlane[ps] = (uint32_t)(lane / Tile<E, D>::kChunks) * r.vstep + r.chunk(ps);
  }
  return r;
}

// ---- a lane's column, and what it sees of the item's keys (counted from k0 on)
struct Column {
  int t, h;      // row and head
  bool live;
  int lim;       // last key of the lane's row
  int all, any;  // last key that all columns of the wave see, that any of them sees
};
template <typename E, int D>
__device__ __forceinline__ Column column_of(const PagedArgs& a, const Item& it, int rep, int wave_col, int lane, Query<E, D>& q) {
  const segpt_paged_params& p = a.p;
  Column c;
  const bool works = wave_col < it.cols;
  const int col = wave_col + (lane & 31), safe = min(col, it.cols - 1), i = a.rep.of(safe);
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
  q.fetch(p, row_of<E>(p.q, c.t, c.h), (p.rope_pos0 + pos) * (D / 2), lane >> 5);
  c.lim = min((it.prefix ? p.prefix_len : 0) + own - it.k0, it.nk - 1);
  if (it.prefix) {
    const bool cut = __builtin_amdgcn_ballot_w64(c.live && c.lim < it.nk - 1) != 0;  // rows that stand in the prefix
    c.all = !works || cut ? -1 : it.nk - 1;
    c.any = works ? it.nk - 1 : -1;
  } else {
    c.all = works ? min(it.past + a.rep.of(wave_col) - it.k0, it.nk - 1) : -1;
    c.any = works ? min(it.past + a.rep.of(min(wave_col + 31, it.cols - 1)) - it.k0, it.nk - 1) : -1;
  }
  return c;
}

// ---- one block of 32 keys: operands, softmax, products
// K' rows as the A operand
template <typename E, int D>
struct Keys;
template <int D>
struct Keys<uint16_t, D> {
  bf16x8 k[D / 16];
  __device__ __forceinline__ void read(uint32_t tile, int lane) {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) k[ks] = swz_frag_rm<D>(tile + swz_off_rm<D>(lane), 0, ks);
  }
  __device__ __forceinline__ f32x16 scores(const Query<uint16_t, D>& q, f32x16 s) const {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) s = mfma32(k[ks], q.rest[ks], s);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) s = mfma32(k[ks], q.reg[ks], s);
    return s;
  }
};
template <int D>
struct Keys<float, D> {
  f32x4 k[D / 8];
  __device__ __forceinline__ void read(uint32_t tile, int lane) {
    const uint32_t row = tile + (lane & 31) * (4 * D);
    const int fx = Tile<float, D>::f(lane & 31), hh = lane >> 5;
#pragma unroll
    for (int c = 0; c < D / 8; ++c) k[c] = lds_read_f4(row + (((2 * c + hh) ^ fx) << 4));
  }
  __device__ __forceinline__ f32x16 scores(const Query<float, D>& q, f32x16 s) const {
#pragma unroll
    for (int c = 0; c < D / 8; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[c][t], q.reg[c][t], s, 0, 0, 0);
    return s;
  }
};
// V' rows as the A operand of O^T.  A value that is not finite must reach the rows that see its key, and not the others as 0 * inf: in a block
// that not all rows see, clear() makes those 0 and says whether there were any; add_odd_values() puts them back behind the loop.
template <typename E, int D>
struct Values;
template <int D>
struct Values<uint16_t, D> {
  static constexpr int MB = D / 32;
  u32x4 v[MB][2];
  __device__ __forceinline__ void read(uint32_t tile, int lane) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) v[mb][s2] = __builtin_bit_cast(u32x4, swz_frag_tr<D>(tile + swz_off_tr<D>(lane), mb, s2));
  }
  __device__ __forceinline__ bool clear() {
    typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
    uint32_t all = ~0u;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // sign of |x| - inf: all ones where x is finite
          const uint32_t finite = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(i16x2, v[mb][s2][e] & 0x7fff7fffu) - (int16_t)0x7f80) >> 15);
          v[mb][s2][e] &= finite;
          all &= finite;
        }
        asm volatile("" : "+v"(v[mb][s2]));  // whole registers again: as bf16 vectors they would be taken apart, element by element
      }
    return all != ~0u;
  }
  // Adds the probabilities s to the sums l and their products with the values to o.  FINE: in two bf16 parts, so that y's own rounding is all its error
  // (2.3e-3 of y -> 1.65e-3).  FEW has it beside its loads (32 tokens of 200 .. 8192 keys 44.3 -> 44.7 us, 48 of 255 .. 16000 153 -> 155); in MANY,
  // the prompts above would take 214 us instead of 169: there they are rounded once and summed as rounded.
  template <bool FINE>
  __device__ __forceinline__ void add(f32x16 s, float (&l)[2], f32x16 (&o)[MB]) const {
    bf16x8 pb[2], rest[2];
    if constexpr (FINE) {
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        u32x4 w, r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = s[8 * s2 + 2 * i], b = s[8 * s2 + 2 * i + 1];
          uint32_t first, second;
          two_parts(a, b, first, second);
          w[i] = first;
          r[i] = second;
          l[0] += a;
          l[1] += b;
        }
        pb[s2] = as_bf16x8(w);
        rest[s2] = as_bf16x8(r);
      }
    } else {
      pb[0] = pack_c_half_sum(s, 0, l);
      pb[1] = pack_c_half_sum(s, 1, l);
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        if constexpr (FINE) o[mb] = mfma32(as_bf16x8(v[mb][s2]), rest[s2], o[mb]);
        o[mb] = mfma32(as_bf16x8(v[mb][s2]), pb[s2], o[mb]);
      }
  }
};
template <int D>
struct Values<float, D> {
  static constexpr int MB = D / 32;
  float v[MB][16];  // step r contracts key c_r = 8 (r / 4) + r % 4 (lower half of the wave) and c_r + 4 (upper half): register r of the scores as it is
  __device__ __forceinline__ void read(uint32_t tile, int lane) {
    const int ln = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = 8 * (r >> 2) + (r & 3) + 4 * hh;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) v[mb][r] = lds_read_f(tile + key * (4 * D) + (((8 * mb + (ln >> 2)) ^ Tile<float, D>::f(key)) << 4) + 4 * (ln & 3));
    }
  }
  __device__ __forceinline__ bool clear() {
    bool odd = false;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool no = !(fabsf(v[mb][r]) < INFINITY);
        odd |= no;
        if (no) v[mb][r] = 0.f;
      }
    return odd;
  }
  template <bool FINE>
  __device__ __forceinline__ void add(f32x16 s, float (&l)[2], f32x16 (&o)[MB]) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) l[r & 1] += s[r];
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o[mb] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[mb][r], s[r], o[mb], 0, 0, 0);
  }
};
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

// The values that Values::clear() left out of the product, key by key, for the rows that see them: their probability is positive, so a sum
// with one is that value, or NaN where signs meet.
template <typename E, int D, int BK>
__device__ __forceinline__ void add_odd_values(const PagedArgs& a, const Item& it, const Column& c, int hh, f32x16 (&o)[D / 32]) {
  for (int j = (max(c.all, -1) + 1) / BK * BK; j <= c.any; ++j) {  // tiles that not all rows see whole
    const int key = it.k0 + j, page = it.ids[key >> a.log_page];
    if ((uint32_t)page >= (uint32_t)a.p.n_pages) continue;  // the rows are NaN as a whole
    const E* row = reinterpret_cast<const E*>(page_row<E>(a.p.v_pages, page, it.g, key & ((1 << a.log_page) - 1)));
#pragma unroll
    for (int mb = 0; mb < D / 32; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const E e = row[32 * mb + 8 * (r >> 2) + 4 * hh + (r & 3)];
        float v;
        if constexpr (sizeof(E) == 2) v = bf16_to_f32(e); else v = e;
        if (j <= c.lim && !(fabsf(v) < INFINITY)) o[mb][r] += v;
      }
  }
}

// What an item leaves: y where it is its tile's only one, else a partial result
template <typename E, int D>
__device__ __forceinline__ void store_result(const PagedArgs& a, const Item& it, const Column& c, State<D / 32>& st, bool bad, int slot_col, int hh) {
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

// this wave's LDS reads have returned (before what they came from is requested over), its LDS writes are there
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0) only
}

// ---- FEW: one wave, up to 32 columns.  kDepth buffers for the keys of a block and as many for its values, each requested again as soon
// as its reader has it in registers.  Order of the requests: keys, values of blocks 0 .. kDepth - 1, then keys, values of each further block.
template <typename E, int D>
__device__ __forceinline__ void few_columns(const PagedArgs& a, const Item& it, int rep, int lane, uint32_t lds, int* table, float* gsm) {
  using S = Shape<E, D>;
  constexpr int LOADS = kBlock * S::kRB / 1024;
  const int hh = lane >> 5, window = S::kFewTable << a.log_page;
  constexpr int DEPTH = S::kDepth;
  constexpr uint32_t kBuffer = S::kFewBytes / 2;
  auto rq = requests<E, D, kBlock, LOADS>(a, it, table, 0, 1, lane);
  rq.wn = min(it.nk, window);
  // one round trip: gain, query row and angles, page numbers
  Gain gain[(D + 63) / 64];
#pragma unroll
  for (int i = 0; i < (D + 63) / 64; ++i) gain[i] = fetch_gain(a.p, (64 * i + lane) % D);
  Query<E, D> q;
  const Column c = column_of(a, it, rep, it.tile * kFew, lane, q);
  bool bad = it.x.broken | stage_table(a, it, rq.w0, rq.wn, table, lane, 64);
#pragma unroll
  for (int i = 0; i < (D + 63) / 64; ++i)
    if (64 * i + lane < D) gsm[64 * i + lane] = scale_of(a.p, gain[i]);
  wave_sync();
  auto start_window = [&] {
#pragma unroll
    for (int t = 0; t < DEPTH; ++t)
      if (t * kBlock < rq.wn) {
        rq.template issue<false>(t, lds + 2 * t * kBuffer);
        rq.template issue<true>(t, lds + (2 * t + 1) * kBuffer);
      }
  };
  // leaves the loads of the n youngest tiles (keys or values) in flight
  auto wait_but = [&](int n) {
    if (n == 0) wait_vmcnt<0>();
    else if (n == 1) wait_vmcnt<LOADS>();
    else if (n == 2) wait_vmcnt<2 * LOADS>();
    else wait_vmcnt<3 * LOADS>();
  };
  start_window();
  q.finish(a.p, c.live, hh, gsm);
  State<D / 32> st;
  st.clear();
  bool odd = false;
  while (true) {
    const int n_kt = (rq.wn + kBlock - 1) / kBlock, off = rq.w0 - it.k0;
    wait_vmcnt<0>();  // the loads below are counted: nothing of the start may be in flight with them
    uint32_t buffer = 0;
    for (int jt = 0; jt < n_kt; ++jt) {
      const int left = n_kt - 1 - jt;
      const uint32_t kt = lds + 2 * buffer * kBuffer, vt = kt + kBuffer;
      const int seen = c.lim - off - jt * kBlock;
      const bool masked = off + jt * kBlock + kBlock - 1 > c.all;
      wait_but(1 + 2 * min(left, DEPTH - 1));  // the keys are there; its values and the other buffers' tiles are younger
      wave_sync();
      Keys<E, D> k;
      k.read(kt, lane);
      wave_sync();
      if (left >= DEPTH) rq.template issue<false>(jt + DEPTH, kt);
      f32x16 s[1] = {k.scores(q, st.less)};
      if (masked) hide_unseen(s[0], seen, hh);
      st.raise(s);
      st.exponentials(s);
      wait_but(2 * min(left, DEPTH - 1) + (left >= DEPTH));  // the values; the other buffers' tiles and the keys just requested are younger
      wave_sync();
      Values<E, D> v;
      v.read(vt, lane);
      if (masked) odd |= v.clear();
      wave_sync();
      if (left >= DEPTH) rq.template issue<true>(jt + DEPTH, vt);
      v.template add<true>(s[0], st.l, st.o);
      buffer = buffer == DEPTH - 1 ? 0 : buffer + 1;
    }
    rq.w0 += window;
    if (rq.w0 >= it.k0 + it.nk) break;
    rq.wn = min(it.k0 + it.nk - rq.w0, window);
    bad |= stage_table(a, it, rq.w0, rq.wn, table, lane, 64);
    wave_sync();
    start_window();
  }
  if (__builtin_amdgcn_ballot_w64(odd) != 0) add_odd_values<E, D, kBlock>(a, it, c, hh, st.o);
  store_result<E, D>(a, it, c, st, bad, lane & 31, hh);
}

// ---- MANY: four waves of 32 columns around a ring of stages (K' tile, V' tile); tile jt lives in stage jt % kStages.  A turn computes the
// scores of tile jt + 1 beside the exponentials of tile jt and its product with the values, so that the matrix pipe has work while
// the exponentials are formed.  Per turn: wait for tile jt + 1, barrier (also: everyone has left tile jt - 1), request tile jt + kStages - 1 over
// that one, compute.
// Six prompts of 333 .. 4096 tokens, 18 / 6 heads of 64: the matrix pipe is busy for 41 % of the time (a third of it with the query's second part), the
// vector port for 52 %, 8 vector instructions a matrix instruction; with two waves a SIMD neither is full.  A third of the cycles of the LDS are
// bank conflicts at 128-byte rows.  A prompt of 8192 tokens takes 232 us (666 TFLOP/s without the second part's products); short shares are bound
// by their start, about 10 us until the first products.
template <typename E, int D>
__device__ __forceinline__ void many_columns(const PagedArgs& a, const Item& it, int rep, int tid, uint32_t lds, int* table, float* gsm, int* any_bad) {
  using S = Shape<E, D>;
  constexpr int BK = S::kBK, NS = S::kStages, LOADS = S::kTileBytes / 1024 / 4;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, window = S::kManyTable << a.log_page;
  auto rq = requests<E, D, BK, LOADS>(a, it, table, wave, 4, lane);
  rq.w0 = it.k0;
  rq.wn = min(it.nk, window);
  bool bad = it.x.broken;
  auto stage_pages = [&] {
    const bool mine = stage_table(a, it, rq.w0, rq.wn, table, tid, 256);
    if (lane == 0) any_bad[wave] = mine;
  };
  auto request = [&](int jt, uint32_t stage) {
    rq.template issue<false>(jt, lds + stage);
    rq.template issue<true>(jt, lds + stage + S::kTileBytes);
  };
  auto start_window = [&] {
#pragma unroll
    for (int w = 0; w < 4; ++w) bad |= any_bad[w] != 0;
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
      if (t * BK < rq.wn) request(t, t * S::kStageBytes);
  };
  // one round trip: gain, query row and angles, page numbers
  const Gain gain = fetch_gain(a.p, tid % D);
  Query<E, D> q;
  const Column c = column_of(a, it, rep, it.tile * kMany + wave * 32, lane, q);
  stage_pages();
  if (tid < D) gsm[tid] = scale_of(a.p, gain);
  __syncthreads();
  start_window();
  q.finish(a.p, c.live, hh, gsm);
  State<D / 32> st;
  st.clear();
  bool odd = false;
  constexpr int N = BK / 32;  // blocks of a tile
  typedef f32x16 Scores[N];
  auto read_keys = [&](Keys<E, D> (&k)[N], uint32_t stage) {
#pragma unroll
    for (int n = 0; n < N; ++n) k[n].read(lds + stage + n * 32 * S::kRB, lane);
  };
  auto read_values = [&](Values<E, D> (&v)[N], uint32_t stage) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n].read(lds + stage + S::kTileBytes + n * 32 * S::kRB, lane);
  };
  auto scores = [&](auto masked_c, const Keys<E, D> (&k)[N], Scores& s, int jb) {  // of the tile whose keys begin at jb, from k0 on
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = k[n].scores(q, st.less);
    if (decltype(masked_c)::value != 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) hide_unseen(s[n], c.lim - jb - 32 * n, hh);
    }
  };
  while (true) {
    const int n_kt = (rq.wn + BK - 1) / BK, off = rq.w0 - it.k0;
    wait_vmcnt<0>();  // the loads below are counted: nothing of the start may be in flight with them
    __syncthreads();
    uint32_t stage = 0;  // of tile jt
    auto stage_from = [&](int steps) {  // of tile jt + steps
      const uint32_t x = stage + steps * S::kStageBytes;
      return x >= NS * S::kStageBytes ? x - NS * S::kStageBytes : x;
    };
    auto turn = [&](int jt) {
      if (n_kt - 2 - jt >= NS - 3) wait_vmcnt<(NS - 3) * 2 * LOADS>(); else wait_vmcnt<0>();
      __syncthreads();
      if (jt + NS - 1 < n_kt) request(jt + NS - 1, stage_from(NS - 1));
    };
    auto active = [&](int jt) { return jt < n_kt && off + jt * BK <= c.any; };  // some column of the wave sees a key of the tile
    const int n_whole = max(min((c.all + 1 - off) / BK, n_kt), 0);  // tiles that all columns of the wave see whole
    Scores s0, s1;
    if (active(0)) {
      Keys<E, D> k[N];
      read_keys(k, 0);
      scores(IC<1>{}, k, s0, off);
      st.raise(s0);
    }
    auto both_whole = [&](int jt, Scores& s, Scores& ahead) {  // neither tile jt nor the next needs a mask
      turn(jt);
      Keys<E, D> k[N];
      Values<E, D> v[N];
      read_keys(k, stage_from(1));
      read_values(v, stage);
      scores(IC<0>{}, k, ahead, 0);
      st.exponentials(s);
#pragma unroll
      for (int n = 0; n < N; ++n) v[n].template add<false>(s[n], st.l, st.o);
      st.raise(ahead);
      stage = stage_from(1);
    };
    auto any_tiles = [&](int jt, Scores& s, Scores& ahead) {
      turn(jt);
      if (active(jt)) {
        Values<E, D> v[N];
        read_values(v, stage);
        if (jt >= n_whole) {
#pragma unroll
          for (int n = 0; n < N; ++n) odd |= v[n].clear();
        }
        st.exponentials(s);
#pragma unroll
        for (int n = 0; n < N; ++n) v[n].template add<false>(s[n], st.l, st.o);
      }
      if (active(jt + 1)) {
        Keys<E, D> k[N];
        read_keys(k, stage_from(1));
        scores(IC<1>{}, k, ahead, off + (jt + 1) * BK);
        st.raise(ahead);
      }
      stage = stage_from(1);
    };
    // two turns a round, so that the scores change places without being copied
    int jt = 0;
    for (; jt + 2 < n_whole; jt += 2) {
      both_whole(jt, s0, s1);
      both_whole(jt + 1, s1, s0);
    }
    for (; jt < n_kt; jt += 2) {
      any_tiles(jt, s0, s1);
      if (jt + 1 < n_kt) any_tiles(jt + 1, s1, s0);
    }
    rq.w0 += window;
    if (rq.w0 >= it.k0 + it.nk) break;
    rq.wn = min(it.k0 + it.nk - rq.w0, window);
    __syncthreads();  // everyone is done with the page numbers and the stages
    stage_pages();
    __syncthreads();
    start_window();
  }
  if (__builtin_amdgcn_ballot_w64(odd) != 0) add_odd_values<E, D, BK>(a, it, c, hh, st.o);
  store_result<E, D>(a, it, c, st, bad, wave * 32 + (lane & 31), hh);
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

// Launches whose entries are all FEW: a workgroup is one wave, eight a CU (twelve: the same work in more shares, 49.6 -> 52.5 us).  Bound by HBM:
// 32 tokens, 200 .. 8192 keys, 18 / 6 heads of 64: 213 MB in 45 us (4.7 TB/s); 48 tokens, 255 .. 16000 keys, 16 / 4 heads of 128: 803 MB in 149 us
// (5.4 TB/s).  A single token's 4096 keys take 8.7 us: launch and three dependent round trips (lengths, page numbers, keys); the plan's arithmetic is 0.3.
template <typename E, int D>
__global__ __launch_bounds__(64, (Shape<E, D>::kOcc)) void paged_few_kernel(PagedArgs a) {
  using S = Shape<E, D>;
  __shared__ __attribute__((aligned(1024))) char lds[S::kDepth * S::kFewBytes];
  __shared__ __attribute__((aligned(16))) float gsm[D];
  __shared__ int table[S::kFewTable + 2];
  const int lane = threadIdx.x, rep = a.rep.d;
  clear_rest<E>(a, lane, 64, D);
  const Entries mine = kept_entries(a, lane, rep);
  const Shares share = share_blocks(a, mine);
  leave_plan(a, lane, rep, share, mine);
  const Item it = locate<false>(a, lane, rep, share, mine, blockIdx.x);
  if (it.valid) few_columns<E, D>(a, it, rep, lane, lds_addr_of(lds), table, gsm);
}

// Any launch: the first workgroups are items of many columns, the next four items each of few, the rest have none.  (With a fixed number of
// workgroups for the first kind those without an item, which still go through the plan, kept the second kind waiting: 128 rows beside 15 tokens 45.9
// instead of 40.4 us.)
template <typename E, int D>
__global__ __launch_bounds__(256, (Shape<E, D>::kOcc)) void paged_any_kernel(PagedArgs a) {
  using S = Shape<E, D>;
  constexpr int kLds = std::max(S::kManyBytes, 4 * S::kDepth * S::kFewBytes);
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  __shared__ __attribute__((aligned(16))) float gsm[4][D];
  __shared__ int table[S::kManyTable + 8];
  __shared__ int any_bad[4];
  static_assert(4 * (S::kFewTable + 2) <= S::kManyTable + 8, "four waves' page numbers");
  const int tid = threadIdx.x, lane = tid & 63, rep = a.rep.d;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  clear_rest<E>(a, tid, 256, D);
  const Entries mine = kept_entries(a, lane, rep);
  const Shares share = share_blocks(a, mine);
  leave_plan(a, lane, rep, share, mine);
  const Item it = locate<true>(a, lane, rep, share, mine, blockIdx.x);
  if (it.x.entry >= 0) {
    if (it.valid) many_columns<E, D>(a, it, rep, tid, lds_addr_of(lds), table, gsm[0], any_bad);
  } else {
    const Item it4 = locate<false>(a, lane, rep, share, mine, ((int)blockIdx.x - it.x.base) * 4 + wave);
    if (it4.valid) few_columns<E, D>(a, it4, rep, lane, lds_addr_of(lds) + wave * S::kDepth * S::kFewBytes, table + wave * (S::kFewTable + 2), gsm[wave]);
  }
}

// Joins the partial results of `per_sub` columns of a tile: its sequence's shares and, behind them, the prefix's.  A unit of D / 4 lanes holds a
// row; as many units stand side by side over the shares of a column as leave each one batch of kBatch that is requested together, and
// their sums meet in LDS.  Fixed order: deterministic.  4.9 us for one token of 18 heads (launch and two round trips), 5.9 for 32 of them, 12 for
// 128 tokens of 16 heads of 128 behind a prefix (25 MB).
constexpr int kMergeThreads = 256;
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
  const int which = blockIdx.x / subs, sub = blockIdx.x - which * subs;
  if (which >= joins) return;
  const Shares share = shares_from(few, many);
  const Found own = find_entry<kFindJoin>(a, lane, rep, share, mine, which);
  if (own.entry < 0) return;
  const int tile = a.hkv.of(which - own.base), g = which - own.base - tile * p.Hkv, cols = own.n * rep, tile_cols = own.many ? kMany : kFew;
  Found pre{-1, 0, 0, 0, 0, 0, 0, 0, false, false};
  if (a.shared) pre = find_entry<kFindFirst>(a, lane, rep, share, mine, 0);
  const int pre_cols = pre.many ? kMany : kFew;
  const int n = own.shares + pre.shares;
  int step = min(per_sub, kUnits);  // columns at a time
  while (step > 1 && kUnits / step * kBatch < n) step >>= 1;
  const int wide = kUnits / step;  // units of a column
  for (int c0 = sub * per_sub; c0 < min((sub + 1) * per_sub, tile_cols); c0 += step) {  // the same for all threads
    if (tile * tile_cols + c0 >= cols) return;
    const int col = tile * tile_cols + min(c0 + unit % step, tile_cols - 1);
    const bool live = col < cols && c0 + unit % step < min((sub + 1) * per_sub, tile_cols);
    const int i = a.rep.of(min(col, cols - 1)), t = own.first + i, h = g * rep + (min(col, cols - 1) - i * rep);
    const int pcol = (t - pre.first) * rep + h - g * rep, ptile = pcol / pre_cols;
    auto place = [&](int s) {  // row of share s among all partial results; none: there is no room for it
      const bool is_own = s < own.shares;
      const Found& x = is_own ? own : pre;
      const int slot = x.slot + (((is_own ? tile : ptile) * x.shares + (is_own ? s : s - own.shares)) * p.Hkv + g) * (x.many ? kMany / 32 : 1);
      return slot < a.n_slots - (x.many ? kMany / 32 - 1 : 0) ? (int64_t)slot * 32 + (is_own ? col - tile * tile_cols : pcol - ptile * pre_cols) : (int64_t)-1;
    };
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
    if (p.gate.ptr) f *= gate_factor<E, D>(p, t, h);
    E* out = row_of<E>(p.o, t, h) + 4 * c;
    const float v[4] = {y.x * f, y.y * f, y.z * f, y.w * f};
    if constexpr (sizeof(E) == 2) *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    else store16(out, v);
  }
}

// ---- host side
bool all_few(const segpt_paged_params& p) {  // known on the host
  return !p.prefix_table && !p.seq_start && (int64_t)p.H / p.Hkv * (p.T / p.B) <= kFew;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// fills the plan; returns the scratch bytes
size_t plan(const segpt_paged_params& p, PagedArgs& a) {
  const int row_bytes = p.D * (p.dtype == SEGPT_DTYPE_FP32 ? 4 : 2), rep = p.H / p.Hkv;
  a.rep.set(rep);
  a.hkv.set(p.Hkv);
  a.shared = p.prefix_table ? 1 : 0;
  a.entries = p.B + a.shared;
  a.rows_each = p.seq_start ? 0 : p.T / p.B;
  a.each.set(p.seq_start ? 1 : a.rows_each);
  a.log_page = __builtin_ctz((unsigned)p.page_size);
  a.capacity = paged_capacity(p);
  // 512 workgroups are resident, two a CU.  The shares' length is found in three steps and may leave a few more than asked for, and one that has to wait
  // for a place is a round of its own: 480 are asked for, 496 where all are single waves (us, asked for 512 and now; 18 / 6 heads of 64, up to 8192 keys:
  // 512 rows beside 31 tokens 78, 73; beside 63 132, 111; beside 15 66, 66; 128 rows beside 15 40.7, 45.2; eight fp32 tokens 19.9, 17.8; 128 of bf16
  // 102, 103).  Where the host sees that the work is of many columns (a prefix, prompts of equal length) three on two CUs: longer shares leave a
  // quarter less to be joined, which is more than the idle places would have done (512 and 384: a prompt of 1024 tokens 33.6, 31.0, of 2048 46.2, 42.8,
  // of 8192 237, 237, four of 512 34.8, 21.3; 32 tokens behind 8192 keys 23.3, 21.8; 128 behind 16001, 16 / 4 heads of 128, 57 .. 60 either way).  fp32 rows
  // of 512 bytes: one a CU, all of them (256 and 224: 32 tokens of 16 / 4 heads 48.5, 53.6; 100 122, 134; of 4 / 2 heads 80, 66).
  const bool wide = a.shared || (!p.seq_start && (int64_t)rep * a.rows_each > kFew);
  a.target = row_bytes > 256 ? 256 : wide ? 384 : p.seq_start ? 480 : 496;
  a.min_few = 2;
  a.min_many = 4;
  // Tiles: whole ones of the columns there are, and one begun an entry.  Items: a tile's part of what the target stands for, and one begun.
  const int64_t cols = (int64_t)p.T * rep;
  int64_t many = cols / kMany + std::min<int64_t>(p.B, cols / (kFew + 1)), few = std::min<int64_t>(p.B, p.T);
  if (!p.seq_start) {
    const int64_t each = cols / p.B;
    many = each > kFew ? (each + kMany - 1) / kMany * p.B : 0;
    few = each > kFew ? 0 : p.B;
  }
  const int64_t own = many + few, own_many = many;
  if (a.shared && cols > kFew) many += (cols + kMany - 1) / kMany;
  else if (a.shared) few += 1;
  const int64_t slack = 64;  // the sum that gives the length of a share is rounded
  const int64_t n_many = many ? many * p.Hkv + a.target + slack : 0, n_few = few ? few * p.Hkv + 4 * a.target + slack : 0;
  a.n_many = (int32_t)std::min<int64_t>(n_many, INT32_MAX);
  a.n_few = (int32_t)std::min<int64_t>(n_few, INT32_MAX);
  // a tile that leaves partial results has two shares or more, i.e. at most twice its part of the target; beside a prefix all leave them
  const int64_t most = (int64_t)a.target + slack;
  const int64_t slots = kMany / 32 * (a.shared ? n_many : std::min(n_many, 2 * most)) + (a.shared ? n_few : std::min(n_few, 8 * most));
  a.n_slots = (int32_t)std::min<int64_t>(slots, INT32_MAX / 32);
  const int64_t joins = a.shared ? own * p.Hkv : std::min(own_many * p.Hkv, most) + std::min((own - own_many) * p.Hkv, 4 * most);
  a.n_joins = (int32_t)std::min<int64_t>(joins, INT32_MAX);
  a.planned_bytes = a.entries > kKept * 64 ? (size_t)4 * a.entries * sizeof(int32_t) : 0;
  // a launch has fewer than 2^32 threads (the merge: a workgroup a join at least)
  const int64_t most_groups = UINT32_MAX / 256;
  return n_many + (n_few + 3) / 4 > most_groups || joins > most_groups || slots > INT32_MAX / 32 ? SIZE_MAX : 256 + up256(a.planned_bytes) + (size_t)a.n_slots * 32 * (p.D + 2) * sizeof(float);
}

template <typename E, int D>
int launch(const PagedArgs& a, hipStream_t st) {
  const segpt_paged_params& p = a.p;
  if (a.upto) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  if (all_few(p)) hipLaunchKernelGGL((paged_few_kernel<E, D>), dim3((unsigned)a.n_few), dim3(64), 0, st, a);
  else hipLaunchKernelGGL((paged_any_kernel<E, D>), dim3((unsigned)(a.n_many + (a.n_few + 3) / 4)), dim3(256), 0, st, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
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

extern "C" {

size_t segpt_paged_workspace_bytes(const segpt_paged_params* p) {
  using namespace segpt;
  if (check_paged_sizes(p, false) != SEGPT_OK) return 0;
  PagedArgs a{};
  const size_t n = plan(*p, a);
  return n > SIZE_MAX - 256 ? 0 : up256(n);
}

int segpt_paged_attn(const segpt_paged_params* p, void* stream) {
  using namespace segpt;
  const int rc = check_paged(p, false);
  if (rc) return rc;
  PagedArgs a{};
  a.p = *p;
  const size_t need = plan(*p, a);
  if (need > SIZE_MAX - 256) return SEGPT_E_SHAPE;
  if (!p->workspace || p->workspace_bytes < up256(need)) return SEGPT_E_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(p->workspace) & 255u) return SEGPT_E_ALIGN;
  a.lens = reinterpret_cast<int32_t*>(p->workspace);
  if (a.planned_bytes) a.upto = a.lens + 256 / sizeof(int32_t);
  a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(p->workspace) + 256 + up256(a.planned_bytes));
  a.stat = reinterpret_cast<float2*>(a.part + (size_t)a.n_slots * 32 * p->D);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p->dtype == SEGPT_DTYPE_BF16) return p->D == 64 ? launch<uint16_t, 64>(a, st) : launch<uint16_t, 128>(a, st);
  return p->D == 32 ? launch<float, 32>(a, st) : p->D == 64 ? launch<float, 64>(a, st) : launch<float, 128>(a, st);
}

}  // extern "C"
