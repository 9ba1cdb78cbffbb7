// Attention over a paged key/value cache of 8 or 4 bits, forward only: what paged_attn.hip does for pools of bf16 and fp32, with the same
// division of the work (paged_work.hpp), for pools whose rows are codes in blocks of 32 components with a power-of-two scale each.
//
//   y_i = sum_j exp(s_ij - lse_i) v'_j      s_ij = qhat_i . k'_j      k'_j, v'_j = code * 2^e, exact in bf16
//
// A code times its scale is a bf16 number, so the codes are made bf16 operands in registers (one instruction a pair of components, the scale as
// its operand) and everything behind that is bf16 matrix products with fp32 sums, whatever the rows are: bf16 rows bring their queries in two bf16
// parts, fp32 rows queries and probabilities in three, and neither loses anything of the keys and values as stored.
//
// Single tokens are bound by the bytes of the rows that they read behind a start of 8 us (plan, page numbers, query), longer calls by the issue of vector
// and matrix instructions together.  Tiles of few columns are of 16 here: a wave reads a block of keys with half the registers of 32 and three of them
// fit a SIMD, and two tiles that read the same rows meet in the cache.
#define SEGPT_FEW_COLUMNS 16
#define SEGPT_JOIN_COLUMNS
#include "paged_quant.hpp"
#include "paged_work.hpp"

namespace segpt {
namespace {

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// PARTS bf16 parts of a pair of values: the first ones cut off (two_parts), the last one rounded
template <int PARTS>
__device__ __forceinline__ void parts_of(float a, float b, uint32_t (&w)[PARTS]) {
  if constexpr (PARTS == 1) {
    w[0] = pack_bf16x2(a, b);
  } else {
    constexpr float kBelow = 1.f - 0x1p-9f;
#pragma unroll
    for (int i = 0; i < PARTS - 1; ++i) {
      const uint32_t x = __float_as_uint(a * kBelow) & 0xffff0000u, y = __float_as_uint(b * kBelow) & 0xffff0000u;
      w[i] = x >> 16 | y;
      a -= __uint_as_float(x);
      b -= __uint_as_float(y);
    }
    w[PARTS - 1] = pack_bf16x2(a, b);
  }
}
template <typename E>
constexpr int kQueryParts = sizeof(E) == 2 ? 2 : 3;

// eight elements of a row, as they are stored
template <typename E>
struct Eight;
template <>
struct Eight<uint16_t> {
  u32x4 w;
  __device__ __forceinline__ void load(const uint16_t* p) { w = *reinterpret_cast<const u32x4*>(p); }
  __device__ __forceinline__ void values(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = bf16lo(w[i]); x[2 * i + 1] = bf16hi(w[i]); }
  }
};
template <>
struct Eight<float> {
  f32x4 u, v;
  __device__ __forceinline__ void load(const float* p) { u = *reinterpret_cast<const f32x4*>(p); v = *reinterpret_cast<const f32x4*>(p + 4); }
  __device__ __forceinline__ void values(float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = u[i]; x[4 + i] = v[i]; }
  }
};
// and of a table
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 u = *reinterpret_cast<const float4*>(p), v = *reinterpret_cast<const float4*>(p + 4);
  x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
}

// this wave's LDS reads have returned (before what they came from is written over), its LDS writes are there
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0) only
}

// ---- where the rows of an item lie.  One wave goes through tiles of rows that stand side by side, `STEP` keys from one tile's first to the next one's; a
// lane works out the places of one tile, 64 tiles at a time, from a page number that was asked for 64 tiles before.  A page number that is not in the
// pool is replaced by 0 and remembered.  A tile past the item's last key is the last one there is once more.
// In LDS, or where registers are at hand in those.
template <int ROWS, int STEP, bool LDS>  // ROWS: of a tile, which begins at a multiple of them: of one page, or 16 of two pages of eight
struct Walk {
  static constexpr int kBytes = 64 * 4 * 8;  // of LDS
  const int* ids;
  int first, last, log_page, tiles;  // keys of the first tile and of the item's last; tiles there are
  int upto;                          // tiles that have been worked out, the last 64 of them kept
  int next;                          // page number of tile upto + lane
  int64_t place[LDS ? 1 : 4];        // byte offsets of tile upto - 64 + lane from the kv head's first rows: keys, values, their scales
  uint32_t lds;
  int apart;                         // pages of eight: from the first eight rows' page to that of the others
  bool bad;
  __device__ __forceinline__ int key_of(int tile) const { return min(first + tile * STEP, last & ~(ROWS - 1)); }
  __device__ __forceinline__ int ask(int tile) const { return tiles ? ids[key_of(tile) >> log_page] : 0; }
  __device__ __forceinline__ void start(const PagedArgs& a, const Item& it, int offset, int n, int lane, uint32_t lds_at) {
    lds = lds_at;
    ids = it.ids;
    first = it.k0 + offset;
    last = it.k0 + it.nk - 1;
    log_page = a.log_page;
    tiles = n;
    upto = 0;
    bad = false;
    next = ask(lane);
  }
  __device__ __forceinline__ int checked(const PagedArgs& a, int id) {
    if ((uint32_t)id < (uint32_t)a.p.n_pages) return id;
    bad = true;
    return 0;
  }
  __device__ __forceinline__ void work_out(const QuantArgs& qa, const PagedArgs& a, int lane) {
    const segpt_paged_params& p = qa.p;
    const int key = key_of(upto + lane), id = checked(a, next);
    const uint32_t slot = (uint32_t)(key & ((1 << log_page) - 1));
    const segpt_tensor4* all[4] = {&p.k_pages, &p.v_pages, &qa.k_scales, &qa.v_scales};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t at = (int64_t)id * all[i]->stride_b + (int64_t)slot * all[i]->stride_s;
      if constexpr (LDS) *(__attribute__((address_space(3))) int64_t*)(lds + 512 * i + 8 * lane) = at;
      else place[i] = at;
    }
    if constexpr (LDS) wave_sync();
    if (ROWS > 8 && log_page == 3) apart = key + 8 <= last && tiles ? checked(a, ids[(key + 8) >> 3]) - id : 0;
    upto += 64;
    if (upto < tiles) next = ask(upto + lane);
  }
  // first row of tile l of those, in tensor i
  __device__ __forceinline__ const char* at(int i, const char* base, int l) const {
    uint32_t lo, hi;
    if constexpr (LDS) {
      const u32x2 off = *(const __attribute__((address_space(3))) u32x2*)(lds + 512 * i + 8 * l);
      lo = __builtin_amdgcn_readfirstlane((int)off[0]);
      hi = __builtin_amdgcn_readfirstlane((int)off[1]);
    } else {
      lo = __builtin_amdgcn_readlane((int)place[i], l);
      hi = __builtin_amdgcn_readlane((int)(place[i] >> 32), l);
    }
    return base + (int64_t)((uint64_t)hi << 32 | lo);
  }
};

struct Args {
  PagedArgs w;
  segpt_tensor4 k_scales, v_scales;
};
__device__ __forceinline__ QuantArgs quant_of(const Args& a) { return {a.w.p, a.k_scales, a.v_scales}; }
// The kernel's arguments (its only ones) from memory once more, for what is hardly ever needed: else they wait in registers from the start
__device__ __forceinline__ const Args& arguments() {
  auto at = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return *(const Args*)at;
}

// What a lane asks for of one row of keys or values: WORDS words of codes, and the scales of the whole row
template <int WORDS>
struct RowPart {
  uint32_t w[WORDS];
  uint32_t s;
};
template <int D>
__device__ __forceinline__ uint32_t load_scales(const char* at) {  // D / 32 bytes, aligned to them
  if constexpr (D == 128) return *reinterpret_cast<const uint32_t*>(at);
  else if constexpr (D == 64) return *reinterpret_cast<const uint16_t*>(at);
  else return *reinterpret_cast<const uint8_t*>(at);
}
template <int BYTES>
__device__ __forceinline__ void load_words(const char* at, uint32_t* w) {
  if constexpr (BYTES == 16) { const u32x4 x = *reinterpret_cast<const u32x4*>(at); w[0] = x[0]; w[1] = x[1]; w[2] = x[2]; w[3] = x[3]; }
  else if constexpr (BYTES == 4) w[0] = *reinterpret_cast<const uint32_t*>(at);
  else { const u32x2 x = *reinterpret_cast<const u32x2*>(at); w[0] = x[0]; w[1] = x[1]; }
}
__device__ __forceinline__ float scale_at(uint32_t scales, int block) { return __uint_as_float((scales >> (8 * block) & 255u) << 23); }

// A lane's part of a row of every tile: NP pieces of P bytes, 4 P apart, the first at byte `from`
template <int D, int NP, int P>
struct Source {
  const char *k, *v, *ks, *vs;  // first rows of the kv head
  uint32_t kr, vr, ksr, vsr;    // bytes from row to row
  uint32_t from, klane, vlane, kslane, vslane;  // what a lane adds in a whole tile
  int row;
  __device__ __forceinline__ void start(const QuantArgs& a, int g, int own_row, uint32_t own_from) {
    k = byte_row(a.p.k_pages, 0, g, 0);
    v = byte_row(a.p.v_pages, 0, g, 0);
    ks = byte_row(a.k_scales, 0, g, 0);
    vs = byte_row(a.v_scales, 0, g, 0);
    kr = (uint32_t)a.p.k_pages.stride_s; vr = (uint32_t)a.p.v_pages.stride_s; ksr = (uint32_t)a.k_scales.stride_s; vsr = (uint32_t)a.v_scales.stride_s;
    row = own_row;
    from = own_from;
    klane = row * kr + from; vlane = row * vr + from; kslane = row * ksr; vslane = row * vsr;
  }
  static __device__ __forceinline__ void get(const char* base, uint32_t off, uint32_t (&w)[NP * P / 4]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) load_words<P>(base + (off + i * 4 * P), w + i * P / 4);
  }
  // tile: of the 64 that were worked out last
  template <int ROWS, int STEP, bool LDS>
  __device__ __forceinline__ void ask(const Walk<ROWS, STEP, LDS>& w, const QuantArgs& qa, int tile, RowPart<NP * P / 4>& x, RowPart<NP * P / 4>& y) const {
    const int l = tile & 63, left = w.last - w.key_of(tile);
    const char *kp = w.at(0, k, l), *vp = w.at(1, v, l), *ksp = w.at(2, ks, l), *vsp = w.at(3, vs, l);
    uint32_t ko = klane, vo = vlane, kso = kslane, vso = vslane;
    if (left < ROWS - 1) {  // past the last key: its row once more
      const uint32_t r = min(row, left);
      ko = r * kr + from; vo = r * vr + from; kso = r * ksr; vso = r * vsr;
    }
    if (ROWS > 8 && w.log_page == 3) {  // the second eight rows lie in a page of their own
      const bool second = min(row, left) >= 8;
      const int pages = lane_value(w.apart, l);  // outside the condition: the lane that is asked need not be among those that want it
      const int64_t by = second ? pages : 0;
      auto moved = [&](const char* base, int64_t page, uint32_t step) { return base + (by * page - (second ? (int64_t)8 * step : 0)); };
      get(moved(kp, qa.p.k_pages.stride_b, kr), ko, x.w);
      x.s = load_scales<D>(moved(ksp, qa.k_scales.stride_b, ksr) + kso);
      get(moved(vp, qa.p.v_pages.stride_b, vr), vo, y.w);
      y.s = load_scales<D>(moved(vsp, qa.v_scales.stride_b, vsr) + vso);
    } else {
      get(kp, ko, x.w);
      x.s = load_scales<D>(ksp + kso);
      get(vp, vo, y.w);
      y.s = load_scales<D>(vsp + vso);
    }
  }
};

// ---- FEW: one wave, up to 16 columns.  A score tile is 16 keys by 16 columns; a lane takes a quarter of a key's row, so that a row is read
// whole by four lanes and is the A operand as it is decoded, no LDS in between: the components that a lane contributes to a step are not those of
// the instruction's own order, but the queries' are the same, and a sum does not ask.  Probabilities go to the values in two bf16 parts, fp32 rows' in
// three.  One or two blocks of codes are under way while another is worked on.  32 tokens of 18 / 6 heads of 64, 200 .. 8192 keys, 8 bits: 25.5 us, 110 MB at
// 4.3 TB/s; 48 tokens of 16 / 4 heads of 128, 255 .. 16000 keys, 4 bits: 49 us, 214 MB at 4.3 TB/s; one token, 4096 keys: 7.5.  Of the vector
// instructions of the 32 tokens two fifths are the start of the items, of nine blocks each; fewer and longer ones leave the memory idle (target_of).
template <int D, int FMT>
struct Quarter {
  static constexpr int kBytes = Codes<FMT>::row_bytes(D) / 4;   // of a lane
  static constexpr int P = kBytes < 16 ? kBytes : 16, NP = kBytes / P, kWords = kBytes / 4;
  static constexpr int EP = P * 8 / Codes<FMT>::kBits;          // components of a piece: 8, 16 or 32, of one block
  static constexpr int KS = D / 32;                             // steps of the product
  static constexpr int kWordsOf8 = Codes<FMT>::kBits / 4;       // words of eight components
  static __device__ __forceinline__ int component(int step, int quarter) { return (step * 8 / EP) * 4 * EP + quarter * EP + step * 8 % EP; }
  static __device__ __forceinline__ int block(int piece, int quarter) { return (piece * 4 * EP + quarter * EP) / SEGPT_SCALE_BLOCK; }
  // the row's part as operands, 8 components each
  static __device__ __forceinline__ void decode(const RowPart<kWords>& x, int quarter, u32x4 (&out)[KS]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const float scale = scale_at(x.s, block(i, quarter));
#pragma unroll
      for (int u = 0; u < EP / 8; ++u) {
        uint32_t r[4];
        decode8<FMT>(x.w + i * (P / 4) + u * kWordsOf8, scale, r);
        out[i * (EP / 8) + u] = u32x4{r[0], r[1], r[2], r[3]};
      }
    }
  }
};
// Rows of 32 components lie in LDS as the first halves of rows of 64.
template <int D>
constexpr int kTileDim = D < 64 ? 64 : D;
// The values of a block of 32 keys in LDS, bf16: chunk c (16 bytes) of row r lies at chunk c ^ f(r).  Sixteen lanes write one chunk of 16 rows, and a
// transposing read takes two chunks of eight rows at a time; as groups of sixteen lanes both meet all banks once.  (Two fifths of the LDS cycles are counted
// as conflicts all the same; the LDS is busy for 17 % of the time at head_dim 64, 30 % at 128.)
template <int D>
struct ValueTile {
  static constexpr int kRB = 2 * D, kBytes = kBlock * kRB;
  static __device__ __forceinline__ int f(int row) { return (D == 64 ? 2 * (row >> 1 & 3) : 2 * (row & 7)) | (row >> 3 & 1); }
  static __device__ __forceinline__ uint32_t write_at(int row, int chunk) { return row * kRB + ((chunk ^ f(row & 15)) << 4); }
  // where lane's address lies for the operand of components 16 db .. and, of each quarter of the wave, its four keys of the first 16
  static __device__ __forceinline__ uint32_t read_at(int lane, int db) {
    const int r = lane & 15, row = 4 * (lane >> 4) + (r >> 2);
    return row * kRB + (((2 * db + (r >> 1 & 1)) ^ f(row)) << 4) + ((r & 1) << 3);
  }
  static __device__ __forceinline__ u32x4 read(uint32_t tile, int lane, int db) {
    typedef s16x4 __attribute__((address_space(3))) * lds_s16x4_ptr;
    const uint32_t at = tile + read_at(lane, db);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(at + 16 * kRB));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(u32x4, v);
  }
};
__device__ __forceinline__ void lds_write16(uint32_t addr, u32x4 v) { *(__attribute__((address_space(3))) u32x4*)addr = v; }

// The queries of 16 columns: a lane has a quarter of a column's pairs, works them out, and the parts reach the operand's order through LDS (the
// value tile's, which is not in use yet)
template <typename E, int D, int FMT>
struct Query16 {
  using L = Quarter<D, FMT>;
  static constexpr int KS = L::KS, kCols = 16, kLogCols = 4, PARTS = kQueryParts<E>, N = D < 64 ? 1 : D / 64;
  bf16x8 part[PARTS][KS];
  Eight<E> raw[2][N];
  float cs[N][8], sn[N][8];  // pairs of(quarter, n) .. + 7
  static __device__ __forceinline__ int of(int quarter, int n) { return D < 64 ? (quarter & 1) * 8 : (quarter * N + n) * 8; }  // 16 pairs: twice each
  __device__ __forceinline__ void fetch(const segpt_paged_params& p, const E* at, int64_t angle, int quarter) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int j = of(quarter, n);
      raw[0][n].load(at + j);
      raw[1][n].load(at + j + D / 2);
      if (p.rope_cos) {
        load8(p.rope_cos + angle + j, cs[n]);
        load8(p.rope_sin + angle + j, sn[n]);
      }
    }
  }
  __device__ __forceinline__ void finish(const segpt_paged_params& p, bool live, int lane, const float* gsm, uint32_t lds) {
    using V = ValueTile<kTileDim<D>>;
    const int quarter = lane >> 4, col = lane & 15;
    float x[2][N][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < N; ++n) raw[h][n].values(x[h][n]);
    if (p.rope_cos) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int t = 0; t < 8; ++t) rope_pair(x[0][n][t], x[1][n][t], cs[n][t], sn[n][t]);
    }
    float sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int t = 0; t < 8; ++t) sq[t % 4] += x[h][n][t] * x[h][n][t];
    float ss = (sq[0] + sq[1]) + (sq[2] + sq[3]);
    ss += __shfl_xor(ss, 16, 64);
    if (D >= 64) ss = half_sum(ss);
    const float alpha = !live ? 0.f : (p.flags & SEGPT_FLAG_NO_NORM) ? 1.f : 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
    u32x4 w[PARTS][2][N];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float g[8];
        load8(gsm + of(quarter, n) + h * (D / 2), g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t part_i[PARTS];
          parts_of<PARTS>(live ? x[h][n][2 * i] * alpha * g[2 * i] : 0.f, live ? x[h][n][2 * i + 1] * alpha * g[2 * i + 1] : 0.f, part_i);
#pragma unroll
          for (int u = 0; u < PARTS; ++u) w[u][h][n][i] = part_i[u];
        }
      }
#pragma unroll
    for (int u = 0; u < PARTS; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < N; ++n) lds_write16(lds + V::write_at(col, of(quarter, n) / 8 + h * (D / 16)), w[u][h][n]);
      wave_sync();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) part[u][ks] = as_bf16x8(lds_read16(lds + V::write_at(col, L::component(ks, quarter) / 8)));
      wave_sync();
    }
  }
};

// A value that is not finite (NaN by its scale or code, or beyond the largest number) must reach the rows that see its key, and not the others as 0 * NaN:
// in a block that not all rows see it is made 0 and noted, and put back behind the loop
__device__ __forceinline__ bool clear_odd(u32x4& v) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  uint32_t all = ~0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {  // sign of |x| - inf: all ones where x is finite
    const uint32_t finite = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(i16x2, v[e] & 0x7fff7fffu) - (int16_t)0x7f80) >> 15);
    v[e] &= finite;
    all &= finite;
  }
  asm volatile("" : "+v"(v));  // whole registers again: as bf16 vectors they would be taken apart, element by element
  return all != ~0u;
}
// Adds those that clear_odd() left out to what the item has left, y or a partial result, key by key from j0 on (counted from k0) for the rows that see them:
// their probability is positive, so a sum with one is that value, or NaN where signs meet.  A lane has the components that it wrote: four of every STEP,
// from `from` on.  Behind the results, in memory, and with the arguments read again, so that the loop before has the registers to itself (32 tokens 30.2 us;
// added to the sums before they are written 32.2).
template <typename E, int D, int FMT, int STEP>
__device__ __forceinline__ void add_odd_values(const Item& it, const Column& c, int j0, int slot_col, int from) {
  if (!c.live) return;
  const Args& qa = arguments();
  const PagedArgs& a = qa.w;
  float* part = a.part + ((int64_t)it.slot * 32 + slot_col) * D;
  E* out = row_of<E>(a.p.o, c.t, c.h);
  const float f = it.direct && a.p.gate.ptr ? gate_factor<E, D>(a.p, c.t, c.h) : 1.f;
  for (int j = j0; j <= c.lim; ++j) {
    const int key = it.k0 + j, page = it.ids[key >> a.log_page], slot = key & ((1 << a.log_page) - 1);
    if ((uint32_t)page >= (uint32_t)a.p.n_pages) continue;  // the row is NaN as a whole
    const char* row = byte_row(a.p.v_pages, page, it.g, slot);
    const uint32_t scales = load_scales<D>(byte_row(qa.v_scales, page, it.g, slot));
#pragma unroll 1
    for (int at = from; at < D; at += STEP) {
      const float scale = scale_at(scales, at / SEGPT_SCALE_BLOCK);
      uint32_t w;
      if constexpr (Codes<FMT>::k8) w = *reinterpret_cast<const uint32_t*>(row + at);
      else w = *reinterpret_cast<const uint16_t*>(row + at / 2);
      const uint32_t x[2] = {decode_bf16x2<FMT, 0>(w, scale), decode_bf16x2<FMT, 1>(w, scale)};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = r & 1 ? bf16hi(x[r / 2]) : bf16lo(x[r / 2]);
        if (fabsf(v) < INFINITY) continue;
        if (!it.direct) part[at + r] += v;
        else if constexpr (sizeof(E) == 2) out[at + r] = f32_to_bf16(bf16_to_f32(out[at + r]) + v * f);
        else out[at + r] += v * f;
      }
    }
  }
}

// AHEAD: blocks under way
template <typename E, int D, int FMT, int AHEAD>
__device__ __forceinline__ void few_columns(const QuantArgs& qa, const PagedArgs& a, const Item& it, int rep, int lane, uint32_t lds, float* gsm) {
  using L = Quarter<D, FMT>;
  using V = ValueTile<kTileDim<D>>;
  constexpr int KS = L::KS, DB = D / 16, PARTS = kQueryParts<E>;
  const segpt_paged_params& p = a.p;
  const int quarter = lane >> 4, r16 = lane & 15;
  const int blocks = (it.nk + kBlock - 1) / kBlock;
  // one round trip: gain, query rows and angles, page numbers
  Walk<16, 16, false> walk;
  walk.start(a, it, 0, 2 * blocks, lane, 0);
  Gain gain[(D + 63) / 64];
#pragma unroll
  for (int i = 0; i < (D + 63) / 64; ++i) gain[i] = fetch_gain(p, (64 * i + lane) % D);
  Query16<E, D, FMT> q;
  const Column c = column_of<E, D>(a, it, rep, it.tile * kFew, lane, q);
  Source<D, L::NP, L::P> src;
  src.start(qa, it.g, r16, (uint32_t)quarter * L::P);
  struct Block {
    RowPart<L::kWords> k[2], v[2];
  };
  auto ask = [&](Block& b, int j) {
#pragma unroll
    for (int t = 0; t < 2; ++t) src.ask(walk, qa, 2 * j + t, b.k[t], b.v[t]);
  };
  Block b0, b1;
  walk.work_out(qa, a, lane);
  if (blocks > 0) ask(b0, 0);
#pragma unroll
  for (int i = 0; i < (D + 63) / 64; ++i)
    if (64 * i + lane < D) gsm[64 * i + lane] = scale_of(p, gain[i]);
  wave_sync();
  q.finish(p, c.live, lane, gsm, lds);
  if (AHEAD == 2 && blocks > 1) ask(b1, 1);

  f32x4 o[DB];
  float m = 0.f, limit = -INFINITY, l = 0.f;  // reference (log2 units); by how much a score may exceed it; sum over this lane's keys
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  bool odd = false;
  auto step = [&](Block& b, int j) {
    const bool masked = j * kBlock + kBlock - 1 > c.all;
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u32x4 k[KS];
      L::decode(b.k[t], quarter, k);
      s[t] = f32x4{-m, -m, -m, -m};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int u = PARTS - 1; u >= 0; --u) s[t] = mfma16(as_bf16x8(k[ks]), q.part[u][ks], s[t]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u32x4 v[KS];
      L::decode(b.v[t], quarter, v);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) lds_write16(lds + V::write_at(16 * t + r16, L::component(ks, quarter) / 8), v[ks]);
    }
    if (j + AHEAD < blocks) ask(b, j + AHEAD);
    if (masked) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int seen = c.lim - j * kBlock - 16 * t - 4 * quarter;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r > seen) s[t][r] = -INFINITY;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i / 4][i % 4]);
    if (__builtin_amdgcn_ballot_w64(top > limit) != 0) {  // a lane's own keys may tell; the column's reference is one for its four lanes
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = half_max(top);
      const float up = top > limit ? top : 0.f, corr = limit == -INFINITY ? 1.f : fast_exp2(-up);  // nothing to scale before the first key
      m += up;
      if (top > limit) limit = kLazy;
      l *= corr;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[db][r] *= corr;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i % 4] -= up;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i / 4][i % 4] = fast_exp2(s[i / 4][i % 4]);
      l += s[i / 4][i % 4];
    }
    u32x4 pb[PARTS];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t w[PARTS];
      parts_of<PARTS>(s[i / 2][i % 2 * 2], s[i / 2][i % 2 * 2 + 1], w);
#pragma unroll
      for (int u = 0; u < PARTS; ++u) pb[u][i] = w[u];
    }
    wave_sync();
    u32x4 v[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) v[db] = V::read(lds, lane, db);
    if (masked) {
#pragma unroll
      for (int db = 0; db < DB; ++db) odd |= clear_odd(v[db]);
    }
#pragma unroll
    for (int u = PARTS - 1; u >= 0; --u)
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = mfma16(as_bf16x8(v[db]), as_bf16x8(pb[u]), o[db]);
    wave_sync();
  };
  for (int j = 0; j < blocks; j += AHEAD) {
    if ((2 * j + 2 * AHEAD) % 64 == 0 && j + AHEAD < blocks) walk.work_out(qa, a, lane);  // the next tiles asked for: 2 AHEAD of them from 2 j + 2 AHEAD on
    step(b0, j);
    if (AHEAD == 2 && j + 1 < blocks) step(b1, j + 1);
  }
  const bool bad = it.x.broken | (__builtin_amdgcn_ballot_w64(walk.bad) != 0);
  float sum = l + __shfl_xor(l, 16, 64), ref = limit == -INFINITY ? -INFINITY : m;
  sum = half_sum(sum);
  if (bad) { sum = __builtin_nanf(""); ref = 0.f; }
  if (c.live && !it.direct) {
    const int64_t at = (int64_t)it.slot * 32 + r16;
#pragma unroll
    for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(a.part + at * D + 16 * db + 4 * quarter) = o[db];
    if (quarter == 0) a.stat[at] = make_float2(ref, sum);
  } else if (c.live) {
    float f = sum == 0.f ? 0.f : 1.0f / sum;
    if (p.lse && quarter == 0) p.lse[(int64_t)c.t * p.H + c.h] = sum == 0.f ? -INFINITY : (ref + __log2f(sum)) * kLn2;
    if (p.gate.ptr) f *= gate_factor<E, D>(p, c.t, c.h);
    E* out = row_of<E>(p.o, c.t, c.h) + 4 * quarter;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const float y[4] = {o[db][0] * f, o[db][1] * f, o[db][2] * f, o[db][3] * f};
      if constexpr (sizeof(E) == 2) *reinterpret_cast<u32x2*>(out + 16 * db) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      else store16(out + 16 * db, y);
    }
  }
  if (__builtin_amdgcn_ballot_w64(odd) != 0) add_odd_values<E, D, FMT, 16>(it, c, (max(c.all, -1) + 1) / kBlock * kBlock, r16, 4 * quarter);
}

// ---- MANY: four waves of 32 columns around a ring of three stages (K' tile, V' tile of bf16); tile jt lives in stage jt % 3.  The codes of a tile are
// asked for three turns before its products, kept in registers for one, and decoded into LDS.  The scores of a block of 32 keys are computed beside the
// exponentials of the block before it and its product with the values.  bf16 rows' probabilities are rounded once: with their second part the error of y
// would go from 2.3e-3 to its own rounding's 1.7e-3, for half as many matrix instructions again.  One prompt of 8192 rows, 18 / 6 heads of 64: 246 us,
// 0.94 PFLOP/s with the queries' second part; 512 rows beside 31 tokens, 100 .. 8192 keys: 62 us, vector instructions half of it, matrix a quarter.
// At heads of 128 with bf16 rows, two workgroups a CU, 57 (8 bits) and 39 (4 bits) vector registers live in scratch, 168 and 156 bytes a lane.
template <int D>
struct ManyShape {
  static constexpr int kBK = D == 128 ? 32 : 64, kRB = 2 * kTileDim<D>, kTileBytes = kBK * kRB, kStageBytes = 2 * kTileBytes, kStages = 3;
  static constexpr int kPart = D == 32 ? 8 : 16, kLanes = D / kPart, kRows = 64 / kLanes;  // components of a lane, lanes of a row, rows of a wave
  static_assert(4 * kRows == kBK);
};
template <typename E, int D>
struct Query32 {
  static constexpr int KS = D / 16, kCols = 32, kLogCols = 5, PARTS = kQueryParts<E>;
  bf16x8 part[PARTS][KS];
  Eight<E> raw[KS];
  float cs[KS / 2][8], sn[KS / 2][8];
  __device__ __forceinline__ void fetch(const segpt_paged_params& p, const E* row, int64_t angle, int hh) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) raw[ks].load(row + 16 * ks + 8 * hh);
    if (!p.rope_cos) return;
#pragma unroll
    for (int ks = 0; ks < KS / 2; ++ks) {
      load8(p.rope_cos + angle + 16 * ks + 8 * hh, cs[ks]);
      load8(p.rope_sin + angle + 16 * ks + 8 * hh, sn[ks]);
    }
  }
  __device__ __forceinline__ void finish(const segpt_paged_params& p, bool live, int hh, const float* gsm) {
    float x[KS][8];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) raw[ks].values(x[ks]);
    if (p.rope_cos) {
#pragma unroll
      for (int ks = 0; ks < KS / 2; ++ks)
#pragma unroll
        for (int t = 0; t < 8; ++t) rope_pair(x[ks][t], x[ks + KS / 2][t], cs[ks][t], sn[ks][t]);
    }
    float sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int t = 0; t < 8; ++t) sq[t % 4] += x[ks][t] * x[ks][t];
    const float ss = half_sum((sq[0] + sq[1]) + (sq[2] + sq[3]));
    const float alpha = (p.flags & SEGPT_FLAG_NO_NORM) ? 1.f : 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float g[8];
      load8(gsm + 16 * ks + 8 * hh, g);
      u32x4 w[PARTS];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t part_i[PARTS];
        parts_of<PARTS>(x[ks][2 * i] * alpha * g[2 * i], x[ks][2 * i + 1] * alpha * g[2 * i + 1], part_i);
#pragma unroll
        for (int u = 0; u < PARTS; ++u) w[u][i] = live ? part_i[u] : 0u;
      }
#pragma unroll
      for (int u = 0; u < PARTS; ++u) part[u][ks] = as_bf16x8(w[u]);
    }
  }
};

// Sums of a column at head_dim 128.  State keeps the reference's negative in sixteen registers, so that scores come out of the product less it; here
// those registers hold keys on their way to it, and the reference is taken off behind the product, beside matrix instructions that take longer.
template <int MB>
struct StateLess {
  f32x16 o[MB], less;  // less: 0
  float m, top_allowed;  // reference (log2 units), and by what a score may exceed it
  float l[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) o[mb] = splat16(0.f);
    less = splat16(0.f);
    m = 0.f;
    top_allowed = -INFINITY;
    l[0] = l[1] = 0.f;
  }
  __device__ __forceinline__ float reference() const { return top_allowed == -INFINITY ? -INFINITY : m; }
  __device__ __forceinline__ void raise(f32x16 (&s)[1]) {
    float top = s[0][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[0][r]);
    top = half_max(top);
    if (__builtin_amdgcn_ballot_w64(top > top_allowed) != 0) {
      const bool up = top > top_allowed;
      const float corr = !up || top_allowed == -INFINITY ? 1.f : fast_exp2(m - top);  // nothing to scale before the first key
      if (up) { m = top; top_allowed = top + kLazy; }
      l[0] *= corr;
      l[1] *= corr;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[mb][r] *= corr;
    }
  }
  __device__ __forceinline__ void exponentials(f32x16 (&s)[1]) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = fast_exp2(s[0][r] - m);
  }
};

template <typename E, int D, int FMT>
__device__ __forceinline__ void many_columns(const QuantArgs& qa, const PagedArgs& a, const Item& it, int rep, int tid, uint32_t lds, uint32_t places, float* gsm,
                                             int* any_bad) {
  using S = ManyShape<D>;
  constexpr int BK = S::kBK, N = BK / 32, MB = D / 32, KS = D / 16, PARTS = kQueryParts<E>, PROBS = sizeof(E) == 2 ? 1 : 3;
  constexpr int P = S::kPart * Codes<FMT>::kBits / 8, TD = kTileDim<D>;  // P: bytes of a lane's components
  const segpt_paged_params& p = a.p;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const int own_row = lane / S::kLanes, own_part = lane % S::kLanes, n_kt = (it.nk + BK - 1) / BK;
  // one round trip: gain, query row and angles, page numbers
  Walk<S::kRows, BK, true> walk;
  walk.start(a, it, wave * S::kRows, n_kt, lane, places + wave * decltype(walk)::kBytes);
  const Gain gain = fetch_gain(p, tid % D);
  Query32<E, D> q;
  const Column c = column_of<E, D>(a, it, rep, it.tile * kMany + wave * 32, lane, q);
  Source<D, 1, P> src;
  src.start(qa, it.g, own_row, (uint32_t)own_part * P);
  struct Raw2 {
    RowPart<P / 4> k, v;
  };
  auto ask = [&](Raw2& x, int jt) {
    if (jt >= n_kt) return;
    src.ask(walk, qa, jt, x.k, x.v);
  };
  auto put = [&](const Raw2& x, int jt, uint32_t stage) {
    if (jt >= n_kt) return;
    const int row = wave * S::kRows + own_row, f = Swz<TD>::f(row);
    auto tensor = [&](const RowPart<P / 4>& r, uint32_t at) {
      const float scale = scale_at(r.s, own_part * S::kPart / SEGPT_SCALE_BLOCK);
#pragma unroll
      for (int u = 0; u < S::kPart / 8; ++u) {
        uint32_t w[4];
        decode8<FMT>(r.w + u * (Codes<FMT>::kBits / 4), scale, w);
        lds_write16(at + row * S::kRB + (((S::kPart / 8 * own_part + u) ^ f) << 4), u32x4{w[0], w[1], w[2], w[3]});
      }
    };
    tensor(x.k, lds + stage);
    tensor(x.v, lds + stage + S::kTileBytes);
  };
  Raw2 x, x1;
  walk.work_out(qa, a, lane);
  ask(x, 0);
  ask(x1, 1);
  if (tid < D) gsm[tid] = scale_of(p, gain);
  __syncthreads();
  q.finish(p, c.live, hh, gsm);
  put(x, 0, 0);
  ask(x, 2);
  put(x1, 1, S::kStageBytes);
  std::conditional_t<D != 128, State<MB>, StateLess<MB>> st;
  st.clear();
  bool odd = false;
  typedef f32x16 Scores[1];
  // Keys of the block after this one: read as soon as they are there, beside the decoding of a later tile's codes; at head_dim 128 there are no
  // registers for that (with more of them in scratch six prompts take 301 us instead of 288).
  constexpr bool EARLY = D != 128;
  typedef bf16x8 Keys[KS];
  auto read_keys = [&](uint32_t block, Keys& k) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k[ks] = swz_frag_rm<TD>(lds + block + swz_off_rm<TD>(lane), 0, ks);
  };
  auto scores = [&](bool masked, const Keys& k, Scores& s, int jb) {  // of the block of 32 keys k, jb on from k0
    s[0] = st.less;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = PARTS - 1; u >= 0; --u) s[0] = mfma32(k[ks], q.part[u][ks], s[0]);
    if (masked) hide_unseen(s[0], c.lim - jb, hh);
  };
  auto products = [&](bool masked, uint32_t block, Scores& s) {
    st.exponentials(s);
    u32x4 pb[PROBS][2];
    if constexpr (PROBS == 1) {
      pb[0][0] = __builtin_bit_cast(u32x4, pack_c_half_sum(s[0], 0, st.l));
      pb[0][1] = __builtin_bit_cast(u32x4, pack_c_half_sum(s[0], 1, st.l));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t w[PROBS];
        parts_of<PROBS>(s[0][2 * i], s[0][2 * i + 1], w);
#pragma unroll
        for (int u = 0; u < PROBS; ++u) pb[u][i / 4][i % 4] = w[u];
        st.l[0] += s[0][2 * i];
        st.l[1] += s[0][2 * i + 1];
      }
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        u32x4 v = __builtin_bit_cast(u32x4, swz_frag_tr<TD>(lds + block + S::kTileBytes + swz_off_tr<TD>(lane), mb, s2));
        if (masked) odd |= clear_odd(v);
#pragma unroll
        for (int u = PROBS - 1; u >= 0; --u) st.o[mb] = mfma32(as_bf16x8(v), as_bf16x8(pb[u][s2]), st.o[mb]);
      }
  };
  uint32_t stage = 0;  // of the tile that the turn is about
  auto stage_from = [&](int steps) {
    const uint32_t at = stage + steps * S::kStageBytes;
    return at >= S::kStages * S::kStageBytes ? at - S::kStages * S::kStageBytes : at;
  };
  const int n_blocks = n_kt * N;
  auto active = [&](int b) { return b < n_blocks && b * 32 <= c.any; };  // some column of the wave sees a key of the block
  const int n_whole = max(min((c.all + 1) / 32, n_blocks), 0);             // blocks that all columns of the wave see whole
  Scores s0, s1;
  __syncthreads();
  if (active(0)) {
    Keys k;
    read_keys(0, k);
    scores(true, k, s0, 0);
    st.raise(s0);
  }
  Keys ahead_k;
  auto turn = [&](int jt, uint32_t block) {  // block: whose keys are wanted next
    __syncthreads();  // tile jt + 1 is there; everyone has left tile jt - 1
    if (EARLY) read_keys(block, ahead_k);
    put(x, jt + 2, stage_from(2));
    if ((jt + 3) % 64 == 0 && jt + 3 < n_kt) walk.work_out(qa, a, lane);
    ask(x, jt + 3);
  };
  // block b of s, and the scores of the next one beside it; HALF: b is the first of a tile of two
  auto whole = [&](auto half, Scores& s, Scores& ahead) {
    constexpr bool HALF = decltype(half)::value != 0;
    if (!EARLY || !HALF) read_keys(HALF ? stage + 32 * S::kRB : stage_from(1), ahead_k);
    scores(false, ahead_k, ahead, 0);
    products(false, HALF || N == 1 ? stage : stage + 32 * S::kRB, s);
    st.raise(ahead);
    if (!HALF) stage = stage_from(1);
  };
  auto any = [&](auto half, int b, Scores& s, Scores& ahead) {
    constexpr bool HALF = decltype(half)::value != 0;
    if (active(b)) products(b >= n_whole, HALF || N == 1 ? stage : stage + 32 * S::kRB, s);
    if (active(b + 1)) {
      if (!EARLY || !HALF) read_keys(HALF ? stage + 32 * S::kRB : stage_from(1), ahead_k);
      scores(true, ahead_k, ahead, (b + 1) * 32);
      st.raise(ahead);
    }
    if (!HALF) stage = stage_from(1);
  };
  // two blocks a round, so that the scores change places without being copied
  int b = 0;
  for (; b + 2 < n_whole; b += 2) {
    turn(b / N, N == 2 ? stage + 32 * S::kRB : stage_from(1));
    whole(IC<N == 2>{}, s0, s1);
    if (N == 1) turn(b + 1, stage_from(1));
    whole(IC<0>{}, s1, s0);
  }
  for (; b < n_blocks; b += 2) {
    turn(b / N, N == 2 ? stage + 32 * S::kRB : stage_from(1));
    any(IC<N == 2>{}, b, s0, s1);
    if (b + 1 >= n_blocks) break;
    if (N == 1) turn(b + 1, stage_from(1));
    any(IC<0>{}, b + 1, s1, s0);
  }
  // a wave looks up the pages of its own rows of a tile, and multiplies by all of them
  const bool mine = __builtin_amdgcn_ballot_w64(walk.bad) != 0;
  if (lane == 0) any_bad[wave] = mine;
  __syncthreads();
  const bool bad = it.x.broken | ((any_bad[0] | any_bad[1] | any_bad[2] | any_bad[3]) != 0);
  store_result<E, D>(a, it, c, st, bad, wave * 32 + (lane & 31), hh);
  if (__builtin_amdgcn_ballot_w64(odd) != 0) add_odd_values<E, D, FMT, 8>(it, c, (max(c.all, -1) + 1) / BK * BK, wave * 32 + (lane & 31), 4 * hh);
}

// Launches whose entries are all FEW: a workgroup is one wave
template <int D>
constexpr int kFewWaves = D == 128 ? 2 : 3;  // waves a SIMD that registers leave room for (128 tokens of up to 3000 keys: 62 us with two, 53)
template <typename E, int D, int FMT>
__global__ __launch_bounds__(64, kFewWaves<D>) void paged_quant_few_kernel(Args args) {
  const PagedArgs& a = args.w;
  __shared__ __attribute__((aligned(1024))) char lds[ValueTile<kTileDim<D>>::kBytes];
  __shared__ __attribute__((aligned(16))) float gsm[D];
  const int lane = threadIdx.x, rep = a.rep.d;
  clear_rest<E>(a, lane, 64, D);
  const Entries mine = kept_entries(a, lane, rep);
  const Shares share = share_blocks(a, mine);
  leave_plan(a, lane, rep, share, mine);
  const Item it = locate<false>(a, lane, rep, share, mine, blockIdx.x);
  if (!it.valid) return;
  const QuantArgs qa = quant_of(args);
  // one where a second would not leave the registers for the waves: 48 tokens of heads of 128 at 8 bits 97 -> 89 us, with fp32 rows 142 -> 91, at 4 bits the
  // other way for bf16 rows (57 and 58); 128 tokens of heads of 64 in fp32 59 -> 52 with the third wave, 32 in bf16 the other way (30.7 and 32.1).
  // The kernel below has two for all: its registers go by the items of many columns.
  constexpr int AHEAD = sizeof(E) == 2 && Codes<FMT>::row_bytes(D) <= 64 ? 2 : 1;
  few_columns<E, D, FMT, AHEAD>(qa, a, it, rep, lane, lds_addr_of(lds), gsm);
}

// Any launch: the first workgroups are items of many columns, the next four items each of few, the rest have none
template <typename E, int D, int FMT>
__global__ __launch_bounds__(256, (sizeof(E) == 2 || D != 128 ? 2 : 1)) void paged_quant_any_kernel(Args args) {
  const PagedArgs& a = args.w;
  using S = ManyShape<D>;
  constexpr int kLds = std::max(S::kStages * S::kStageBytes, 4 * ValueTile<kTileDim<D>>::kBytes);
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  __shared__ __attribute__((aligned(16))) float gsm[4][D];
  __shared__ __attribute__((aligned(16))) char places[4 * Walk<S::kRows, S::kBK, true>::kBytes];
  __shared__ int any_bad[4];
  const int tid = threadIdx.x, lane = tid & 63, rep = a.rep.d;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  clear_rest<E>(a, tid, 256, D);
  const Entries mine = kept_entries(a, lane, rep);
  const Shares share = share_blocks(a, mine);
  leave_plan(a, lane, rep, share, mine);
  const QuantArgs qa = quant_of(args);
  const Item it = locate<true>(a, lane, rep, share, mine, blockIdx.x);
  if (it.x.entry >= 0) {
    if (it.valid) many_columns<E, D, FMT>(qa, a, it, rep, tid, lds_addr_of(lds), lds_addr_of(places), gsm[0], any_bad);
  } else {
    const Item it4 = locate<false>(a, lane, rep, share, mine, ((int)blockIdx.x - it.x.base) * 4 + wave);
    if (!it4.valid) return;
    few_columns<E, D, FMT, 2>(qa, a, it4, rep, lane, lds_addr_of(lds) + wave * ValueTile<kTileDim<D>>::kBytes, gsm[wave]);
  }
}

// ---- host side
// Workgroups of four waves that the items are to fill.  Tokens alone: as many waves as are resident (32 tokens 31 us; for 496 workgroups 32, 384 36, 1000 37;
// heads of 128, where two waves fit a SIMD, 55, for 744 69).  Tiles of many columns: 512 are resident, but one a CU runs faster than two, and what
// rounding adds must not wait for a place (32 tokens behind 8192 keys 22.1, for 496 23.9, 256 24.1; four prompts of 512 22.3, for 496 34.7).  Ragged rows:
// few and many columns, and many workgroups of the first kind (512 rows beside 31 tokens 63, for 384 85, 640 69).
int target_of(const segpt_paged_params& p) {
  const int rep = p.H / p.Hkv;
  const bool wide = p.prefix_table || (!p.seq_start && (int64_t)rep * (p.T / p.B) > kMostFew);
  if (all_few(p)) return p.D == 128 ? 496 : 744;
  return wide ? 384 : p.seq_start ? 480 : 496;
}

template <typename E, int D, int FMT>
int launch(const Args& args, hipStream_t st) {
  const PagedArgs& a = args.w;
  int rc = launch_plan(a, st);
  if (rc) return rc;
  if (all_few(a.p)) hipLaunchKernelGGL((paged_quant_few_kernel<E, D, FMT>), dim3((unsigned)a.n_few), dim3(64), 0, st, args);
  else hipLaunchKernelGGL((paged_quant_any_kernel<E, D, FMT>), dim3((unsigned)(a.n_many + (a.n_few + 3) / 4)), dim3(256), 0, st, args);
  rc = (int)hipGetLastError();
  if (rc) return rc;
  return launch_merge<E, D>(a, st);
}

}  // namespace
}  // namespace segpt

extern "C" {

size_t segpt_paged_quant_workspace_bytes(const segpt_paged_params* p, const segpt_paged_quant* q) {
  using namespace segpt;
  if (check_paged_sizes(p, PagedCall::kAttend) != SEGPT_OK || !q || q->struct_bytes != sizeof(segpt_paged_quant)) return 0;
  if ((q->format != SEGPT_POOL_E4M3 && q->format != SEGPT_POOL_E2M1) || !quant_head_dim(*p)) return 0;
  PagedArgs a{};
  const size_t n = plan(*p, a, target_of(*p));
  return n > SIZE_MAX - 256 ? 0 : up256(n);
}

int segpt_paged_attn_quant(const segpt_paged_params* p, const segpt_paged_quant* q, void* stream) {
  using namespace segpt;
  int rc = check_quant(p, q, PagedCall::kAttend);
  if (rc) return rc;
  Args args{{}, q->k_scales, q->v_scales};
  if ((rc = prepare_call(p, args.w, target_of(*p)))) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool e4m3 = q->format == SEGPT_POOL_E4M3;
  if (p->dtype == SEGPT_DTYPE_BF16) {
    if (p->D == 64) return e4m3 ? launch<uint16_t, 64, SEGPT_POOL_E4M3>(args, st) : launch<uint16_t, 64, SEGPT_POOL_E2M1>(args, st);
    return e4m3 ? launch<uint16_t, 128, SEGPT_POOL_E4M3>(args, st) : launch<uint16_t, 128, SEGPT_POOL_E2M1>(args, st);
  }
  if (p->D == 32) return e4m3 ? launch<float, 32, SEGPT_POOL_E4M3>(args, st) : launch<float, 32, SEGPT_POOL_E2M1>(args, st);
  if (p->D == 64) return e4m3 ? launch<float, 64, SEGPT_POOL_E4M3>(args, st) : launch<float, 64, SEGPT_POOL_E2M1>(args, st);
  return e4m3 ? launch<float, 128, SEGPT_POOL_E4M3>(args, st) : launch<float, 128, SEGPT_POOL_E2M1>(args, st);
}

}  // extern "C"
