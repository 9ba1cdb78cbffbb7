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
#include "paged_work.hpp"

namespace segpt {
namespace {

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
  static constexpr int KS = D / 16, kCols = 32, kLogCols = 5;
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
  static constexpr int C = D / 8, kCols = 32, kLogCols = 5;
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
  const Column c = column_of<E, D>(a, it, rep, it.tile * kFew, lane, q);
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
  const Column c = column_of<E, D>(a, it, rep, it.tile * kMany + wave * 32, lane, q);
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

int target_of(const segpt_paged_params& p) {
  const int row_bytes = p.D * (p.dtype == SEGPT_DTYPE_FP32 ? 4 : 2), rep = p.H / p.Hkv;
  // 512 workgroups are resident, two a CU.  The shares' length is found in three steps and may leave a few more than asked for, and one that has to wait
  // for a place is a round of its own: 480 are asked for, 496 where all are single waves (us, asked for 512 and now; 18 / 6 heads of 64, up to 8192 keys:
  // 512 rows beside 31 tokens 78, 73; beside 63 132, 111; beside 15 66, 66; 128 rows beside 15 40.7, 45.2; eight fp32 tokens 19.9, 17.8; 128 of bf16
  // 102, 103).  Where the host sees that the work is of many columns (a prefix, prompts of equal length) three on two CUs: longer shares leave a
  // quarter less to be joined, which is more than the idle places would have done (512 and 384: a prompt of 1024 tokens 33.6, 31.0, of 2048 46.2, 42.8,
  // of 8192 237, 237, four of 512 34.8, 21.3; 32 tokens behind 8192 keys 23.3, 21.8; 128 behind 16001, 16 / 4 heads of 128, 57 .. 60 either way).  fp32 rows
  // of 512 bytes: one a CU, all of them (256 and 224: 32 tokens of 16 / 4 heads 48.5, 53.6; 100 122, 134; of 4 / 2 heads 80, 66).
  const bool wide = p.prefix_table || (!p.seq_start && (int64_t)rep * (p.T / p.B) > kFew);
  return row_bytes > 256 ? 256 : wide ? 384 : p.seq_start ? 480 : 496;
}

template <typename E, int D>
int launch(const PagedArgs& a, hipStream_t st) {
  const segpt_paged_params& p = a.p;
  int rc = launch_plan(a, st);
  if (rc) return rc;
  if (all_few(p)) hipLaunchKernelGGL((paged_few_kernel<E, D>), dim3((unsigned)a.n_few), dim3(64), 0, st, a);
  else hipLaunchKernelGGL((paged_any_kernel<E, D>), dim3((unsigned)(a.n_many + (a.n_few + 3) / 4)), dim3(256), 0, st, a);
  rc = (int)hipGetLastError();
  if (rc) return rc;
  return launch_merge<E, D>(a, st);
}

}  // namespace
}  // namespace segpt

extern "C" {

size_t segpt_paged_workspace_bytes(const segpt_paged_params* p) {
  using namespace segpt;
  if (check_paged_sizes(p, PagedCall::kAttend) != SEGPT_OK) return 0;
  PagedArgs a{};
  const size_t n = plan(*p, a, target_of(*p));
  return n > SIZE_MAX - 256 ? 0 : up256(n);
}

int segpt_paged_attn(const segpt_paged_params* p, void* stream) {
  using namespace segpt;
  const int rc = check_paged(p, PagedCall::kAttend);
  if (rc) return rc;
  PagedArgs a{};
  const int bad = prepare_call(p, a, target_of(*p));
  if (bad) return bad;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p->dtype == SEGPT_DTYPE_BF16) return p->D == 64 ? launch<uint16_t, 64>(a, st) : launch<uint16_t, 128>(a, st);
  return p->D == 32 ? launch<float, 32>(a, st) : p->D == 64 ? launch<float, 64>(a, st) : launch<float, 128>(a, st);
}

}  // extern "C"
