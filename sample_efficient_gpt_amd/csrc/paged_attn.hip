// Attention over a paged key/value cache, forward only: ragged rows of B sequences, each against the pages its table names, and, if the
// batch shares one, against the pages of a common prefix.
//
//   y_i = sum_j exp(s_ij - lse_i) v'_j      s_ij = qhat_i . k'_j      qhat = sm_scale rot(q) rsqrt(mean q^2 + eps) g_q g_k
//
// over the prefix's keys and the sequence's keys j <= kv_len - n + i.  The pool's rows are already rotated and normalised, so that what is
// left per key is a product on either side of the softmax.
//
// Work.  The heads of a kv group and the rows of a sequence are the columns n = i * (H / Hkv) + head of one product, in tiles of 32 columns a
// wave.  An ENTRY is a set of columns that read the same pages: a sequence, or the shared prefix with the rows of the whole batch.  An
// item of work is (entry, tile, share of its keys, kv head).  Lengths live on the device, so the device deals out the work: the length of
// a share follows from the sum over all entries such that the items fill the card once, and every workgroup finds its own item in
// the running sum of the entries' items (one load and a few register moves for up to 64 sequences).  A tile with one share writes y; others
// leave (reference m, sum l, products O) in fp32, which paged_merge_kernel joins.
//
// Scores are transposed as in the other forward kernels: lane = query column, S^T = K' . Qhat^T, and the probabilities are already the
// B operand of O^T = V'^T . P^T.
#include <algorithm>

#include "mfma_common.hpp"
#include "paged_common.hpp"

namespace segpt {
namespace {

struct PagedArgs {
  segpt_paged_params p;
  int32_t entries, shared;        // shared: 1 if entry 0 is the prefix
  int32_t rows_each, log_page, capacity;
  int32_t target;                 // items that fill the card once
  int32_t min_share;              // shortest share, in blocks of 32 keys
  int32_t n_items;                // workgroups: items there may be
  int32_t n_slots;                // partial results there is room for
  float* part;                    // [n_slots][tile columns][D]
  float2* stat;                   // [n_slots][tile columns]
};

constexpr int kBlock = 32;          // keys of a score tile
constexpr float kLazy = 8.f;        // the reference is raised where a score exceeds it by 2^8: probabilities stay below 2^8
constexpr int kTablePages = 512;    // page numbers held in LDS: a longer share takes its keys in windows

// ---- the plan, computed by every wave for itself
struct Entry {
  int first, n, len;   // rows, keys
  int tiles, blocks;
  bool broken;         // a length no sequence can have: every row of the entry is NaN
};
__device__ __forceinline__ Entry entry_at(const PagedArgs& a, int e, int rep, int tile_cols) {
  const segpt_paged_params& p = a.p;
  Entry x{0, 0, 0, 0, 0, false};
  if (e >= a.entries) return x;
  if (a.shared && e == 0) {
    int f, n;
    sequence_rows(p, a.rows_each, 0, &x.first, &n);
    sequence_rows(p, a.rows_each, p.B - 1, &f, &n);
    x.n = max(f + n - x.first, 0);
    x.len = p.prefix_len;
  } else {
    sequence_rows(p, a.rows_each, e - a.shared, &x.first, &x.n);
    const int len = p.kv_len[e - a.shared];
    x.broken = len < 0 || len > a.capacity;
    x.len = min(max(len, 0), a.capacity);
  }
  x.tiles = (x.n * rep + tile_cols - 1) / tile_cols;
  x.blocks = (x.len + kBlock - 1) / kBlock;
  return x;
}
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
// blocks of a share.  The sum is a float: it may round, but to the same value in every wave of both kernels.
__device__ __forceinline__ int share_blocks(const PagedArgs& a, int lane, int rep, int tile_cols, Entry* mine) {
  float work = 0.f;
  *mine = entry_at(a, lane, rep, tile_cols);
  work = (float)mine->tiles * (float)mine->blocks;
  for (int e = 64; e < a.entries; e += 64) {
    const Entry x = entry_at(a, e + lane, rep, tile_cols);
    work += (float)x.tiles * (float)x.blocks;
  }
  work = lane_value(lane_prefix_sum(work), 63) * (float)a.p.Hkv;
  return max((int)fminf(ceilf(work / (float)a.target), 1e9f), a.min_share);
}
// an entry as the whole wave sees it
struct Found {
  int entry;          // -1: none
  int first, n, len, blocks;
  int shares, base;   // shares of its keys; number of its first item
  int slot;           // of its first partial result (entries whose tiles leave any)
  bool broken;
};
// the first entry, from lane order on, for which hit(entry, number of its first item, its items) holds
template <typename Hit>
__device__ __forceinline__ Found find_entry(const PagedArgs& a, int lane, int rep, int tile_cols, int share, const Entry& mine, int from, Hit hit) {
  int base = 0, slot = 0;
  for (int e0 = 0; e0 < a.entries; e0 += 64) {
    const Entry x = e0 == 0 ? mine : entry_at(a, e0 + lane, rep, tile_cols);
    const int shares = (x.blocks + share - 1) / share, items = x.tiles * shares * a.p.Hkv;
    const int upto = base + lane_prefix_sum(items);
    const int slots = a.shared || shares > 1 ? items : 0, slots_upto = slot + lane_prefix_sum(slots);
    const uint64_t hits = __builtin_amdgcn_ballot_w64(e0 + lane >= from && e0 + lane < a.entries && hit(x, upto - items, items));
    if (hits) {
      const int l = __builtin_ctzll(hits);
      return Found{e0 + l, lane_value(x.first, l), lane_value(x.n, l), lane_value(x.len, l), lane_value(x.blocks, l), lane_value(shares, l),
                   lane_value(upto - items, l), lane_value(slots_upto - slots, l), lane_value((int)x.broken, l) != 0};
    }
    base = lane_value(upto, 63);
    slot = lane_value(slots_upto, 63);
  }
  return Found{-1, 0, 0, 0, 0, 0, 0, 0, false};
}
// shares are as even as whole blocks allow
__device__ __forceinline__ int blocks_per_share(const Found& x) { return (x.blocks + x.shares - 1) / x.shares; }

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

// NW waves share the keys of a tile; each owns 32 columns.  NW == 1: a wave of its own, nothing to wait for but its own loads.
template <typename E, int D, int NW>
struct Shape {
  static constexpr int kBK = NW == 4 && D * sizeof(E) <= 128 ? 64 : 32;  // keys per staged tile
  static constexpr int kTileBytes = kBK * D * (int)sizeof(E), kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = kStageBytes >= 32768 ? 2 : 3;
  static constexpr int kPasses = kTileBytes / 1024 / NW;  // loads of a wave per tensor and tile
  static constexpr int kCols = 32 * NW;
  static constexpr int kOcc = D * sizeof(E) <= 128 ? 3 : D * sizeof(E) <= 256 ? 2 : 1;  // waves per SIMD
};

// query columns in the B operand's layout, scaled by everything that does not depend on the key (gsm: g_q g_k sm_scale log2 e); D / 2 values
// a lane.  bf16: element 16 ks + 8 hh + t; fp32: chunk 2 c + hh of four.
template <typename E, int D>
struct Query;
template <int D>
struct Query<uint16_t, D> {
  bf16x8 reg[D / 16];
  __device__ __forceinline__ void load(const segpt_paged_params& p, const uint16_t* row, int64_t angle, bool live, int hh, const float* gsm) {
    constexpr int KS = D / 16;
    u32x4 raw[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) raw[ks] = *reinterpret_cast<const u32x4*>(row + 16 * ks + 8 * hh);
    float x[KS][8];
    unpack_b_layout<KS>(raw, x);
    if (p.rope_cos) rope_b_layout<KS>(x, p.rope_cos + angle, p.rope_sin + angle, hh);
    float ss = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int t = 0; t < 8; ++t) ss += x[ks][t] * x[ks][t];
    ss = half_sum(ss);
    const float alpha = !live ? 0.f : (p.flags & SEGPT_FLAG_NO_NORM) ? 1.f : __builtin_amdgcn_rsqf(ss * (1.0f / D) + p.eps);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* g = gsm + 16 * ks + 8 * hh + 2 * i;
        w[i] = live ? pack_bf16x2(x[ks][2 * i] * alpha * g[0], x[ks][2 * i + 1] * alpha * g[1]) : 0u;
      }
      reg[ks] = as_bf16x8(w);
    }
  }
};
template <int D>
struct Query<float, D> {
  float reg[D / 8][4];
  __device__ __forceinline__ void load(const segpt_paged_params& p, const float* row, int64_t angle, bool live, int hh, const float* gsm) {
    constexpr int C = D / 8;
#pragma unroll
    for (int c = 0; c < C; ++c) load16(row + 8 * c + 4 * hh, reg[c]);
    if (p.rope_cos) {
#pragma unroll
      for (int c = 0; c < C / 2; ++c) {
        float cs[4], sn[4];
        load16(p.rope_cos + angle + 8 * c + 4 * hh, cs);
        load16(p.rope_sin + angle + 8 * c + 4 * hh, sn);
#pragma unroll
        for (int t = 0; t < 4; ++t) rope_pair(reg[c][t], reg[c + C / 2][t], cs[t], sn[t]);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) ss += reg[c][t] * reg[c][t];
    ss = half_sum(ss);
    const float alpha = (p.flags & SEGPT_FLAG_NO_NORM) ? 1.f : 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) reg[c][t] = live ? reg[c][t] * alpha * gsm[8 * c + 4 * hh + t] : 0.f;
  }
};

__device__ __forceinline__ float lds_read_f(uint32_t addr) { return *(const __attribute__((address_space(3))) float*)addr; }
__device__ __forceinline__ uint16_t lds_read_h(uint32_t addr) { return *(const __attribute__((address_space(3))) uint16_t*)addr; }

template <typename E, int D>
__device__ __forceinline__ float gate_factor(const segpt_paged_params& p, int t, int h) {
  const E z = row_of<E>(p.gate, t, h)[0];
  float x;
  if constexpr (sizeof(E) == 2) x = bf16_to_f32(z); else x = z;
  return p.gate_scale / (1.0f + __expf(-x));
}

// Workgroup = NW waves = one item.  LDS holds the page numbers of the item's share and a ring of stages (K' tile, V' tile); tile jt lives
// in stage jt % kStages.  Per tile: wait for its loads, barrier (also: everyone has left the tile before), request tile jt + kStages - 1
// over the one before, compute.
template <typename E, int D, int NW>
__global__ __launch_bounds__(64 * NW, (Shape<E, D, NW>::kOcc)) void paged_attn_kernel(PagedArgs a) {
  using S = Shape<E, D, NW>;
  using Z = Tile<E, D>;
  constexpr bool BF16 = sizeof(E) == 2;
  constexpr int MB = D / 32, BK = S::kBK, NS = S::kStages, PASSES = S::kPasses;
  const segpt_paged_params& p = a.p;
  __shared__ __attribute__((aligned(1024))) char lds[NS * S::kStageBytes];
  __shared__ __attribute__((aligned(16))) float gsm[D];
  __shared__ int table[kTablePages + 2];
  __shared__ int any_bad[NW];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, hh = lane >> 5;
  const int rep = p.H / p.Hkv;
  auto sync = [&] {
    if constexpr (NW == 1) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): reads of a tile have returned before it is requested over
    } else {
      __syncthreads();
    }
  };

  if (p.flags & SEGPT_FLAG_ZERO_REST) {  // rows in no sequence: before the first one and behind the last
    int head, f, n;
    sequence_rows(p, a.rows_each, 0, &head, &n);
    sequence_rows(p, a.rows_each, p.B - 1, &f, &n);
    const int tail = max(f + n, head);
    for (int i = blockIdx.x; i < head + p.T - tail; i += gridDim.x) {
      const int t = i < head ? i : i - head + tail;
      for (int x = tid; x < p.H * D; x += 64 * NW) row_of<E>(p.o, t, x / D)[x % D] = 0;
    }
  }

  Entry mine;
  const int share = share_blocks(a, lane, rep, S::kCols, &mine);
  const int item = blockIdx.x;
  const Found x = find_entry(a, lane, rep, S::kCols, share, mine, 0, [&](const Entry&, int base, int items) { return item >= base && item < base + items; });
  if (x.entry < 0) return;
  const int cols = x.n * rep, n_tiles = (cols + S::kCols - 1) / S::kCols;
  const int local = item - x.base, g = local % p.Hkv, part = local / p.Hkv % x.shares;
  const int tile = n_tiles - 1 - local / p.Hkv / x.shares;  // the last tiles see the most keys: they start first
  const bool prefix = a.shared && x.entry == 0, direct = !a.shared && x.shares == 1;
  const int slot = x.slot + (tile * x.shares + part) * p.Hkv + g;
  if (tile < 0 || (!direct && slot >= a.n_slots)) return;
  const int per = blocks_per_share(x) * kBlock;

  // this item's keys: k0 .. k1 - 1, the last ones cut off where no row of the tile sees them
  const int past = x.len - x.n;  // row i of a sequence sees its keys up to past + i; the prefix's all rows see, but for those that stand in it
  const int last_col = min(cols, (tile + 1) * S::kCols) - 1;
  const int k0 = part * per, sees = prefix ? x.len : min(x.len, past + last_col / rep + 1), k1 = min(sees, k0 + per);
  const int nk = max(k1 - k0, 0);

  // ---- page numbers of a window of the keys into LDS; one that is not in the pool is replaced by page 0 and remembered
  const int window = kTablePages << a.log_page;
  const int* const ids = prefix ? p.prefix_table : p.block_table + (int64_t)(x.entry - a.shared) * p.table_stride;
  bool bad = x.broken;
  int w0 = k0, wn = min(nk, window);  // first key and keys of the window
  auto stage_table = [&] {
    const int p0 = w0 >> a.log_page, pages = wn ? ((w0 + wn - 1) >> a.log_page) - p0 + 1 : 0;
    bool mine_bad = false;
    for (int i = tid; i < pages; i += 64 * NW) {
      int id = ids[p0 + i];
      if ((uint32_t)id >= (uint32_t)p.n_pages) { id = 0; mine_bad = true; }
      table[i] = id;
    }
    const bool wave_bad = __builtin_amdgcn_ballot_w64(mine_bad) != 0;
    if (lane == 0) any_bad[wave] = wave_bad;
  };
  stage_table();
  for (int d = tid; d < D; d += 64 * NW) {
    float v = (p.gq_numel == 1 ? p.g_q[0] : p.g_q[d]) * p.sm_scale * kLog2e;
    if (p.gk_numel) v *= p.gk_numel == 1 ? p.g_k[0] : p.g_k[d];
    gsm[d] = v;
  }
  sync();

  // ---- tile requests.  A load covers kRowsPerLoad rows, at most 8, of one page: its address is a scalar base and a lane offset
  const uint32_t lds0 = lds_addr_of(lds);
  const int lrow = lane / Z::kChunks;
  const char* const kbase = page_row<E>(p.k_pages, 0, g, 0);
  const char* const vbase = page_row<E>(p.v_pages, 0, g, 0);
  const int64_t kpage = p.k_pages.stride_b * (int)sizeof(E), vpage = p.v_pages.stride_b * (int)sizeof(E);
  const uint32_t kstep = (uint32_t)p.k_pages.stride_s * (int)sizeof(E), vstep = (uint32_t)p.v_pages.stride_s * (int)sizeof(E);
  auto first_row = [&](int jt, int ps) {  // of load ps, from w0 on; past the last key: the last rows once more
    return min(jt * BK + (ps * NW + wave) * Z::kRowsPerLoad, (wn - 1) & ~(Z::kRowsPerLoad - 1));
  };
  auto page_of = [&](int jt) {  // lane ps: the page number of load ps
    return table[((w0 + first_row(jt, min(lane, PASSES - 1))) >> a.log_page) - (w0 >> a.log_page)];
  };
  auto issue = [&](int jt, int pages) {
    const uint32_t dst = lds0 + (uint32_t)(jt % NS) * S::kStageBytes + wave * 1024;
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int r0 = first_row(jt, ps), slot_row = (w0 + r0) & ((1 << a.log_page) - 1);
      const int64_t page = __builtin_amdgcn_readlane(pages, ps);
      const int r = min(lrow, wn - 1 - r0);
      const uint32_t col = (uint32_t)((lane % Z::kChunks) ^ Z::f((ps * NW + wave) * Z::kRowsPerLoad + lrow)) << 4;
      gload_lds16_so(kbase + page * kpage + (int64_t)slot_row * kstep, (uint32_t)r * kstep + col, dst + ps * NW * 1024);
      gload_lds16_so(vbase + page * vpage + (int64_t)slot_row * vstep, (uint32_t)r * vstep + col, dst + S::kTileBytes + ps * NW * 1024);
    }
  };
  auto start_window = [&] {
#pragma unroll
    for (int w = 0; w < NW; ++w) bad |= any_bad[w] != 0;
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
      if (t * BK < wn) issue(t, page_of(t));
  };
  start_window();

  // ---- this lane's column
  const int col = tile * S::kCols + wave * 32 + ln;
  const bool live = col < cols;
  const int i = (live ? col : tile * S::kCols) / rep, t_row = x.first + i, h = g * rep + (live ? col : tile * S::kCols) % rep;
  Query<E, D> q;
  int own = past + i;  // position among the sequence's own keys: negative where it stands in the prefix
  {
    if (prefix) {  // the row's own sequence says where it stands
      int b = 0, f = 0, n = 0;
      if (p.seq_start) {
        for (int lo = 0, hi = p.B - 1; lo <= hi;) {  // last sequence that starts at or before the row
          const int m = (lo + hi) >> 1;
          if (p.seq_start[m] <= t_row) { b = m; lo = m + 1; } else hi = m - 1;
        }
      } else {
        b = t_row / a.rows_each;
      }
      sequence_rows(p, a.rows_each, b, &f, &n);
      own = (int)min((int64_t)p.kv_len[b] - n + (t_row - f), (int64_t)a.capacity - 1);
    }
    const int64_t pos = max((int64_t)p.prefix_len + own, (int64_t)0);
    q.load(p, row_of<E>(p.q, t_row, h), (p.rope_pos0 + pos) * (D / 2), live, hh, gsm);
  }
  // keys from k0 on that the lane's row sees, and what the whole wave sees; a wave without columns computes nothing
  const int lim = min((prefix ? p.prefix_len : 0) + own - k0, nk - 1);
  const int wave_col = tile * S::kCols + wave * 32;
  const bool works = wave_col < cols;
  const bool cut = prefix && __builtin_amdgcn_ballot_w64(lim < nk - 1) != 0;  // rows that stand in the prefix
  const int all_see = !works || cut ? -1 : prefix ? nk - 1 : min(past + wave_col / rep - k0, nk - 1);
  const int any_sees = !works ? -1 : prefix ? nk - 1 : min(past + min(wave_col + 31, cols - 1) / rep - k0, nk - 1);

  f32x16 oacc[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) oacc[mb] = splat16(0.f);
  float m_ref = -INFINITY, l_run[2] = {0.f, 0.f};

  auto block = [&](uint32_t stage, int kb, int jb) {  // keys jb .. jb + 31 from k0 on, rows 32 kb .. of the tile
    const uint32_t kt = stage + kb * 32 * Z::kRB, vt = stage + S::kTileBytes + kb * 32 * Z::kRB;
    f32x16 s = splat16(0.f);
    if constexpr (BF16) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) s = mfma32(swz_frag_rm<D>(kt + swz_off_rm<D>(lane), 0, ks), q.reg[ks], s);
    } else {
      const uint32_t row = kt + ln * Z::kRB;
      const int fx = Z::f(ln);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const f32x4 k4 = lds_read_f4(row + (((2 * c + hh) ^ fx) << 4));
#pragma unroll
        for (int t = 0; t < 4; ++t) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[t], q.reg[c][t], s, 0, 0, 0);
      }
    }
    const bool masked = jb + 31 > all_see;  // register r holds key jb + 4 hh + c_r, c_r = 8 (r / 4) + r % 4
    if (masked) {
      const int t = lim - jb - 4 * hh;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) > t) s[r] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = half_max(mx);
    const bool need = mx > m_ref + kLazy;
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
      const float m_new = need ? mx : m_ref, corr = need ? fast_exp2(m_ref - m_new) : 1.f;
      m_ref = m_new;
      l_run[0] *= corr;
      l_run[1] *= corr;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[mb][r] *= corr;
    }
    const float mu = m_ref == -INFINITY ? 0.f : m_ref;  // nothing seen yet: keep exp2 away from inf - inf
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = fast_exp2(s[r] - mu);

    if constexpr (BF16) {
      const bf16x8 pb[2] = {pack_c_half_sum(s, 0, l_run), pack_c_half_sum(s, 1, l_run)};
      bf16x8 vT[MB][2];
      bool odd = false;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2) vT[mb][s2] = swz_frag_tr<D>(vt + swz_off_tr<D>(lane), mb, s2);
      if (masked) {  // a value that is not finite must not reach rows that do not see its key through 0 * inf
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            u32x4 w = __builtin_bit_cast(u32x4, vT[mb][s2]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool lo = (w[e] & 0x7f80u) == 0x7f80u, hi = (w[e] & 0x7f800000u) == 0x7f800000u;
              odd |= lo | hi;
              w[e] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
            }
            vT[mb][s2] = as_bf16x8(w);
          }
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) oacc[mb] = mfma32(vT[mb][s2], pb[s2], oacc[mb]);
      if (masked && __builtin_amdgcn_ballot_w64(odd) != 0) {  // rare: those values once more, key by key, for the rows that see them
        for (int key = 0; key < 32; ++key) {
          const bool visible = key <= lim - jb;
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int d = 32 * mb + 8 * (r >> 2) + 4 * hh + (r & 3);
              const float v = bf16_to_f32(lds_read_h(vt + key * Z::kRB + (((d >> 3) ^ Z::f(key)) << 4) + 2 * (d & 7)));
              if (visible && !(fabsf(v) < INFINITY)) oacc[mb][r] += v;  // its probability is positive: v, or NaN where signs meet
            }
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) l_run[r & 1] += s[r];
      bool odd = false;
      // step r contracts key c_r (lower half of the wave) and c_r + 4 (upper half): register r of the probabilities as it is
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = 8 * (r >> 2) + (r & 3) + 4 * hh;
        const uint32_t at = vt + key * Z::kRB;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          float v = lds_read_f(at + (((8 * mb + (ln >> 2)) ^ Z::f(key)) << 4) + 4 * (ln & 3));
          if (masked) {  // as above
            const bool no_number = !(fabsf(v) < INFINITY);
            odd |= no_number;
            if (no_number) v = 0.f;
          }
          oacc[mb] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[r], oacc[mb], 0, 0, 0);
        }
      }
      if (masked && __builtin_amdgcn_ballot_w64(odd) != 0) {
        for (int key = 0; key < 32; ++key) {
          const bool visible = key <= lim - jb;
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const f32x4 v = lds_read_f4(vt + key * Z::kRB + (((8 * mb + 2 * c + hh) ^ Z::f(key)) << 4));
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (visible && !(fabsf(v[e]) < INFINITY)) oacc[mb][4 * c + e] += v[e];
            }
        }
      }
    }
  };

  while (true) {
    wait_vmcnt<0>();  // the loads below are counted: nothing of the start may be in flight with them
    const int n_kt = (wn + BK - 1) / BK;
    int next_pages = n_kt ? page_of(min(NS - 1, n_kt - 1)) : 0;
    for (int jt = 0; jt < n_kt; ++jt) {
      if (n_kt - 1 - jt >= NS - 2) wait_vmcnt<(NS - 2) * 2 * PASSES>(); else wait_vmcnt<0>();
      sync();
      if (jt + NS - 1 < n_kt) {
        issue(jt + NS - 1, next_pages);
        next_pages = page_of(min(jt + NS, n_kt - 1));
      }
      const uint32_t stage = lds0 + (uint32_t)(jt % NS) * S::kStageBytes;
      const int jb = w0 - k0 + jt * BK;
#pragma unroll
      for (int kb = 0; kb < BK / 32; ++kb)
        if (jb + 32 * kb <= any_sees) block(stage, kb, jb + 32 * kb);
    }
    w0 += window;
    if (w0 >= k1) break;
    wn = min(k1 - w0, window);
    sync();  // everyone is done with the page numbers and the stages
    stage_table();
    sync();
    start_window();
  }

  // ---- result: row = lane, columns 32 mb + 8 (r / 4) + 4 hh + r % 4
  float l = half_sum(l_run[0] + l_run[1]);
  if (bad) { l = __builtin_nanf(""); m_ref = 0.f; }
  if (!live) return;
  if (!direct) {
    const int64_t at = (int64_t)slot * S::kCols + wave * 32 + ln;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<float4*>(a.part + at * D + 32 * mb + 8 * c + 4 * hh) =
            make_float4(oacc[mb][4 * c], oacc[mb][4 * c + 1], oacc[mb][4 * c + 2], oacc[mb][4 * c + 3]);
    if (hh == 0) a.stat[at] = make_float2(m_ref, l);
    return;
  }
  float f = l == 0.f ? 0.f : 1.0f / l;
  if (p.lse && hh == 0) p.lse[(int64_t)t_row * p.H + h] = l == 0.f ? -INFINITY : (m_ref + __log2f(l)) * kLn2;
  if (p.gate.ptr) f *= gate_factor<E, D>(p, t_row, h);
  E* out = row_of<E>(p.o, t_row, h);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float y[4] = {oacc[mb][4 * c] * f, oacc[mb][4 * c + 1] * f, oacc[mb][4 * c + 2] * f, oacc[mb][4 * c + 3] * f};
      E* at = out + 32 * mb + 8 * c + 4 * hh;
      if constexpr (BF16) *reinterpret_cast<u32x2*>(at) = u32x2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
      else store16(at, y);
    }
}

// Joins the shares of a row: its sequence's own and the prefix's.  WAVES waves a row (one: as many rows as waves), D / 4 lanes side by side,
// the rest over the shares.  Fixed order: deterministic.
constexpr int kMergeThreads = 256;
template <typename E, int D, int WAVES>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_kernel(PagedArgs a, int tile_cols) {
  const segpt_paged_params& p = a.p;
  constexpr int LPR = D / 4, G = 64 / LPR, GROUPS = G * WAVES;
  __shared__ float4 sums[WAVES > 1 ? kMergeThreads : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rep = p.H / p.Hkv;
  const int64_t row = WAVES > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (kMergeThreads / 64) + wave;
  if (row >= (int64_t)p.T * p.H) return;
  const int t = (int)(row / p.H), h = (int)(row - (int64_t)t * p.H), g = h / rep;
  Entry mine;
  const int share = share_blocks(a, lane, rep, tile_cols, &mine);
  const Found own = find_entry(a, lane, rep, tile_cols, share, mine, a.shared, [&](const Entry& x, int, int) { return t >= x.first && t < x.first + x.n; });
  if (own.entry < 0) return;  // in no sequence
  if (!a.shared && own.shares == 1) return;  // written by its only share
  Found pre{-1, 0, 0, 0, 0, 0, 0, 0, false};
  if (a.shared) pre = find_entry(a, lane, rep, tile_cols, share, mine, 0, [&](const Entry&, int, int) { return true; });
  const int n = pre.shares + own.shares;
  auto slot = [&](int s) {  // of share s: the prefix's first
    const bool in_prefix = s < pre.shares;
    const Found& x = in_prefix ? pre : own;
    const int col = (t - x.first) * rep + h - g * rep, tile = col / tile_cols;
    const int64_t at = x.slot + ((int64_t)tile * x.shares + (in_prefix ? s : s - pre.shares)) * p.Hkv + g;
    return at < a.n_slots ? at * tile_cols + (col - tile * tile_cols) : (int64_t)-1;
  };
  auto stat_of = [&](int64_t at) { return at < 0 ? make_float2(0.f, __builtin_nanf("")) : a.stat[at]; };

  float m = -INFINITY;
  for (int s = lane; s < n; s += 64) {
    const float2 x = stat_of(slot(s));
    m = fmaxf(m, x.x);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float mu = m == -INFINITY ? 0.f : m;
  const int gi = lane / LPR + (WAVES > 1 ? wave * G : 0), c = lane % LPR;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int s = gi; s < n; s += GROUPS) {
    const int64_t at = slot(s);
    const float2 x = stat_of(at);
    if (x.y == 0.f) continue;  // saw no key
    const float w = fast_exp2(x.x - mu);
    l += w * x.y;
    if (at < 0) continue;
    const float4 o = *reinterpret_cast<const float4*>(a.part + at * D + 4 * c);
    y.x += w * o.x; y.y += w * o.y; y.z += w * o.z; y.w += w * o.w;
  }
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1) {
    l += __shfl_xor(l, o, 64);
    y.x += __shfl_xor(y.x, o, 64); y.y += __shfl_xor(y.y, o, 64); y.z += __shfl_xor(y.z, o, 64); y.w += __shfl_xor(y.w, o, 64);
  }
  if constexpr (WAVES > 1) {
    __shared__ float ls[WAVES];
    sums[tid] = y;
    if (lane == 0) ls[wave] = l;
    __syncthreads();
    if (wave) return;
    l = 0.f;
    y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float4 o = sums[w * 64 + lane];
      l += ls[w];
      y.x += o.x; y.y += o.y; y.z += o.z; y.w += o.w;
    }
  }
  if (own.broken) l = __builtin_nanf("");
  if (lane >= LPR) return;
  float f = l == 0.f ? 0.f : 1.0f / l;
  if (p.lse && c == 0) p.lse[(int64_t)t * p.H + h] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
  if (p.gate.ptr) f *= gate_factor<E, D>(p, t, h);
  E* out = row_of<E>(p.o, t, h) + 4 * c;
  const float v[4] = {y.x * f, y.y * f, y.z * f, y.w * f};
  if constexpr (sizeof(E) == 2) *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
  else store16(out, v);
}

// ---- host side
int waves_of(const segpt_paged_params& p) {
  if (p.dtype == SEGPT_DTYPE_FP32 && p.D == 128) return 4;
  return p.prefix_table || (int64_t)p.H / p.Hkv * p.T > 32ll * p.B ? 4 : 1;
}

// fills the plan; returns the scratch bytes of the partials
size_t plan(const segpt_paged_params& p, PagedArgs& a) {
  const int nw = waves_of(p), cols = 32 * nw, elem = p.dtype == SEGPT_DTYPE_FP32 ? 4 : 2;
  a.shared = p.prefix_table ? 1 : 0;
  a.entries = p.B + a.shared;
  a.rows_each = p.seq_start ? 0 : p.T / p.B;
  a.log_page = __builtin_ctz((unsigned)p.page_size);
  a.capacity = paged_capacity(p);
  const int row_bytes = p.D * elem;
  a.target = nw == 4 ? 256 * (row_bytes <= 128 ? 3 : row_bytes <= 256 ? 2 : 1) : 256 * (row_bytes <= 128 ? 6 : row_bytes <= 256 ? 3 : 2);
  a.min_share = nw == 4 ? 4 : 2;
  // every entry's tiles: whole ones of the rows there are, and one begun; every tile's shares: its part of the target, and one begun
  const int64_t all_cols = (int64_t)p.T * (p.H / p.Hkv);
  int64_t tiles = all_cols / cols + p.B;
  if (!p.seq_start) tiles = (all_cols / p.B + cols - 1) / cols * p.B;
  if (a.shared) tiles += (all_cols + cols - 1) / cols;
  const int64_t items = tiles * p.Hkv + a.target + 64;  // the sum that gives the length of a share is rounded
  a.n_items = (int32_t)std::min<int64_t>(items, INT32_MAX);
  // a tile that leaves partial results has two shares or more, i.e. at most twice its part of the target; beside a prefix all leave them
  a.n_slots = a.shared ? a.n_items : (int32_t)std::min<int64_t>(items, 2 * a.target + 64);
  return items > INT32_MAX ? SIZE_MAX : (size_t)a.n_slots * cols * (p.D + 2) * sizeof(float);
}

template <typename E, int D, int NW>
int launch(const PagedArgs& a, hipStream_t st) {
  const segpt_paged_params& p = a.p;
  hipLaunchKernelGGL((paged_attn_kernel<E, D, NW>), dim3((unsigned)a.n_items), dim3(64 * NW), 0, st, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  const int64_t rows = (int64_t)p.T * p.H;
  if (rows <= 4096) hipLaunchKernelGGL((paged_merge_kernel<E, D, 4>), dim3((unsigned)rows), dim3(kMergeThreads), 0, st, a, 32 * NW);
  else hipLaunchKernelGGL((paged_merge_kernel<E, D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(kMergeThreads), 0, st, a, 32 * NW);
  return (int)hipGetLastError();
}
template <typename E, int D>
int launch_waves(const PagedArgs& a, int nw, hipStream_t st) {
  if constexpr (D * sizeof(E) > 256) return launch<E, D, 4>(a, st);
  else return nw == 4 ? launch<E, D, 4>(a, st) : launch<E, D, 1>(a, st);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace
}  // namespace segpt

extern "C" {

size_t segpt_paged_workspace_bytes(const segpt_paged_params* p) {
  using namespace segpt;
  if (!p || p->struct_bytes != sizeof(segpt_paged_params) || (p->dtype != SEGPT_DTYPE_BF16 && p->dtype != SEGPT_DTYPE_FP32)) return 0;
  if (p->T <= 0 || p->B <= 0 || p->H <= 0 || p->Hkv <= 0 || p->H % p->Hkv || p->D <= 0 || p->page_size < 8 || p->table_width <= 0 || p->prefix_len < 0) return 0;
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
  a.part = reinterpret_cast<float*>(p->workspace);
  a.stat = reinterpret_cast<float2*>(a.part + (size_t)a.n_slots * 32 * waves_of(*p) * p->D);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int nw = waves_of(*p);
  if (p->dtype == SEGPT_DTYPE_BF16) return p->D == 64 ? launch_waves<uint16_t, 64>(a, nw, st) : launch_waves<uint16_t, 128>(a, nw, st);
  return p->D == 32 ? launch_waves<float, 32>(a, nw, st) : p->D == 64 ? launch_waves<float, 64>(a, nw, st) : launch_waves<float, 128>(a, nw, st);
}

}  // extern "C"
