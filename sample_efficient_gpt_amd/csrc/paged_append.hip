// Rows of keys and values into the pages of their sequences: the keys rotated and normalised, the values mixed with the first
// layer's, each rounded once.  The cache then holds what the attention multiplies, and a key is prepared once instead of once a token
// generated after it.
//
//   k'_p = rot_p(k) * rsqrt(mean k^2 + eps)        v'_p = c1 v + c2 v_first        p = kv_len[b] - n + i
//
// The rotation keeps a pair's sum of squares, so that the normaliser may be taken before or after it; here it is taken of
// the rotated row, as the other kernels do.
//
// A row is D * sizeof(E) / 32 lanes: a lane holds 16 bytes of the first half and the 16 bytes of the second half that they rotate with, so
// that no element crosses lanes.  Bound by HBM (every row read and written once) or, for the rows of a generation step, by the chain
// of loads: length and table, then the row's page.  16 prompts of 301 .. 2048 tokens, 4 kv heads of 128: 88 MB in 16.9 us (5.2 TB/s of reads and
// writes; a copy of 2 GiB reaches 4.9); 64 single tokens of 6 kv heads of 64 with the value mix 4.0 us, one token 2.5.
#include "paged_common.hpp"

namespace segpt {

namespace {

constexpr int kThreads = 256;

// Sequence of row t, for a whole wave: the number of the last sequence that starts at or before it.  64 starts are looked at a time, so
// that a batch of up to 64 sequences is one load, of up to 4096 two one after the other.
__device__ __forceinline__ int sequence_of_row(const segpt_paged_params& p, int t, int lane) {
  int lo = 0, n = p.B;
  while (true) {
    const int step = (n + 63) / 64, i = lane * step;
    const bool before = i < n && p.seq_start[lo + i] <= t;
    const int k = __popcll(__builtin_amdgcn_ballot_w64(before));
    if (k > 0) lo += (k - 1) * step;
    if (step == 1) return lo;
    n = min(step, p.B - lo);
  }
}

template <typename E, int D, bool ROPE, bool MIX>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(segpt_paged_params p, int log_page, int rows_each, int capacity) {
  constexpr int VEC = 16 / sizeof(E), LPR = D / 2 / VEC, kRowsPerWave = 64 / LPR;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t first = ((int64_t)blockIdx.x * (kThreads / 64) + wave) * kRowsPerWave, total = (int64_t)p.T * p.Hkv;
  if (first >= total) return;
  const int64_t row = min(first + lane / LPR, total - 1);
  const bool live = first + lane / LPR < total;
  const int t = (int)(row / p.Hkv), g = (int)(row - (int64_t)t * p.Hkv), c = (lane % LPR) * VEC;

  float k[2][VEC], v[2][VEC], f[2][VEC];
  auto load = [&](const segpt_rows& r, float (&x)[2][VEC]) {
    const E* at = row_of<E>(r, t, g) + c;
#pragma unroll
    for (int i = 0; i < 2; ++i) load16(at + i * (D / 2), x[i]);
  };
  load(p.k, k);
  load(p.v, v);
  if constexpr (MIX) load(p.v_first, f);

  int b, r0, n;
  if (p.seq_start) {
    b = sequence_of_row(p, (int)(first / p.Hkv), lane);
    // a later row of the wave: mostly the next sequence, but any number without rows may lie between
    int step = 1;
    for (; b + step < p.B && p.seq_start[b + step] <= t; step *= 2) b += step;
    while (step >>= 1)
      if (b + step < p.B && p.seq_start[b + step] <= t) b += step;
  } else {
    b = t / rows_each;
  }
  sequence_rows(p, rows_each, b, &r0, &n);
  const int64_t pos = (int64_t)p.kv_len[b] - n + (t - r0);
  const bool placed = live && t >= r0 && t < r0 + n && pos >= 0 && pos < capacity;
  const int at = placed ? (int)pos : 0;
  const int page = p.block_table[(int64_t)b * p.table_stride + (at >> log_page)];
  if constexpr (ROPE) {
    const int64_t angle = ((int64_t)p.rope_pos0 + at) * (D / 2) + c;  // within the tables: they cover every position of the table
    float cs[VEC], sn[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p.rope_cos + angle + i), y = *reinterpret_cast<const float4*>(p.rope_sin + angle + i);
      cs[i] = x.x; cs[i + 1] = x.y; cs[i + 2] = x.z; cs[i + 3] = x.w;
      sn[i] = y.x; sn[i + 1] = y.y; sn[i + 2] = y.z; sn[i + 3] = y.w;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) rope_pair(k[0][i], k[1][i], cs[i], sn[i]);
  }
  if (!(p.flags & SEGPT_FLAG_NO_NORM)) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss += k[0][i] * k[0][i] + k[1][i] * k[1][i];
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor(ss, o, 64);
    const float beta = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
    for (int i = 0; i < VEC; ++i) { k[0][i] *= beta; k[1][i] *= beta; }
  }
  if constexpr (MIX) {
    const float c1 = p.vr_coef[0], c2 = p.vr_coef[1];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[h][i] = fmaf(c2, f[h][i], c1 * v[h][i]);
  }
  if (!placed || (uint32_t)page >= (uint32_t)p.n_pages) return;
  const int slot = at & ((1 << log_page) - 1);
  E* kd = reinterpret_cast<E*>(page_row<E>(p.k_pages, page, g, slot)) + c;
  E* vd = reinterpret_cast<E*>(page_row<E>(p.v_pages, page, g, slot)) + c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    store16(kd + i * (D / 2), k[i]);
    store16(vd + i * (D / 2), v[i]);
  }
}

template <typename E, int D>
int launch(const segpt_paged_params& p, hipStream_t st) {
  constexpr int kRows = kThreads / 64 * (64 / (D / 2 / (16 / (int)sizeof(E))));
  const int64_t groups = ((int64_t)p.T * p.Hkv + kRows - 1) / kRows;
  if (groups > UINT32_MAX / kThreads) return SEGPT_E_SHAPE;  // a launch has fewer than 2^32 threads: rows of 128 GiB and more
  const dim3 grid((unsigned)groups);
  const int log_page = __builtin_ctz((unsigned)p.page_size), each = p.seq_start ? 0 : p.T / p.B;
  const bool mix = p.v_first.ptr != nullptr;
  if (p.rope_cos) {
    if (mix) hipLaunchKernelGGL((paged_append_kernel<E, D, true, true>), grid, dim3(kThreads), 0, st, p, log_page, each, paged_capacity(p));
    else hipLaunchKernelGGL((paged_append_kernel<E, D, true, false>), grid, dim3(kThreads), 0, st, p, log_page, each, paged_capacity(p));
  } else {
    if (mix) hipLaunchKernelGGL((paged_append_kernel<E, D, false, true>), grid, dim3(kThreads), 0, st, p, log_page, each, paged_capacity(p));
    else hipLaunchKernelGGL((paged_append_kernel<E, D, false, false>), grid, dim3(kThreads), 0, st, p, log_page, each, paged_capacity(p));
  }
  return (int)hipGetLastError();
}

int64_t elem_bytes(const segpt_paged_params& p) { return p.dtype == SEGPT_DTYPE_FP32 ? 4 : 2; }
bool aligned(const void* ptr, uintptr_t n) { return (reinterpret_cast<uintptr_t>(ptr) & (n - 1)) == 0; }

// extents sorted by stride: each stride has to step over everything below it
bool overlaps_itself(int64_t (&st)[3], int64_t (&ex)[3], int D) {
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (st[j] < st[i]) {
        const int64_t a = st[i], b = ex[i];
        st[i] = st[j]; ex[i] = ex[j];
        st[j] = a; ex[j] = b;
      }
  int64_t span = D;
  for (int i = 0; i < 3; ++i) {
    if (ex[i] <= 1) continue;
    if (st[i] < span) return true;
    span = st[i] * ex[i];
  }
  return false;
}

int check_pool(const segpt_tensor4& t, const segpt_paged_params& p, bool out) {
  if (!t.ptr) return SEGPT_E_NULL;
  if (!aligned(t.ptr, 16)) return SEGPT_E_ALIGN;
  const int64_t per16 = 16 / elem_bytes(p);
  if (t.stride_b < 0 || t.stride_h < 0 || t.stride_s < p.D) return SEGPT_E_STRIDE;
  if (t.stride_b % per16 || t.stride_h % per16 || t.stride_s % per16) return SEGPT_E_STRIDE;
  if (t.stride_s > (int64_t)(UINT32_MAX / (16 * 4))) return SEGPT_E_STRIDE;  // rows of a wave-wide load: 32-bit offsets
  int64_t st[3] = {t.stride_b, t.stride_h, t.stride_s}, ex[3] = {p.n_pages, p.Hkv, p.page_size};
  return out && overlaps_itself(st, ex, p.D) ? SEGPT_E_STRIDE : SEGPT_OK;
}

int check_rows(const segpt_rows& r, const segpt_paged_params& p, int heads, bool out) {
  if (!r.ptr) return SEGPT_E_NULL;
  if (!aligned(r.ptr, 16)) return SEGPT_E_ALIGN;
  const int64_t per16 = 16 / elem_bytes(p);
  if (r.stride_t < 0 || r.stride_h < 0 || (p.T > 1 && r.stride_t % per16) || (heads > 1 && r.stride_h % per16)) return SEGPT_E_STRIDE;
  int64_t st[3] = {r.stride_t, r.stride_h, p.D}, ex[3] = {p.T, heads, 1};
  return out && overlaps_itself(st, ex, p.D) ? SEGPT_E_STRIDE : SEGPT_OK;
}

}  // namespace

// what can be said of the sizes alone, without an address being looked at
int check_paged_sizes(const segpt_paged_params* p, bool append) {
  if (!p) return SEGPT_E_NULL;
  if (p->struct_bytes != sizeof(segpt_paged_params)) return SEGPT_E_STRUCT;
  if (p->dtype != SEGPT_DTYPE_BF16 && p->dtype != SEGPT_DTYPE_FP32) return SEGPT_E_DTYPE;
  if (p->T <= 0 || p->B <= 0 || p->Hkv <= 0 || (!append && (p->H <= 0 || p->H % p->Hkv))) return SEGPT_E_SHAPE;
  if (p->Hkv > 65535 || (!append && p->H > 65535) || p->B > (1 << 24)) return SEGPT_E_SHAPE;
  if ((int64_t)p->T * (append ? p->Hkv : p->H) > (1 << 30) || (!p->seq_start && p->T % p->B)) return SEGPT_E_SHAPE;
  if (p->D != 64 && p->D != 128 && !(p->D == 32 && p->dtype == SEGPT_DTYPE_FP32)) return SEGPT_E_HEAD_DIM;
  if (p->page_size < 8 || p->page_size > 65536 || (p->page_size & (p->page_size - 1)) || p->table_width <= 0) return SEGPT_E_PAGES;
  if (p->prefix_len < 0 || p->max_len < 0 || (int64_t)p->table_width * p->page_size + p->prefix_len > INT32_MAX - (1 << 20)) return SEGPT_E_PAGES;
  return SEGPT_OK;
}

int check_paged(const segpt_paged_params* p, bool append) {
  int rc = check_paged_sizes(p, append);
  if (rc) return rc;
  if (p->n_pages <= 0) return SEGPT_E_PAGES;
  const int64_t positions = (int64_t)paged_capacity(*p) + (append ? 0 : p->prefix_len);
  if (!p->block_table || !p->kv_len) return SEGPT_E_NULL;
  if (p->table_stride < 0) return SEGPT_E_STRIDE;
  if (!aligned(p->block_table, 4) || !aligned(p->kv_len, 4) || !aligned(p->seq_start, 4)) return SEGPT_E_ALIGN;
  if ((rc = check_pool(p->k_pages, *p, append))) return rc;
  if ((rc = check_pool(p->v_pages, *p, append))) return rc;
  if (p->rope_cos || p->rope_sin) {
    if (!p->rope_cos || !p->rope_sin || !aligned(p->rope_cos, 16) || !aligned(p->rope_sin, 16)) return SEGPT_E_ROPE;
    if (p->rope_pos0 < 0 || p->rope_pos0 + positions > p->rope_len) return SEGPT_E_ROPE;
  }
  if (append) {
    if ((rc = check_rows(p->k, *p, p->Hkv, false))) return rc;
    if ((rc = check_rows(p->v, *p, p->Hkv, false))) return rc;
    if ((p->v_first.ptr != nullptr) != (p->vr_coef != nullptr)) return SEGPT_E_EXTRAS;
    return p->v_first.ptr ? check_rows(p->v_first, *p, p->Hkv, false) : SEGPT_OK;
  }
  if (p->gq_numel != 1 && p->gq_numel != p->D) return SEGPT_E_SHAPE;
  if (p->gk_numel != 0 && p->gk_numel != 1 && p->gk_numel != p->D) return SEGPT_E_SHAPE;
  if ((p->gk_numel != 0) != (p->g_k != nullptr)) return SEGPT_E_SHAPE;
  if (!p->g_q) return SEGPT_E_NULL;
  if ((p->prefix_table != nullptr) != (p->prefix_len > 0)) return SEGPT_E_EXTRAS;
  if (!aligned(p->prefix_table, 4)) return SEGPT_E_ALIGN;
  if ((rc = check_rows(p->q, *p, p->H, false))) return rc;
  if ((rc = check_rows(p->o, *p, p->H, true))) return rc;
  if (p->gate.ptr && (p->gate.stride_t < 0 || p->gate.stride_h < 0)) return SEGPT_E_STRIDE;
  return SEGPT_OK;
}

}  // namespace segpt

extern "C" int segpt_paged_append(const segpt_paged_params* p, void* stream) {
  using namespace segpt;
  const int rc = check_paged(p, true);
  if (rc) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (p->dtype == SEGPT_DTYPE_BF16) return p->D == 64 ? launch<uint16_t, 64>(*p, st) : launch<uint16_t, 128>(*p, st);
  return p->D == 32 ? launch<float, 32>(*p, st) : p->D == 64 ? launch<float, 64>(*p, st) : launch<float, 128>(*p, st);
}
