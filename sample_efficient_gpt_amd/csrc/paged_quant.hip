// Rows of keys and values into paged caches of 8 or 4 bits, and back.
//
//   k'_p = rot_p(k) * rsqrt(mean k^2 + eps)        v'_p = c1 v + c2 v_first        p = kv_len[b] - n + i
//   block of 32 components:  e = min{ e >= -110 : max |x| <= 2^e top },   code_i = nearest(x_i / 2^e)
//
// The codes are to be those of the exact value: a value projected in bf16 lies on the border of two codes once in sixteen times (once in 2^8 with 4
// bits), and a key next to one would go either way with the order of a sum.  Keys, and values that are mixed, are therefore worked out in 64 bits
// (products of two fp32 numbers are exact there) and reach the codes through a float that is rounded to odd: cut off, its last bit set where
// anything was cut, so that the second rounding sees which side of a border the value lay on.
#include <algorithm>
#include <type_traits>

#include "paged_quant.hpp"

namespace segpt {

namespace {

constexpr int kThreads = 256;

// ---- a block's scale.  The size of a number as 32 bits that keep its order: exponent, leading fraction and, of a double, whether there is more behind
// them, so that a value just above the largest code's multiple is told from it.  What is not finite comes last.
__device__ __forceinline__ uint32_t size_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return (uint32_t)(u >> 32) << 1 | min((uint32_t)u, 1u);
}
__device__ __forceinline__ uint32_t size_of(float x) { return __float_as_uint(x) << 1; }
// smallest e with size <= 2^e top
template <int FMT, typename T>
__device__ __forceinline__ int exponent_of(uint32_t size) {
  constexpr int kFraction = sizeof(T) == 8 ? 21 : 24, kBias = sizeof(T) == 8 ? 1023 : 127;
  constexpr uint32_t kTop = FMT == SEGPT_POOL_E4M3 ? 3u << (kFraction - 2) : 1u << (kFraction - 1);  // fraction of 448 = 1.75 2^8, of 6 = 1.5 2^2
  return (int)(size >> kFraction) - kBias - (FMT == SEGPT_POOL_E4M3 ? 8 : 2) + ((size & ((1u << kFraction) - 1)) > kTop);
}

// x 2^-e as a float that rounds on as x 2^-e does: exponent moved and fraction cut off in whole-number arithmetic, the last bit set where a bit that is
// cut off was.  Under 2^-100 all rounds to 0.
__device__ __forceinline__ float scaled(double x, int e) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
  const uint32_t size = hi & 0x7FFFFFFFu, moved = size - ((uint32_t)e << 20);
  const uint32_t f = (__builtin_amdgcn_alignbit(moved, lo, 29) - (896u << 23)) | min(lo & 0x1FFFFFFFu, 1u);
  // size: below the exponent of 2^(e - 100) there is nothing left, 0 itself and what is no normal double among it
  return __uint_as_float((size < (uint32_t)(1023 - 100 + e) << 20 ? 0u : f) | (hi & 0x80000000u));
}
__device__ __forceinline__ float scaled(float x, int e) { return x * __uint_as_float((uint32_t)(127 - e) << 23); }

template <int VEC, typename T>
__device__ __forceinline__ uint32_t largest_of(const T (&x)[VEC]) {
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < VEC; ++i) largest = max(largest, size_of(x[i]));
  return largest;
}
// VEC components of a block spread over LANES lanes: their codes, VEC * bits / 8 bytes, and the block's scale; largest: of this lane's
template <int FMT, int VEC, int LANES, typename T>
__device__ __forceinline__ uint32_t encode(const T (&x)[VEC], uint32_t largest, uint32_t (&w)[2]) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) largest = max(largest, (uint32_t)__shfl_xor((int)largest, o, 64));
  const int e = max(exponent_of<FMT, T>(largest), kLeastExponent);
  const bool none = e > Codes<FMT>::kMostExponent;
  float y[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) y[i] = scaled(x[i], e);
  w[0] = w[1] = 0u;
  if constexpr (FMT == SEGPT_POOL_E4M3) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4)
      w[i / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(y[i + 2], y[i + 3], __builtin_amdgcn_cvt_pk_fp8_f32(y[i], y[i + 1], 0, false), true);
  } else {
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.f, 0);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], y[2], y[3], 1.f, 1);
    if constexpr (VEC == 8) {
      w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], y[4], y[5], 1.f, 2);
      w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], y[6], y[7], 1.f, 3);
    }
  }
  if (none) w[0] = w[1] = 0u;
  return none ? kNoNumber : (uint32_t)(e + 127);
}
// a lane's components of either half of a row: codes and scales
template <int FMT, int D, int VEC, typename T>
__device__ __forceinline__ void encode_halves(const T (&x)[2][VEC], uint32_t (&w)[2][2], uint32_t (&scale)[2]) {
  constexpr bool kOneBlock = D == SEGPT_SCALE_BLOCK;  // both halves are of one block
  constexpr int kLanes = (kOneBlock ? D / 2 : SEGPT_SCALE_BLOCK) / VEC;
  uint32_t largest[2] = {largest_of(x[0]), largest_of(x[1])};
  if (kOneBlock) largest[0] = largest[1] = max(largest[0], largest[1]);
#pragma unroll
  for (int h = 0; h < 2; ++h) scale[h] = encode<FMT, VEC, kLanes>(x[h], largest[h], w[h]);
}
template <int BYTES>
__device__ __forceinline__ void store_codes(char* at, const uint32_t (&w)[2]) {
  if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
  else if constexpr (BYTES == 4) *reinterpret_cast<uint32_t*>(at) = w[0];
  else *reinterpret_cast<uint16_t*>(at) = (uint16_t)w[0];
}

// A row is D * sizeof(E) / 32 lanes, as in the append of whole numbers: a lane holds 16 bytes of the first half and the 16 bytes of the second half
// that they rotate with, and the lanes of a block stand side by side.  Bound by what a wave waits for, one after the other: its sequence, the page number
// and the angles, then the sum of squares and the blocks' largest.  One token 3.4 us; 16 ragged prompts of head_dim 128, 69 MB with the codes: 20.8 us,
// 3.3 TB/s.  Fewer instructions for scales and codes did not change that.  At head_dim 32 both halves are of one block.  (Eight bytes of each, so that every SIMD holds its eight waves and not four: the
// prompts below take 24.4 us, since a lane's share of finding its row and its block's scale does not halve.  Rows kept as stored and values first, for
// five waves: 21.4.)
template <typename E, int D, int FMT, bool ROPE, bool MIX>
__global__ __launch_bounds__(kThreads) void paged_append_quant_kernel(QuantArgs a, int log_page, int rows_each, int capacity) {
  const segpt_paged_params& p = a.p;
  constexpr int VEC = 16 / sizeof(E), LPR = D / 2 / VEC, kRowsPerWave = 64 / LPR, kBytes = VEC * Codes<FMT>::kBits / 8;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t first = (blockIdx.x * (kThreads / 64) + wave) * kRowsPerWave, total = (uint32_t)p.T * (uint32_t)p.Hkv, heads = p.Hkv;  // at most 2^30 rows
  if (first >= total) return;
  const uint32_t row = min(first + lane / LPR, total - 1);
  const bool live = first + lane / LPR < total;
  const int t = (int)(row / heads), g = (int)(row - t * heads), c = (lane % LPR) * VEC;

  float k[2][VEC], v[2][VEC], f[2][VEC];
  auto load = [&](const segpt_rows& r, float (&x)[2][VEC]) {
    const E* at = row_of<E>(r, t, g) + c;
#pragma unroll
    for (int i = 0; i < 2; ++i) load16(at + i * (D / 2), x[i]);
  };
  load(p.k, k);
  load(p.v, v);
  if constexpr (MIX) load(p.v_first, f);

  int r0, n;
  const int b = lane_sequence(p, rows_each, (int)(first / heads), t, lane);
  sequence_rows(p, rows_each, b, &r0, &n);
  const int64_t pos = (int64_t)p.kv_len[b] - n + (t - r0);
  const bool placed = live && t >= r0 && t < r0 + n && pos >= 0 && pos < capacity;
  const int at = placed ? (int)pos : 0;
  const int page = p.block_table[(int64_t)b * p.table_stride + (at >> log_page)];

  double kd[2][VEC];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < VEC; ++i) kd[h][i] = k[h][i];
  if constexpr (ROPE) {
    const int64_t angle = ((int64_t)p.rope_pos0 + at) * (D / 2) + c;  // within the tables: they cover every position of the table
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(p.rope_cos + angle + i), y = *reinterpret_cast<const float4*>(p.rope_sin + angle + i);
      const double cs[4] = {x.x, x.y, x.z, x.w}, sn[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double u = kd[0][i + j], w = kd[1][i + j];
        kd[0][i + j] = u * cs[j] - w * sn[j];
        kd[1][i + j] = u * sn[j] + w * cs[j];
      }
    }
  }
  if (!(p.flags & SEGPT_FLAG_NO_NORM)) {
    double ss = 0.;
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss += kd[0][i] * kd[0][i] + kd[1][i] * kd[1][i];
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor(ss, o, 64);
    const double beta = 1.0 / sqrt(ss * (1.0 / D) + (double)p.eps);
#pragma unroll
    for (int i = 0; i < VEC; ++i) { kd[0][i] *= beta; kd[1][i] *= beta; }
  }
  uint32_t kw[2][2], vw[2][2], ks[2], vs[2];
  encode_halves<FMT, D>(kd, kw, ks);
  if constexpr (MIX) {
    const double c1 = p.vr_coef[0], c2 = p.vr_coef[1];
    double x[2][VEC];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[h][i] = fma(c2, (double)f[h][i], c1 * v[h][i]);
    encode_halves<FMT, D>(x, vw, vs);
  } else {
    encode_halves<FMT, D>(v, vw, vs);
  }
  if (!placed || (uint32_t)page >= (uint32_t)p.n_pages) return;
  const int slot = at & ((1 << log_page) - 1);
  char* kc = byte_row(p.k_pages, page, g, slot) + c * Codes<FMT>::kBits / 8;
  char* vc = byte_row(p.v_pages, page, g, slot) + c * Codes<FMT>::kBits / 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    store_codes<kBytes>(kc + h * Codes<FMT>::row_bytes(D / 2), kw[h]);
    store_codes<kBytes>(vc + h * Codes<FMT>::row_bytes(D / 2), vw[h]);
  }
  if (c % SEGPT_SCALE_BLOCK == 0) {
    char* kb = byte_row(a.k_scales, page, g, slot) + c / SEGPT_SCALE_BLOCK;
    char* vb = byte_row(a.v_scales, page, g, slot) + c / SEGPT_SCALE_BLOCK;
#pragma unroll
    for (int h = 0; h < (D == SEGPT_SCALE_BLOCK ? 1 : 2); ++h) {
      kb[h * (D / 2 / SEGPT_SCALE_BLOCK)] = (char)ks[h];
      vb[h * (D / 2 / SEGPT_SCALE_BLOCK)] = (char)vs[h];
    }
  }
}

// ---- stored rows back as rows.  FMT 0: rows of E.  A lane writes 16 bytes of a row of keys and of one of values; bound by the bytes that it moves.
// Eight sequences of 1,641 .. 8,185 positions, head_dim 64, 91 MB with what is written: 19 us, 4.8 TB/s, the rate of a large copy.
template <typename E, int D, int FMT>
__global__ __launch_bounds__(kThreads) void paged_read_kernel(QuantArgs a, int log_page, int rows_each, int capacity) {
  const segpt_paged_params& p = a.p;
  constexpr int VEC = 16 / sizeof(E), LPR = D / VEC, kRowsPerWave = 64 / LPR;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t first = (blockIdx.x * (kThreads / 64) + wave) * kRowsPerWave, total = (uint32_t)p.T * (uint32_t)p.Hkv, heads = p.Hkv;  // at most 2^30 rows
  if (first >= total) return;
  const uint32_t row = min(first + lane / LPR, total - 1);
  const int t = (int)(row / heads), g = (int)(row - t * heads), c = (lane % LPR) * VEC;
  int r0, n;
  const int b = lane_sequence(p, rows_each, (int)(first / heads), t, lane);
  sequence_rows(p, rows_each, b, &r0, &n);
  if (first + lane / LPR >= total) return;  // not before: the whole wave looks for its sequence
  const bool owned = t >= r0 && t < r0 + n;
  if (!owned && !(p.flags & SEGPT_FLAG_ZERO_REST)) return;
  const int len = p.kv_len[b];
  const int64_t pos = (int64_t)len - n + (t - r0);
  const bool broken = len < 0 || len > capacity, there = owned && !broken && pos >= 0;
  const int at = there ? (int)pos : 0;
  const int page = p.block_table[(int64_t)b * p.table_stride + (at >> log_page)];
  const bool held = there && (uint32_t)page < (uint32_t)p.n_pages;
  const float other = owned && (broken || (there && !held)) ? __builtin_nanf("") : 0.f;
  const int slot = at & ((1 << log_page) - 1), from = held ? page : 0;
  auto back = [&](const segpt_tensor4& pages, const segpt_tensor4& scales, const segpt_rows& to) {
    E* out = row_of<E>(to, t, g) + c;
    if constexpr (FMT == 0) {
      float x[VEC];
      if (held) load16(reinterpret_cast<const E*>(page_row<E>(pages, from, g, slot)) + c, x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = held ? x[i] : other;
      store16(out, x);
    } else {
      const char* codes = byte_row(pages, from, g, slot) + c * Codes<FMT>::kBits / 8;
      const float scale = scale_of_byte(*reinterpret_cast<const uint8_t*>(byte_row(scales, from, g, slot) + c / SEGPT_SCALE_BLOCK));
      uint32_t w[2] = {0u, 0u}, x[4];
      if constexpr (VEC * Codes<FMT>::kBits == 64) { const uint2 r = *reinterpret_cast<const uint2*>(codes); w[0] = r.x; w[1] = r.y; }
      else if constexpr (VEC * Codes<FMT>::kBits == 32) w[0] = *reinterpret_cast<const uint32_t*>(codes);
      else w[0] = *reinterpret_cast<const uint16_t*>(codes);
      decode8<FMT>(w, scale, x);
      if constexpr (sizeof(E) == 2) {
        const uint32_t z = pack_bf16x2(other, other);
        *reinterpret_cast<uint4*>(out) = held ? make_uint4(x[0], x[1], x[2], x[3]) : make_uint4(z, z, z, z);
      } else {
        *reinterpret_cast<float4*>(out) = held ? make_float4(bf16lo(x[0]), bf16hi(x[0]), bf16lo(x[1]), bf16hi(x[1])) : make_float4(other, other, other, other);
      }
    }
  };
  back(p.k_pages, a.k_scales, p.k);
  back(p.v_pages, a.v_scales, p.v);
}

template <int LANES>
bool grid_of(const segpt_paged_params& p, dim3* grid) {
  constexpr int kRows = kThreads / LANES;
  const int64_t groups = ((int64_t)p.T * p.Hkv + kRows - 1) / kRows;
  *grid = dim3((unsigned)std::min<int64_t>(groups, UINT32_MAX));
  return groups <= UINT32_MAX / kThreads;  // a launch has fewer than 2^32 threads
}

template <typename E, int D, int FMT>
int launch_append(const QuantArgs& a, hipStream_t st) {
  const segpt_paged_params& p = a.p;
  dim3 grid;
  if (!grid_of<D * (int)sizeof(E) / 32>(p, &grid)) return SEGPT_E_SHAPE;
  const int log_page = __builtin_ctz((unsigned)p.page_size), each = p.seq_start ? 0 : p.T / p.B, room = paged_capacity(p);
  const bool mix = p.v_first.ptr != nullptr;
  if (p.rope_cos) {
    if (mix) hipLaunchKernelGGL((paged_append_quant_kernel<E, D, FMT, true, true>), grid, dim3(kThreads), 0, st, a, log_page, each, room);
    else hipLaunchKernelGGL((paged_append_quant_kernel<E, D, FMT, true, false>), grid, dim3(kThreads), 0, st, a, log_page, each, room);
  } else {
    if (mix) hipLaunchKernelGGL((paged_append_quant_kernel<E, D, FMT, false, true>), grid, dim3(kThreads), 0, st, a, log_page, each, room);
    else hipLaunchKernelGGL((paged_append_quant_kernel<E, D, FMT, false, false>), grid, dim3(kThreads), 0, st, a, log_page, each, room);
  }
  return (int)hipGetLastError();
}
template <typename E, int D, int FMT>
int launch_read(const QuantArgs& a, hipStream_t st) {
  const segpt_paged_params& p = a.p;
  dim3 grid;
  if (!grid_of<D * (int)sizeof(E) / 16>(p, &grid)) return SEGPT_E_SHAPE;
  hipLaunchKernelGGL((paged_read_kernel<E, D, FMT>), grid, dim3(kThreads), 0, st, a, __builtin_ctz((unsigned)p.page_size), p.seq_start ? 0 : p.T / p.B, paged_capacity(p));
  return (int)hipGetLastError();
}

}  // namespace

// heads of 32 are an extension that a caller asks for: the entries' first callers go by the refusal
bool quant_head_dim(const segpt_paged_params& p) { return p.D == 64 || p.D == 128 || (p.D == 32 && (p.flags & SEGPT_FLAG_HEAD_32)); }

int check_quant(const segpt_paged_params* p, const segpt_paged_quant* q, PagedCall call) {
  int rc = check_paged_sizes(p, call);
  if (rc) return rc;
  if (!q) return SEGPT_E_NULL;
  if (q->struct_bytes != sizeof(segpt_paged_quant)) return SEGPT_E_STRUCT;
  if (q->format != SEGPT_POOL_E4M3 && q->format != SEGPT_POOL_E2M1) return SEGPT_E_DTYPE;
  if (!quant_head_dim(*p)) return SEGPT_E_HEAD_DIM;
  if ((rc = check_paged(p, call, q->format == SEGPT_POOL_E4M3 ? p->D : p->D / 2, 16))) return rc;
  if (p->n_pages <= 0) return SEGPT_E_PAGES;
  const int scales = p->D / SEGPT_SCALE_BLOCK;
  const bool out = call == PagedCall::kAppend;
  if ((rc = check_pool(q->k_scales, *p, scales, scales, scales, out))) return rc;
  return check_pool(q->v_scales, *p, scales, scales, scales, out);
}

}  // namespace segpt

extern "C" {

int segpt_paged_append_quant(const segpt_paged_params* p, const segpt_paged_quant* q, void* stream) {
  using namespace segpt;
  const int rc = check_quant(p, q, PagedCall::kAppend);
  if (rc) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const QuantArgs a{*p, q->k_scales, q->v_scales};
  const bool e4m3 = q->format == SEGPT_POOL_E4M3;
  if (p->dtype == SEGPT_DTYPE_BF16) {
    if (p->D == 64) return e4m3 ? launch_append<uint16_t, 64, SEGPT_POOL_E4M3>(a, st) : launch_append<uint16_t, 64, SEGPT_POOL_E2M1>(a, st);
    return e4m3 ? launch_append<uint16_t, 128, SEGPT_POOL_E4M3>(a, st) : launch_append<uint16_t, 128, SEGPT_POOL_E2M1>(a, st);
  }
  if (p->D == 32) return e4m3 ? launch_append<float, 32, SEGPT_POOL_E4M3>(a, st) : launch_append<float, 32, SEGPT_POOL_E2M1>(a, st);
  if (p->D == 64) return e4m3 ? launch_append<float, 64, SEGPT_POOL_E4M3>(a, st) : launch_append<float, 64, SEGPT_POOL_E2M1>(a, st);
  return e4m3 ? launch_append<float, 128, SEGPT_POOL_E4M3>(a, st) : launch_append<float, 128, SEGPT_POOL_E2M1>(a, st);
}

int segpt_paged_read(const segpt_paged_params* p, const segpt_paged_quant* q, void* stream) {
  using namespace segpt;
  const int rc = q ? check_quant(p, q, PagedCall::kRead) : check_paged(p, PagedCall::kRead);
  if (rc) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const QuantArgs a{*p, q ? q->k_scales : segpt_tensor4{}, q ? q->v_scales : segpt_tensor4{}};
  const int format = q ? q->format : 0;
  auto go = [&](auto elem, auto dim) {
    using E = decltype(elem);
    constexpr int D = decltype(dim)::value;
    if (format == 0) return launch_read<E, D, 0>(a, st);
    return format == SEGPT_POOL_E4M3 ? launch_read<E, D, SEGPT_POOL_E4M3>(a, st) : launch_read<E, D, SEGPT_POOL_E2M1>(a, st);
  };
  if (p->dtype == SEGPT_DTYPE_BF16) return p->D == 64 ? go(uint16_t{}, std::integral_constant<int, 64>{}) : go(uint16_t{}, std::integral_constant<int, 128>{});
  return p->D == 32 ? go(0.f, std::integral_constant<int, 32>{}) : p->D == 64 ? go(0.f, std::integral_constant<int, 64>{}) : go(0.f, std::integral_constant<int, 128>{});
}

}  // extern "C"
