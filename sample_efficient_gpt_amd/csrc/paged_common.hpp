// What the kernels around the paged key/value cache share: host-side checks, and which sequence a row belongs to.
#pragma once

#include "common.hpp"

namespace segpt {

enum class PagedCall { kAppend, kRead, kAttend };
int check_paged_sizes(const segpt_paged_params* p, PagedCall call);
// row, whole: elements of the pool's rows and elements of 16 bytes; 0: the pool holds rows of p's dtype
int check_paged(const segpt_paged_params* p, PagedCall call, int64_t row = 0, int64_t whole = 0);
int check_pool(const segpt_tensor4& t, const segpt_paged_params& p, int64_t row, int64_t whole, int bytes, bool out);
// keys a sequence may hold (checked: fits an int)
__host__ __device__ inline int paged_capacity(const segpt_paged_params& p) {
  const int64_t room = (int64_t)p.table_width * p.page_size;
  return (int)(p.max_len > 0 && p.max_len < room ? p.max_len : room);
}

// Row range of sequence b, cut off at the rows there are
__device__ __forceinline__ void sequence_rows(const segpt_paged_params& p, int rows_each, int b, int* first, int* n) {
  if (!p.seq_start) {
    *first = b * rows_each;
    *n = rows_each;
    return;
  }
  const int r0 = min(max(p.seq_start[b], 0), p.T), r1 = min(max(p.seq_start[b + 1], 0), p.T);
  *first = r0;
  *n = max(r1 - r0, 0);
}

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

// the same for lanes whose rows t begin with the wave's row t0 and follow it
__device__ __forceinline__ int lane_sequence(const segpt_paged_params& p, int rows_each, int t0, int t, int lane) {
  if (!p.seq_start) return t / rows_each;
  int b = sequence_of_row(p, t0, lane);
  // a later row of the wave: mostly the next sequence, but any number without rows may lie between
  int step = 1;
  for (; b + step < p.B && p.seq_start[b + step] <= t; step *= 2) b += step;
  while (step >>= 1)
    if (b + step < p.B && p.seq_start[b + step] <= t) b += step;
  return b;
}

// byte address of row (page, head, slot) of a pool
template <typename E>
__device__ __forceinline__ char* page_row(const segpt_tensor4& t, int page, int head, int slot) {
  return reinterpret_cast<char*>(t.ptr) + ((int64_t)page * t.stride_b + (int64_t)head * t.stride_h + (int64_t)slot * t.stride_s) * (int)sizeof(E);
}
template <typename E>
__device__ __forceinline__ E* row_of(const segpt_rows& r, int t, int h) {
  return reinterpret_cast<E*>(r.ptr) + (int64_t)t * r.stride_t + (int64_t)h * r.stride_h;
}

// sixteen bytes of a row
__device__ __forceinline__ void load16(const uint16_t* p, float (&x)[8]) { Elem<uint16_t>::load(p, x); }
__device__ __forceinline__ void load16(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void store16(uint16_t* p, const float (&x)[8]) { Elem<uint16_t>::store(p, x); }
__device__ __forceinline__ void store16(float* p, const float (&x)[4]) { *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]); }

}  // namespace segpt
