// What the kernels around the paged key/value cache share: host-side checks, and which sequence a row belongs to.
#pragma once

#include "common.hpp"

namespace segpt {

int check_paged_sizes(const segpt_paged_params* p, bool append);
int check_paged(const segpt_paged_params* p, bool append);
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
