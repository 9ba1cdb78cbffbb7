// What the kernels around paged caches of 8 and 4 bits share: the stored form of a row, and the numbers it stands for.
#pragma once

#include "paged_common.hpp"

namespace segpt {

// Operands of a call beside the params: format and scales.  The pools' strides in the params are bytes.
struct QuantArgs {
  segpt_paged_params p;
  segpt_tensor4 k_scales, v_scales;
};
int check_quant(const segpt_paged_params* p, const segpt_paged_quant* q, PagedCall call);
bool quant_head_dim(const segpt_paged_params& p);

constexpr int kLeastExponent = -110;  // of a scale: the smallest code times it is a normal bf16 number
constexpr int kNoNumber = 255;        // scale of a block with a component that cannot be held
template <int FMT>
struct Codes {
  static constexpr bool k8 = FMT == SEGPT_POOL_E4M3;
  static constexpr int kBits = k8 ? 8 : 4;
  static constexpr int kMostExponent = k8 ? 119 : 125;  // the largest code times it is a float
  static constexpr int row_bytes(int D) { return D * kBits / 8; }
};

// Components of a stored block, in pairs, times its scale: exact (4 bits of significand or fewer, and the scale a power of two).  The instruction
// takes the scale as the float 2^e, i.e. the byte as its exponent; 255 makes NaN of every code.
__device__ __forceinline__ float scale_of_byte(uint32_t byte) { return __uint_as_float(byte << 23); }
template <int FMT, int PAIR>  // of the 32-bit word w: two pairs of E4M3, four of E2M1
__device__ __forceinline__ uint32_t decode_bf16x2(uint32_t w, float scale) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  bf2 x;
  if constexpr (FMT == SEGPT_POOL_E4M3) x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, PAIR != 0);
  else x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, PAIR);
  return __builtin_bit_cast(uint32_t, x);
}
// 8 components: two words of E4M3, one of E2M1
template <int FMT>
__device__ __forceinline__ void decode8(const uint32_t* w, float scale, uint32_t (&x)[4]) {
  if constexpr (FMT == SEGPT_POOL_E4M3) {
    x[0] = decode_bf16x2<FMT, 0>(w[0], scale);
    x[1] = decode_bf16x2<FMT, 1>(w[0], scale);
    x[2] = decode_bf16x2<FMT, 0>(w[1], scale);
    x[3] = decode_bf16x2<FMT, 1>(w[1], scale);
  } else {
    x[0] = decode_bf16x2<FMT, 0>(w[0], scale);
    x[1] = decode_bf16x2<FMT, 1>(w[0], scale);
    x[2] = decode_bf16x2<FMT, 2>(w[0], scale);
    x[3] = decode_bf16x2<FMT, 3>(w[0], scale);
  }
}

// byte address of row (page, head, slot) of codes or scales
__device__ __forceinline__ char* byte_row(const segpt_tensor4& t, int page, int head, int slot) {
  return reinterpret_cast<char*>(t.ptr) + (int64_t)page * t.stride_b + (int64_t)head * t.stride_h + (int64_t)slot * t.stride_s;
}

}  // namespace segpt
