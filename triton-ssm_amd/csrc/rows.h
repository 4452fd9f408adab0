// Pieces of the kernels that go step by step with the state in registers.
#pragma once

#include <type_traits>

#include "common.h"

namespace tssm {
namespace {

// Sum over the lanes that share lane % CQ.
template <int CQ>
__device__ inline float sum_kg(float v) {
  if constexpr (CQ == 4) v += dpp_mov<0x124>(v);  // row_ror:4
  v += dpp_mov<0x128>(v);                         // row_ror:8
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// N consecutive elements of T as floats; VEC: p is aligned to the widest access.
template <typename T, int N, bool VEC>
struct Row {
  static constexpr int kBytes = N * (int)sizeof(T);
  static constexpr int kW = VEC ? (kBytes < 16 ? kBytes : 16) : (int)sizeof(T);
  static constexpr int kN = kBytes / kW;
  typedef std::conditional_t<
      kW == 16, u32x4,
      std::conditional_t<kW == 8, uint2, std::conditional_t<kW == 4, uint32_t, uint16_t>>>
      word;
  union {
    word w[kN];
    T e[N];
  };
  // elements lim and up read element 0 (which exists) and count as zero
  __device__ inline void load(const T* p, int lim) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      w[i] = reinterpret_cast<const word*>(p)[VEC || i < lim ? i : 0];
  }
  __device__ inline float get(int i, int lim) const {
    return VEC || i < lim ? ldf(&e[i]) : 0.0f;
  }
};

}  // namespace
}  // namespace tssm
