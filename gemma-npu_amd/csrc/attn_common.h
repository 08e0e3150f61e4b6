// Device helpers that the attention kernels share.
#pragma once
#include "w8a8_common.h"

namespace w8a8 {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

// v combined over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the same row of an MFMA tile in the four
// 16-lane groups) by the gfx950 lane swaps, in VALU instead of two ds_bpermute round trips through
// LDS: v_permlane16_swap exchanges 16-lane groups 0 <-> 1 and 2 <-> 3, v_permlane32_swap the two
// halves, and of the two results one holds the lane's own value and the other its partner's.  The
// pairs are those of a xor-16 then xor-32 butterfly and both combines are commutative, so the result
// is bit-identical to that butterfly on every lane.
__device__ __forceinline__ float lanes4_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lanes4_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Waits until at most N of the wave's vector memory operations are outstanding.
template <int N>
__device__ __forceinline__ void attn_wait_vmcnt() {
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}

__device__ __forceinline__ void attn_dma16(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}

// s where `vis`, else -inf, as a select of the bit patterns
__device__ __forceinline__ float attn_mask(float s, bool vis) {
  return __uint_as_float(vis ? __float_as_uint(s) : 0xff800000u);
}

// Compute units of the current device (256 on MI355X), read once.
int attn_cu_count();

}  // namespace w8a8
