// Rows put into the 8-bit key / value cache (blocks.h) and read back.
//
// A block's scale is max |x| / 127 (int8) or times 1 / 448 (e4m3) over its 64 rows of one KV head, its codes the nearest to
// x / scale, as the engine quantises activations (pipeline.py:51).  A block gets its codes once, when its last
// row arrives; until then its rows stay bf16 in the ring, so what the cache holds does not depend on how the
// rows came, and rows may be written again (drafted tokens taken back) while the ring has their block's others.
//
// block_append_kernel: a workgroup takes a block's keys (or values) of one head.  New rows go into the ring if their block is
// one of the call's last two.  A block that has become whole is taken from the ring, which lies as the codes do, if some
// of its rows were there before, else staged in LDS; its largest magnitude is taken on the way.  Memory bounds long calls
// (65521 rows of 8 heads of 128: 86 us of 79 at a copy's rate), one kernel's start and two round trips short ones.
#include <algorithm>

#include "blocks.h"

namespace w8a8 {

struct AppendParams {
  BlockCache c;
  const uint16_t *k, *v;  // bf16 [KV, m, D] (element strides of heads and rows)
  int64_t khs, krs, vhs, vrs;
  int m, n, capacity;
  const int32_t* n_dev;   // n in device memory, or null
};

// int8: the engine's own step.  e4m3: the magnitude times 1 / 448 rounded to fp32, which keeps x / scale off the e4m3
// midpoints that an exact quotient of short bf16 magnitudes would meet.
__device__ __forceinline__ float code_scale(float amax, bool e4m3) {
  return e4m3 ? (amax != amax ? amax : fmaxf(amax, 1e-8f)) * (1.0f / 448.0f) : quant_scale(amax);
}

// Eight values' codes.  A block with a NaN or an infinity has a scale that is one, and codes of 0: all of it reads NaN.
template <bool E4M3>
__device__ __forceinline__ v2u block_codes(const float (&x)[8], float s, float rs, bool finite) {
  if (!finite) return v2u{0u, 0u};
  if constexpr (E4M3) {
    v2u w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] / s, x[4 * h + 1] / s, 0, false);
      w[h] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] / s, x[4 * h + 3] / s, r, true));
    }
    return w;
  } else {
    return quant8(x, s, rs, true);
  }
}

template <int D, bool E4M3>
__global__ __launch_bounds__(256) void block_append_kernel(AppendParams p) {
  constexpr int KCH = D / 8;           // 16-byte chunks of a row
  constexpr int NU = BLK * KCH / 256;  // chunks of a thread
  constexpr int LD = D + 8;            // padded row, elements
  __shared__ __attribute__((aligned(16))) uint16_t st[BLK * LD];
  __shared__ uint32_t red[4];
  const int t = threadIdx.x, g = blockIdx.y, value = blockIdx.z;
  const int n = p.n_dev ? max(0, min(*p.n_dev, p.capacity - p.m)) : p.n;
  const int b0 = n / BLK, b = b0 + int(blockIdx.x), end = n + p.m, bl = (end - 1) / BLK;
  if (b > bl) return;
  const uint16_t* const src = value ? p.v + int64_t(g) * p.vhs : p.k + int64_t(g) * p.khs;
  const int64_t rs = value ? p.vrs : p.krs;
  uint16_t* const ring = (value ? p.c.vt : p.c.kt) + int64_t(g) * 2 * BLK * D;
  const int lo = max(n, b * BLK) - b * BLK, hi = min(end, (b + 1) * BLK) - b * BLK;  // the new rows

  // new rows of block x into the ring
  auto to_ring = [&](int x) __attribute__((always_inline)) {
    uint16_t* const at = ring + (x & 1) * BLK * D;
    const int first = max(n, x * BLK) - x * BLK, count = min(end, (x + 1) * BLK) - x * BLK - first;
    for (int i = t; i < count * KCH; i += 256) {
      const int r = first + i / KCH, d = i % KCH * 8;
      const v4u w = *reinterpret_cast<const v4u*>(src + (int64_t(x) * BLK + r - n) * rs + d);
      if (value) {
#pragma unroll
        for (int e = 0; e < 8; ++e) at[ring_value(r, d + e)] = uint16_t(w[e >> 1] >> (16 * (e & 1)));
      } else {
        *reinterpret_cast<v4u*>(at + ring_key(r, d, D)) = w;
      }
    }
  };

  const bool whole = hi == BLK, old = lo > 0;  // (old rows: the call's first block alone)
  const int64_t blk = int64_t(g) * p.c.blocks + b;
  uint8_t* const out = (value ? p.c.v : p.c.k) + blk * BLK * D;
  auto block_top = [&](uint32_t m2) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m2 = absmax_bf16x2(m2, __shfl_xor(m2, o, 64));
    if ((t & 63) == 0) red[t >> 6] = m2;
    __syncthreads();
    return absmax_pair(absmax_bf16x2(absmax_bf16x2(red[0], red[1]), absmax_bf16x2(red[2], red[3])));
  };
  if (whole && old) {
    // its new rows join the others in the ring, which lies as the codes do: 16 codes are two of its chunks
    to_ring(b);
    __syncthreads();
    const uint16_t* const at = ring + (b & 1) * BLK * D;
    v4u w[NU];
    uint32_t m2 = 0u;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int i = t + 256 * (u >> 1);
      w[u] = *reinterpret_cast<const v4u*>(at + ((2 * (i >> 6) + (u & 1)) * 64 + (i & 63)) * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) m2 = absmax_bf16x2(m2, w[u][e]);
    }
    const float s = code_scale(block_top(m2), E4M3), inv = 1.0f / s;
    const bool finite = quant_finite(s);
    if (t == 0) (value ? p.c.vs : p.c.ks)[blk] = s;
#pragma unroll
    for (int u = 0; u < NU; u += 2) {
      float x[2][8];
      unpack8(w[u], x[0]);
      unpack8(w[u + 1], x[1]);
      const v2u a = block_codes<E4M3>(x[0], s, inv, finite), c = block_codes<E4M3>(x[1], s, inv, finite);
      *reinterpret_cast<v4u*>(out + int64_t(t + 128 * u) * 16) = v4u{a[0], a[1], c[0], c[1]};
    }
  } else if (whole) {
    uint32_t m2 = 0u;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int i = u * 256 + t, r = i / KCH, d = i % KCH * 8;
      const v4u w = *reinterpret_cast<const v4u*>(src + (int64_t(b) * BLK + r - n) * rs + d);
      *reinterpret_cast<v4u*>(st + r * LD + d) = w;
#pragma unroll
      for (int e = 0; e < 4; ++e) m2 = absmax_bf16x2(m2, w[e]);
    }
    const float s = code_scale(block_top(m2), E4M3), inv = 1.0f / s;
    const bool finite = quant_finite(s);
    if (t == 0) (value ? p.c.vs : p.c.ks)[blk] = s;
    for (int i = t; i < BLK * D / 16; i += 256) {  // 16 codes: lane i % 64 of fragment i / 64
      const int f = i >> 6, qi = i & 15, qq = (i >> 4) & 3;
      float x[2][8];
      if (value) {
        const int d = 16 * f + qi;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[h][e] = bf16_to_f32(st[(32 * h + 16 * (e >> 2) + 4 * qq + (e & 3)) * LD + d]);
      } else {
        const int r = 16 * (f / (D / 64)) + qi, d = 64 * (f % (D / 64)) + 16 * qq;
#pragma unroll
        for (int h = 0; h < 2; ++h) unpack8(*reinterpret_cast<const v4u*>(st + r * LD + d + 8 * h), x[h]);
      }
      const v2u a = block_codes<E4M3>(x[0], s, inv, finite), c = block_codes<E4M3>(x[1], s, inv, finite);
      *reinterpret_cast<v4u*>(out + int64_t(i) * 16) = v4u{a[0], a[1], c[0], c[1]};
    }
  }
  // The ring.  A later block in the slot of the call's first one is written by that one's workgroup, once it has read
  // the slot.
  if (b >= bl - 1 && (b == b0 || ((b ^ b0) & 1)) && !(whole && old)) to_ring(b);
  if (b == b0 && bl - b0 >= 2) {
    const int later = bl - ((bl ^ b0) & 1);  // of bl and bl - 1 the one in b0's slot
    if (later > b0) {
      __syncthreads();
      to_ring(later);
    }
  }
}

struct ReadParams {
  BlockCache c;
  uint16_t *k, *v;  // bf16 [KV, count, D], contiguous
  int start, n;     // rows start .. n - 1 of n
};

// A code as fp32.
template <bool E4M3>
__device__ __forceinline__ void code_values(uint32_t w, float (&x)[4]) {
  if constexpr (E4M3) {
    const v2f a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = float(int(w << (24 - 8 * e)) >> 24);
  }
}

template <int D, bool E4M3>
__global__ __launch_bounds__(256) void block_read_kernel(ReadParams p) {
  constexpr int KCH = D / 8, LD = D + 8;
  __shared__ __attribute__((aligned(16))) uint16_t st[BLK * LD];
  const int t = threadIdx.x, g = blockIdx.y, value = blockIdx.z;
  const int b = p.start / BLK + int(blockIdx.x);
  const int lo = max(p.start, b * BLK) - b * BLK, hi = min(p.n, (b + 1) * BLK) - b * BLK;
  if (hi == BLK) {
    const int64_t blk = int64_t(g) * p.c.blocks + b;
    const uint8_t* const in = (value ? p.c.v : p.c.k) + blk * BLK * D;
    const float s = (value ? p.c.vs : p.c.ks)[blk];
    for (int i = t; i < BLK * D / 16; i += 256) {
      const int f = i >> 6, qi = i & 15, qq = (i >> 4) & 3;
      const v4u w = *reinterpret_cast<const v4u*>(in + int64_t(i) * 16);
      float x[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float y[4];
        code_values<E4M3>(w[j], y);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * j + e] = y[e] * s;
      }
      if (value) {
        const int d = 16 * f + qi;
#pragma unroll
        for (int e = 0; e < 16; ++e) st[(32 * (e >> 3) + 16 * ((e >> 2) & 1) + 4 * qq + (e & 3)) * LD + d] = f32_to_bf16(x[e]);
      } else {
        const int r = 16 * (f / (D / 64)) + qi, d = 64 * (f % (D / 64)) + 16 * qq;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = x[8 * h + e];
          *reinterpret_cast<v4u*>(st + r * LD + d + 8 * h) = pack8(y);
        }
      }
    }
  } else {
    const uint16_t* const at = (value ? p.c.vt : p.c.kt) + (int64_t(g) * 2 + (b & 1)) * BLK * D;
    for (int i = t; i < hi * KCH; i += 256) {
      const int r = i / KCH, d = i % KCH * 8;
      if (value) {
#pragma unroll
        for (int e = 0; e < 8; ++e) st[r * LD + d + e] = at[ring_value(r, d + e)];
      } else {
        *reinterpret_cast<v4u*>(st + r * LD + d) = *reinterpret_cast<const v4u*>(at + ring_key(r, d, D));
      }
    }
  }
  __syncthreads();
  uint16_t* const out = (value ? p.v : p.k) + (int64_t(g) * (p.n - p.start) + int64_t(b) * BLK - p.start) * D;
  for (int i = t + lo * KCH; i < hi * KCH; i += 256)
    *reinterpret_cast<v4u*>(out + int64_t(i) * 8) = *reinterpret_cast<const v4u*>(st + i / KCH * LD + i % KCH * 8);
}

}  // namespace w8a8

using namespace w8a8;

extern "C" int64_t w8a8_block_cache_bytes(int64_t KV, int64_t capacity, int64_t D) {
  if (!block_shape_ok(KV, capacity, D)) return -1;
  BlockCache c;
  return block_layout(nullptr, KV, capacity, D, c);
}

static int block_check(const char* what, const void* data, int64_t KV, int64_t capacity, int64_t D) {
  if (D != 128 && D != 256 && D != 512)
    return fail(W8A8_ENOTSUP, "%s: head_dim %lld (supported: 128, 256, 512)", what, (long long)D);
  if (!block_shape_ok(KV, capacity, D))
    return fail(W8A8_EINVAL, "%s: KV=%lld capacity=%lld", what, (long long)KV, (long long)capacity);
  if (!data) return fail(W8A8_EINVAL, "%s: null pointer", what);
  if ((uintptr_t)data % 16) return fail(W8A8_EALIGN, "%s: the cache must be 16-byte aligned", what);
  return W8A8_OK;
}

extern "C" int w8a8_block_append(void* cache, int64_t KV, int64_t capacity, int64_t D, int e4m3, const uint16_t* k,
                                 int64_t k_head_stride, int64_t k_row_stride, const uint16_t* v, int64_t v_head_stride,
                                 int64_t v_row_stride, int64_t m, int64_t n, const int32_t* n_dev, hipStream_t stream) {
  const char* what = "block_append";
  if (int rc = block_check(what, cache, KV, capacity, D)) return rc;
  if (m < 0 || m > capacity || (n_dev ? n != -1 : (n < 0 || n > capacity - m)))
    return fail(W8A8_EINVAL, "%s: %lld rows from %lld on in a cache of %lld (-1 with a device position)", what, (long long)m,
                (long long)n, (long long)capacity);
  if (m == 0) return W8A8_OK;
  if (!k || !v) return fail(W8A8_EINVAL, "%s: null pointer", what);
  const int64_t rs[2] = {m > 1 ? k_row_stride : D, m > 1 ? v_row_stride : D};
  const int64_t hs[2] = {KV > 1 ? k_head_stride : 0, KV > 1 ? v_head_stride : 0};
  for (int i = 0; i < 2; ++i) {
    if (rs[i] < D || hs[i] < 0) return fail(W8A8_EINVAL, "%s: row strides smaller than head_dim, or negative", what);
    if (rs[i] % 8 || hs[i] % 8) return fail(W8A8_EALIGN, "%s: strides must be multiples of 8 elements", what);
  }
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)n_dev % 4)
    return fail(W8A8_EALIGN, "%s: k and v 16-byte, the position 4-byte aligned", what);
  AppendParams p{};
  block_layout(cache, KV, capacity, D, p.c);
  p.k = k; p.khs = hs[0]; p.krs = rs[0]; p.v = v; p.vhs = hs[1]; p.vrs = rs[1];
  p.m = int(m); p.n = int(n_dev ? 0 : n); p.capacity = int(capacity); p.n_dev = n_dev;
  // blocks touched, whatever the position if it is in device memory
  const int64_t blocks = n_dev ? (m + BLK - 2) / BLK + 1 : (n + m - 1) / BLK - n / BLK + 1;
  const dim3 grid{unsigned(blocks), unsigned(KV), 2};
  switch (int(D) + (e4m3 ? 1 : 0)) {
    case 128: block_append_kernel<128, false><<<grid, 256, 0, stream>>>(p); break;
    case 129: block_append_kernel<128, true><<<grid, 256, 0, stream>>>(p); break;
    case 256: block_append_kernel<256, false><<<grid, 256, 0, stream>>>(p); break;
    case 257: block_append_kernel<256, true><<<grid, 256, 0, stream>>>(p); break;
    case 512: block_append_kernel<512, false><<<grid, 256, 0, stream>>>(p); break;
    default: block_append_kernel<512, true><<<grid, 256, 0, stream>>>(p);
  }
  return check_launch(what);
}

extern "C" int w8a8_block_read(const void* cache, int64_t KV, int64_t capacity, int64_t D, int e4m3, int64_t start,
                               int64_t n, uint16_t* k, uint16_t* v, hipStream_t stream) {
  const char* what = "block_read";
  if (int rc = block_check(what, cache, KV, capacity, D)) return rc;
  if (start < 0 || n < start || n > capacity)
    return fail(W8A8_EINVAL, "%s: rows %lld .. %lld of a cache of %lld", what, (long long)start, (long long)n, (long long)capacity);
  if (start == n) return W8A8_OK;
  if (!k || !v) return fail(W8A8_EINVAL, "%s: null pointer", what);
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16) return fail(W8A8_EALIGN, "%s: k and v must be 16-byte aligned", what);
  ReadParams p{};
  block_layout(const_cast<void*>(cache), KV, capacity, D, p.c);
  p.k = k; p.v = v; p.start = int(start); p.n = int(n);
  const dim3 grid{unsigned((n - 1) / BLK - start / BLK + 1), unsigned(KV), 2};
  switch (int(D) + (e4m3 ? 1 : 0)) {
    case 128: block_read_kernel<128, false><<<grid, 256, 0, stream>>>(p); break;
    case 129: block_read_kernel<128, true><<<grid, 256, 0, stream>>>(p); break;
    case 256: block_read_kernel<256, false><<<grid, 256, 0, stream>>>(p); break;
    case 257: block_read_kernel<256, true><<<grid, 256, 0, stream>>>(p); break;
    case 512: block_read_kernel<512, false><<<grid, 256, 0, stream>>>(p); break;
    default: block_read_kernel<512, true><<<grid, 256, 0, stream>>>(p);
  }
  return check_launch(what);
}
