// Parts of an attention row's keys, computed by different workgroups and joined by their logsumexp.
#pragma once
#include "attn_common.h"

namespace w8a8 {

constexpr int PART_MAX = 512;

struct PartParams {
  uint16_t* o; int64_t ohs, ors;  // bf16 [H, N, D]
  float* lse;                     // fp32 [H, N], or null
  int KV, G, rows, nparts;        // rows (query, head) of a KV head; parts at most
  float* part_o;                  // [KV][nparts][rows][D] unnormalised sums
  float* part_ml;                 // [KV][nparts][rows][2] reference exponent (log2) and sum
};

// Natural-log logsumexp from the reference exponent and the sum against it: -inf where nothing was seen.
__device__ __forceinline__ float part_lse(float m, float l) {
  return l > 0.0f ? m * 0.69314718055994531f + __logf(l) : (l == l ? -__builtin_inff() : l);
}

// Joins the np parts of row blockIdx.x: M = max m_s, w_s = exp2(m_s - M), o = sum_s w_s o_s / sum_s w_s l_s.  A
// workgroup of 256 takes 64 columns (blockIdx.y): thread t sums column group t % 16 over parts t / 16, + 16, ..,
// eight loads in flight, and the 16 sums are added in order (the same result whatever the timing).
template <int D>
__device__ __forceinline__ void part_merge(const PartParams& p, int np, int N) {
  __shared__ float wsh[PART_MAX];
  __shared__ v4f sums[256];
  __shared__ float red[4][2];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int g = blockIdx.x / p.rows, row = blockIdx.x % p.rows;
  if (np <= 1) return;  // the attention kernel wrote the row
  const int64_t base = int64_t(g) * p.nparts * p.rows + row;  // part s at base + s * rows
  const v2f* ml = reinterpret_cast<const v2f*>(p.part_ml) + base;
  float mx = -__builtin_inff();
  for (int s = t; s < np; s += 256) mx = fmaxf(mx, ml[int64_t(s) * p.rows][0]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (lane == 0) red[wave][0] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
  const float mref = mx == -__builtin_inff() ? 0.0f : mx;
  float L = 0.0f;
  for (int s = t; s < np; s += 256) {
    const v2f v = ml[int64_t(s) * p.rows];
    const float w = __builtin_amdgcn_exp2f(v[0] - mref);
    wsh[s] = w;
    L = __builtin_fmaf(w, v[1], L);
  }
  L = wave_sum(L);
  if (lane == 0) red[wave][1] = L;
  __syncthreads();
  L = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
  const int col = blockIdx.y * 64 + 4 * (t & 15), p0 = t >> 4;
  const float* po = p.part_o + base * D + col;
  v4f acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (int s0 = p0; s0 < np; s0 += 128) {
    v4f v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + 16 * u;
      v[u] = s < np ? *reinterpret_cast<const v4f*>(po + int64_t(s) * p.rows * D) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int s = s0 + 16 * u;
      const float w = s < np ? wsh[s] : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(w, v[u][i], acc[i]);
    }
  }
  sums[t] = acc;
  __syncthreads();
  if (t >= 16) return;
#pragma unroll
  for (int s = 1; s < 16; ++s) acc += sums[16 * s + t];
  const int i = row / p.G, h = g * p.G + row % p.G;
  const float inv = L > 0.0f ? 1.0f / L : (L == L ? 0.0f : L);
  v2u w = v2u{0u, 0u};
  if (inv != 0.0f) {
    w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  }
  *reinterpret_cast<v2u*>(p.o + int64_t(h) * p.ohs + int64_t(i) * p.ors + col) = w;
  if (p.lse && col == 0) p.lse[int64_t(h) * N + i] = part_lse(mx, L);
}

// The same for calls of at most PART_FEW parts, many rows as a rule: a thread takes four columns of a row.
constexpr int PART_FEW = 8;
template <int D, class NP>
__device__ __forceinline__ void part_merge_few(const PartParams& p, NP parts_of, int N) {
  constexpr int T = D / 4;  // threads of a row
  const int64_t at = int64_t(blockIdx.x) * (256 / T) + threadIdx.x / T;
  if (at >= int64_t(p.KV) * p.rows) return;
  const int g = int(at / p.rows), row = int(at % p.rows), col = 4 * (threadIdx.x % T), np = parts_of(row);
  if (np <= 1) return;
  const int64_t base = int64_t(g) * p.nparts * p.rows + row;
  const v2f* ml = reinterpret_cast<const v2f*>(p.part_ml) + base;
  const float* po = p.part_o + base * D + col;
  v2f st[PART_FEW];
  v4f v[PART_FEW];
#pragma unroll
  for (int s = 0; s < PART_FEW; ++s) st[s] = s < np ? ml[int64_t(s) * p.rows] : v2f{-__builtin_inff(), 0.0f};
#pragma unroll
  for (int s = 0; s < PART_FEW; ++s)
    v[s] = s < np ? *reinterpret_cast<const v4f*>(po + int64_t(s) * p.rows * D) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
  float mx = -__builtin_inff();
#pragma unroll
  for (int s = 0; s < PART_FEW; ++s) mx = fmaxf(mx, st[s][0]);
  const float ref = mx == -__builtin_inff() ? 0.0f : mx;
  float L = 0.0f;
  v4f acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int s = 0; s < PART_FEW; ++s) {
    const float w = __builtin_amdgcn_exp2f(st[s][0] - ref);
    L = __builtin_fmaf(w, st[s][1], L);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(w, v[s][i], acc[i]);
  }
  const int i = row / p.G, h = g * p.G + row % p.G;
  const float inv = L > 0.0f ? 1.0f / L : (L == L ? 0.0f : L);
  v2u w = v2u{0u, 0u};
  if (inv != 0.0f) {
    w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  }
  *reinterpret_cast<v2u*>(p.o + int64_t(h) * p.ohs + int64_t(i) * p.ors + col) = w;
  if (p.lse && col == 0) p.lse[int64_t(h) * N + i] = part_lse(mx, L);
}
template <int D>
inline dim3 part_few_grid(const PartParams& p) {
  const int64_t per = 256 / (D / 4);
  return dim3{unsigned((int64_t(p.KV) * p.rows + per - 1) / per), 1, 1};
}

}  // namespace w8a8
