// The attention weight that keys have drawn, summed over queries and the heads of their KV head:
//
//   w[g, j] += sum_{h in g} sum_{i sees j} exp(scale * q[h, i] . k[g, j] - lse[h, i]),
//
// with the logsumexp that the attention call returned, so that each term is that call's softmax weight.  It
// is what a bounded cache keeps its rows by.  The reference has no counterpart (its cache grows with the
// sequence, local_attn.py:44-107); the views are its causal and sliding ones (pipeline.py:140-180).
//
// One product, S^T = K Q^T on the bf16 MFMA with the keys as the A operand: a lane's accumulator column is
// then one query, whose logsumexp is one register, and the sum over queries stays in the lane until the
// end, when 16 lanes are added.  No atomics: a key's sum is made by one workgroup, or (long prompts) by one
// per part of the queries, and the parts are added in order, so the result does not depend on timing.
//
// A term is exp2(s c - lse log2 e), c = scale log2 e held in two parts, both above 0: rounded to one, c's error would
// be the same sign for all keys (6e-8 of |s c|); the others are half a step of the argument, either way.
#include <algorithm>
#include <cmath>

#include "attn_common.h"

namespace w8a8 {

struct KeyWeightParams {
  const uint16_t* q; int64_t qhs, qrs;  // bf16 [H, Tq, D]
  const uint16_t* k; int64_t khs, krs;  // bf16 [KV, Tk, D]
  const float* lse; int64_t lhs;        // fp32 [H, Tq]
  float* w; int64_t whs;                // fp32 [KV, Tk]
  const int32_t* start_dev;             // q_start in device memory, or null: start
  int start, KV, G, Tq, Tk, window;
  int key0;                             // first key of the launch
  float* part; int nparts, len;         // [nparts][KV][keys] partial sums of a split launch; row blocks per part
  int keys, nkb;                        // keys from key0 on, and blocks of them
  float c, c_lo;                        // scale * log2(e) = c + c_lo
};

// log2 of a term: s c - lse log2 e, given minus the latter.
__device__ __forceinline__ float key_weight_log2(float s, float c, float c_lo, float nl2) {
  return __builtin_fmaf(s, c, __builtin_fmaf(s, c_lo, nl2));
}
// -lse log2 e.  +inf is a query that saw nothing and adds nothing: its terms are masked like keys that it does not see, for
// its scores may be NaN (padding that holds anything, or past the last query zeros times an infinite key).
__device__ __forceinline__ float key_weight_ref(float lse) { return -lse * 1.4426950408889634f; }

// v summed over the 16 lanes of a group (every lane gets the sum).
__device__ __forceinline__ float lanes16_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Few rows (a decoded token's heads): a wave takes 16 keys, whose rows it reads once from memory straight
// into the MFMA's A operand, and all RT row tiles.
template <int D, int RT>
__global__ __launch_bounds__(256) void key_weights_few_kernel(KeyWeightParams p) {
  constexpr int NKK = D / 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int qi = lane & 15, qq = lane >> 4;
  const int g = blockIdx.y;
  const int start = p.start_dev ? max(0, min(*p.start_dev, p.Tk - p.Tq)) : p.start;
  const int end = start + p.Tq;                                     // keys at or past it are seen by no query
  const int first = p.window > 0 ? max(0, start - p.window + 1) : 0;
  const int kb = (p.start_dev ? first : p.key0) + (int(blockIdx.x) * 4 + wave) * 16;
  if (kb >= end) return;
  const int nk = min(16, end - kb);
  const uint32_t krs2 = uint32_t(p.krs) * 2u;
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.k + int64_t(g) * p.khs + int64_t(kb) * p.krs,
                                              uint32_t(nk - 1) * krs2 + uint32_t(D) * 2u);
  v8bf kf[NKK];
#pragma unroll
  for (int kk = 0; kk < NKK; ++kk)
    kf[kk] = __builtin_bit_cast(v8bf, buf_load16(rk, uint32_t(qi) * krs2 + uint32_t(32 * kk + 8 * qq) * 2u));
  // lane qi = e of group qq adds key 4 qq + e: its weight so far is asked for with the keys
  float* const wp = p.w + int64_t(g) * p.whs + kb + 4 * qq + qi;
  const bool mine = qi < 4 && 4 * qq + qi < nk;
  const float before = mine ? *wp : 0.0f;
  const int rows = p.Tq * p.G;
  float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = 16 * t + qi;
    const bool valid = r < rows;
    const int i = valid ? r / p.G : 0, h = g * p.G + (valid ? r % p.G : 0);
    const uint16_t* qp = p.q + int64_t(h) * p.qhs + int64_t(i) * p.qrs + 8 * qq;
    const float nl2 = valid ? key_weight_ref(p.lse[int64_t(h) * p.lhs + i]) : __builtin_inff();
    v4f s0 = v4f{0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      v4i x = v4i{0, 0, 0, 0};
      if (valid) x = *reinterpret_cast<const v4i*>(qp + 32 * kk);
      const v8bf b = __builtin_bit_cast(v8bf, x);
      if (kk & 1)
        s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kk], b, s1, 0, 0, 0);
      else
        s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kk], b, s0, 0, 0, 0);
    }
    const int pos = nl2 != __builtin_inff() ? start + i : -1;  // (before every key)
    const uint32_t wlim = p.window > 0 ? uint32_t(p.window) : 0x80000000u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = kb + 4 * qq + e;
      const bool vis = uint32_t(pos - key) < wlim;
      w[e] += __builtin_amdgcn_exp2f(attn_mask(key_weight_log2(s0[e] + s1[e], p.c, p.c_lo, nl2), vis));
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = lanes16_sum(w[e]);
  if (mine) *wp = before + (qi < 2 ? (qi == 0 ? w[0] : w[1]) : (qi == 2 ? w[2] : w[3]));
}

// Many rows (prompts).  A wave holds 16 KT keys in registers as A operands for the whole launch, the waves of
// a workgroup 256; the queries of one head after the other pass through a two-slot LDS ring in blocks of QB
// consecutive positions, each fragment read once per wave, KR of them ahead, and fed to KT MFMAs.  A part is a
// run of (position block, head) pairs among those that see the key block.  At head_dim 512 eight waves of 32
// keys, two a SIMD, whose products and exponentials overlap, beat four of 64 with half the LDS reads:
// 205 -> 66 us for 3658 tokens of 8 heads (832 TFLOP/s; a large library product reaches 1210), 268 us for 8192
// (1024 TFLOP/s).  The LDS reads of the queries (as many cycles as the products) and the first load of the keys
// bound it.
template <int D>
struct KeyWeightShape {
  static constexpr int QB = D == 128 ? 64 : 32;
  static constexpr int KB = 256;
  static constexpr int KT = D == 512 ? 2 : 4;
  static constexpr int NW = KB / (16 * KT);
  static constexpr int KR = 8;
  static constexpr int SLOT = QB * D * 2;
};
constexpr int key_weight_threads(int d) { return d == 512 ? 512 : 256; }

// Position blocks that see keys [kb, kb + 256): first and one past the last.
template <int QB>
__host__ __device__ inline void key_weight_range(int kb, int start, int Tq, int window, int& lo, int& hi) {
  const int a = kb - start, n = (Tq + QB - 1) / QB;
  lo = a > 0 ? a / QB : 0;
  hi = n;
  if (window > 0) {
    const int64_t z = int64_t(a) + 255 + window;  // positions start + z and later see none of them
    hi = z <= 0 ? 0 : int(z < Tq ? (z + QB - 1) / QB : n);
  }
  if (hi < lo) hi = lo;
}

template <int D>
__global__ __launch_bounds__(key_weight_threads(D), D == 512 ? 1 : 2) void key_weights_kernel(KeyWeightParams p) {
  using S = KeyWeightShape<D>;
  constexpr int QB = S::QB, NKK = D / 32, KCH = D / 8, ROW = D * 2, KT = S::KT, NW = S::NW, KR = S::KR, KEYS = 16 * KT;
  constexpr int U = QB * KCH / (NW * 64);  // DMA instructions per thread per block
  static_assert(NW * 64 == key_weight_threads(D) && U * NW * 64 == QB * KCH, "tiling");
  __shared__ __attribute__((aligned(1024))) char lds[2 * S::SLOT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 15, qq = lane >> 4;
  // workgroup x of KV head g: part x of the first key block's, or what is left of the next ones'
  const int g = blockIdx.x % p.KV;
  int part = blockIdx.x / p.KV, b = 0, lo, hi, total, np;
  for (;; ++b) {
    key_weight_range<QB>(p.key0 + b * S::KB, p.start, p.Tq, p.window, lo, hi);
    total = (hi - lo) * p.G;
    np = max(1, (total + p.len - 1) / p.len);
    if (part < np) break;
    part -= np;
    if (b + 1 >= p.nkb) return;  // (never: the grid is the sum of the key blocks' parts)
  }
  const int kb = p.key0 + b * S::KB, kw = kb + wave * KEYS;  // this workgroup's and wave's keys
  const int n0 = int(int64_t(part) * total / np), n1 = int(int64_t(part + 1) * total / np);

  const int end = min(p.start + p.Tq, p.Tk);
  const int nk = max(0, min(KEYS, end - kw));
  const uint32_t krs2 = uint32_t(p.krs) * 2u, qrs2 = uint32_t(p.qrs) * 2u;
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.k + int64_t(g) * p.khs + int64_t(nk > 0 ? kw : 0) * p.krs,
                                              nk > 0 ? uint32_t(nk - 1) * krs2 + uint32_t(ROW) : 0u);
  uint32_t qoff[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int xc = (u * NW + wave) * 64 + lane;
    const int row = xc / KCH, cs = xc % KCH;
    qoff[u] = uint32_t(row) * qrs2 + uint32_t(cs ^ (row & 15)) * 16u;
  }
  float ln[QB / 16];  // the next block's lse of this lane's queries
  auto fetch = [&](int n) __attribute__((always_inline)) {
    const int i0 = (lo + n / p.G) * QB, h = g * p.G + n % p.G;
    const __amdgpu_buffer_rsrc_t rq = make_rsrc(p.q + int64_t(h) * p.qhs + int64_t(i0) * p.qrs,
                                                uint32_t(min(QB, p.Tq - i0) - 1) * qrs2 + uint32_t(ROW));
    char* base = lds + ((n - n0) & 1) * S::SLOT;
#pragma unroll
    for (int u = 0; u < U; ++u) attn_dma16(rq, base + (u * NW + wave) * 1024, qoff[u]);
#pragma unroll
    for (int t = 0; t < QB / 16; ++t) {
      const int i = i0 + 16 * t + qi;
      ln[t] = i < p.Tq ? p.lse[int64_t(h) * p.lhs + i] : -__builtin_inff();
    }
  };
  if (n0 < n1) fetch(n0);
  v8bf kf[KT][NKK];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk)
      kf[t][kk] = __builtin_bit_cast(
          v8bf, buf_load16(rk, uint32_t(16 * t + qi) * krs2 + uint32_t(32 * kk + 8 * qq) * 2u));
  float w[KT][4] = {};
  const uint32_t wlim = p.window > 0 ? uint32_t(p.window) : 0x80000000u;
  const float c = p.c, c_lo = p.c_lo;
  uint32_t qofs[4];  // this lane's fragment kk of a row lies at qofs[kk % 4] + 256 (kk / 4)
#pragma unroll
  for (int j = 0; j < 4; ++j) qofs[j] = uint32_t(qi * ROW + ((4 * j + qq) ^ qi) * 16);
  for (int n = n0; n < n1; ++n) {
    attn_wait_vmcnt<0>();
    __syncthreads();  // block n is in LDS; the other slot is free
    float nl2[QB / 16];
#pragma unroll
    for (int t = 0; t < QB / 16; ++t) nl2[t] = key_weight_ref(ln[t]);
    if (n + 1 < n1) fetch(n + 1);
    const char* base = lds + ((n - n0) & 1) * S::SLOT;
    const int p0 = p.start + (lo + n / p.G) * QB;  // the block's first position
    const bool none = kw > p0 + QB - 1 || (p.window > 0 && int64_t(kw) + KEYS - 1 <= int64_t(p0) - p.window);
    if (none) continue;
    float most = nl2[0];
#pragma unroll
    for (int t = 1; t < QB / 16; ++t) most = fmaxf(most, nl2[t]);
    const bool whole = kw + KEYS - 1 <= p0 && (p.window <= 0 || kw > p0 + QB - 1 - p.window) &&
                       __builtin_amdgcn_ballot_w64(most == __builtin_inff()) == 0;
    auto qfrag = [&](int i) __attribute__((always_inline)) {  // fragment kk = i % NKK of row tile i / NKK
      const int kk = i % NKK;
      return *reinterpret_cast<const v8bf*>(base + qofs[kk % 4] + (kk / 4) * 256 + (i / NKK) * (16 * ROW));
    };
    v8bf qf[KR];
#pragma unroll
    for (int i = 0; i < KR; ++i) qf[i] = qfrag(i);
#pragma unroll
    for (int rt = 0; rt < QB / 16; ++rt) {
      v4f s[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) s[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
        const int i = rt * NKK + kk;
#pragma unroll
        for (int t = 0; t < KT; ++t) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][kk], qf[i % KR], s[t], 0, 0, 0);
        if (i + KR < QB / 16 * NKK) qf[i % KR] = qfrag(i + KR);
      }
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = key_weight_log2(s[t][e], c, c_lo, nl2[rt]);
      if (!whole) {
        const int pos = nl2[rt] != __builtin_inff() ? p0 + 16 * rt + qi : -1;  // (before every key)
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[t][e] = attn_mask(s[t][e], uint32_t(pos - (kw + 16 * t + 4 * qq + e)) < wlim);
      }
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) w[t][e] += __builtin_amdgcn_exp2f(s[t][e]);
    }
  }
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) w[t][e] = lanes16_sum(w[t][e]);
  // lane qi = 4 t + e of group qq holds key 16 t + 4 qq + e
  float v = 0.0f;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) v = qi == 4 * t + e ? w[t][e] : v;
  const int j = 16 * (qi >> 2) + 4 * qq + (qi & 3);
  if (j >= nk) return;
  if (p.nparts > 1)
    p.part[(int64_t(part) * p.KV + g) * p.keys + (kw - p.key0) + j] = v;
  else
    p.w[int64_t(g) * p.whs + kw + j] += v;
}

// Adds the parts of each key to its weight, in order.
template <int QB>
__global__ __launch_bounds__(256) void key_weights_add_kernel(KeyWeightParams p) {
  const int j = blockIdx.x * 256 + threadIdx.x, g = blockIdx.y;  // (a workgroup is one key block)
  if (j >= p.keys) return;
  int lo, hi;
  key_weight_range<QB>(p.key0 + int(blockIdx.x) * 256, p.start, p.Tq, p.window, lo, hi);
  const int np = max(1, ((hi - lo) * p.G + p.len - 1) / p.len);
  float* wp = p.w + int64_t(g) * p.whs + p.key0 + j;
  const float* pp = p.part + int64_t(g) * p.keys + j;
  const int64_t step = int64_t(p.KV) * p.keys;
  float v = 0.0f;
  for (int s0 = 0; s0 < np; s0 += 16) {  // 16 loads in flight
    float x[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) x[u] = s0 + u < np ? pp[(s0 + u) * step] : 0.0f;
#pragma unroll
    for (int u = 0; u < 16; ++u) v += x[u];
  }
  *wp += v;
}

// ---- host ----------------------------------------------------------------------------------------

constexpr int KEYW_FEW = 32;  // rows of the kernel that reads the queries from memory

struct KeyWeightPlan {
  bool few;
  int key0, keys, nkb, nparts, len;
  int64_t wgs;  // parts of all key blocks
};

static int64_t key_weight_total(const KeyWeightPlan& pl, int64_t D, int64_t G, int64_t start, int64_t Tq, int64_t window,
                                int len, int* most) {
  int64_t n = 0;
  *most = 1;
  for (int b = 0; b < pl.nkb; ++b) {
    int lo, hi;
    if (D == 128)
      key_weight_range<64>(pl.key0 + b * 256, int(start), int(Tq), int(window), lo, hi);
    else
      key_weight_range<32>(pl.key0 + b * 256, int(start), int(Tq), int(window), lo, hi);
    const int64_t np = std::max<int64_t>(1, ((hi - lo) * G + len - 1) / len);
    n += np;
    *most = int(std::max<int64_t>(*most, np));
  }
  return n;
}

static KeyWeightPlan key_weight_plan(int64_t H, int64_t KV, int64_t Tq, int64_t D, int64_t start, int64_t window) {
  KeyWeightPlan pl{};
  const int64_t G = H / KV;
  pl.key0 = int(window > 0 && start - window + 1 > 0 ? start - window + 1 : 0);
  pl.keys = int(start + Tq - pl.key0);
  pl.few = Tq * G <= KEYW_FEW;
  pl.nkb = (pl.keys + 255) / 256;
  pl.nparts = 1;
  pl.len = 1;
  pl.wgs = pl.nkb;
  if (pl.few) return pl;
  // Parts of so many row blocks that they fill the chip in whole rounds, each paying its keys' load (about
  // four row blocks' time).  (The grid holds no workgroup without work: with empty ones between them an XCD
  // got more than its CUs' share and the call took two rounds, 133 us for 3658 tokens of 8 heads of 512.)
  const int64_t slots = int64_t(attn_cu_count()) * (D == 512 ? 1 : 2);
  int most;
  const int64_t total = key_weight_total(pl, D, G, start, Tq, window, 1, &most) * KV;
  int64_t best = INT64_MAX;
  for (int64_t rounds = 1; rounds <= 6; ++rounds) {
    int64_t len = std::max<int64_t>(1, total / (rounds * slots)), n;
    for (;; len += 1 + len / 32) {
      n = key_weight_total(pl, D, G, start, Tq, window, int(len), &most) * KV;
      if (n <= rounds * slots || n == int64_t(pl.nkb) * KV) break;
    }
    const int64_t cost = (n + slots - 1) / slots * (len + 4);
    if (cost < best) best = cost, pl.len = int(len), pl.nparts = most, pl.wgs = n / KV;
  }
  return pl;
}

}  // namespace w8a8

using namespace w8a8;

static bool key_weight_shape_ok(int64_t H, int64_t KV, int64_t Tq, int64_t Tk, int64_t D, int64_t window) {
  return H >= 1 && KV >= 1 && H % KV == 0 && H <= (1 << 16) && KV <= 65535 && Tq >= 1 && Tk >= Tq &&
         Tk <= INT32_MAX / 2 && window >= 0 && window <= INT32_MAX / 2 && (D == 128 || D == 256 || D == 512);
}

extern "C" int64_t w8a8_attention_key_weights_workspace_bytes(int64_t H, int64_t KV, int64_t Tq, int64_t Tk, int64_t D,
                                                              int64_t q_start, int64_t window) {
  if (!key_weight_shape_ok(H, KV, Tq, Tk, D, window) || q_start < -1 || q_start > Tk - Tq) return -1;
  if (q_start < 0) return Tq * (H / KV) <= KEYW_FEW ? 0 : -1;
  const KeyWeightPlan pl = key_weight_plan(H, KV, Tq, D, q_start, window);
  return pl.nparts > 1 ? int64_t(pl.nparts) * KV * pl.keys * 4 : 0;
}

template <int D>
static void key_weight_launch(KeyWeightParams& p, const KeyWeightPlan& pl, int64_t keys, hipStream_t stream) {
  if (pl.few) {
    const dim3 grid{unsigned((keys + 63) / 64), unsigned(p.KV), 1};
    if (p.Tq * p.G <= 16)
      key_weights_few_kernel<D, 1><<<grid, 256, 0, stream>>>(p);
    else
      key_weights_few_kernel<D, 2><<<grid, 256, 0, stream>>>(p);
    return;
  }
  key_weights_kernel<D><<<dim3{unsigned(pl.wgs * p.KV), 1, 1}, key_weight_threads(D), 0, stream>>>(p);
  if (pl.nparts > 1)
    key_weights_add_kernel<KeyWeightShape<D>::QB><<<dim3{unsigned(pl.nkb), unsigned(p.KV), 1}, 256, 0, stream>>>(p);
}

extern "C" int w8a8_attention_key_weights(const uint16_t* q, int64_t q_head_stride, int64_t q_row_stride,
                                          const uint16_t* k, int64_t k_head_stride, int64_t k_row_stride,
                                          const float* lse, int64_t lse_head_stride, int64_t H, int64_t KV, int64_t Tq,
                                          int64_t Tk, int64_t D, int64_t q_start, const int32_t* q_start_dev,
                                          int64_t window, float scale, float* weights, int64_t weights_head_stride,
                                          void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const char* what = "attention_key_weights";
  if (D != 128 && D != 256 && D != 512)
    return fail(W8A8_ENOTSUP, "%s: head_dim %lld (supported: 128, 256, 512)", what, (long long)D);
  if (!key_weight_shape_ok(H, KV, Tq, Tk, D, window))
    return fail(W8A8_EINVAL, "%s: H=%lld KV=%lld Tq=%lld Tk=%lld window=%lld", what, (long long)H, (long long)KV,
                (long long)Tq, (long long)Tk, (long long)window);
  if (q_start_dev ? q_start != -1 : (q_start < 0 || q_start > Tk - Tq))
    return fail(W8A8_EINVAL, "%s: q_start=%lld (0 .. Tk - Tq = %lld, or -1 with q_start_dev)", what, (long long)q_start,
                (long long)(Tk - Tq));
  if (q_start_dev && Tq * (H / KV) > KEYW_FEW)
    return fail(W8A8_ENOTSUP, "%s: a position in device memory takes at most %d rows (queries x heads) per KV head", what,
                KEYW_FEW);
  if (!(scale > 0.0f) || scale == __builtin_inff()) return fail(W8A8_EINVAL, "%s: scale must be positive", what);
  if (!q || !k || !lse || !weights) return fail(W8A8_EINVAL, "%s: null pointer", what);
  const int64_t need = w8a8_attention_key_weights_workspace_bytes(H, KV, Tq, Tk, D, q_start, window);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(W8A8_EINVAL, "%s: workspace of %lld bytes, %lld needed", what, (long long)(workspace ? workspace_bytes : 0),
                (long long)need);
  const int64_t rs[2] = {Tk > 1 ? k_row_stride : D, Tq > 1 ? q_row_stride : D};
  const int64_t hs[2] = {KV > 1 ? k_head_stride : 0, H > 1 ? q_head_stride : 0};
  for (int i = 0; i < 2; ++i) {
    if (rs[i] < D || hs[i] < 0) return fail(W8A8_EINVAL, "%s: row strides smaller than head_dim, or negative", what);
    if (rs[i] % 8 != 0 || hs[i] % 8 != 0) return fail(W8A8_EALIGN, "%s: strides must be multiples of 8 elements", what);
    if (rs[i] * 2 * 64 >= INT32_MAX) return fail(W8A8_ENOTSUP, "%s: row stride %lld", what, (long long)rs[i]);
  }
  if ((H > 1 && lse_head_stride < Tq) || (KV > 1 && weights_head_stride < Tk))
    return fail(W8A8_EINVAL, "%s: strides of lse or weights smaller than their rows", what);
  if ((uintptr_t)q % 16 || (uintptr_t)k % 16 || (uintptr_t)lse % 4 || (uintptr_t)weights % 4 || (uintptr_t)workspace % 4 ||
      (uintptr_t)q_start_dev % 4)
    return fail(W8A8_EALIGN, "%s: q and k 16-byte, the others 4-byte aligned", what);
  KeyWeightParams p{};
  p.q = q; p.qhs = hs[1]; p.qrs = rs[1]; p.k = k; p.khs = hs[0]; p.krs = rs[0]; p.lse = lse;
  p.lhs = H > 1 ? lse_head_stride : 0; p.w = weights; p.whs = KV > 1 ? weights_head_stride : 0;
  p.start_dev = q_start_dev; p.start = int(std::max<int64_t>(q_start, 0)); p.KV = int(KV); p.G = int(H / KV);
  p.Tq = int(Tq); p.Tk = int(Tk); p.window = int(window);
  const double c = double(scale) * 1.4426950408889634;
  // c rounded down and c_lo above 0: with parts of either sign, or a c_lo of 0, a score of -inf would make NaN
  p.c = float(c);
  if (double(p.c) > c) p.c = std::nextafter(p.c, 0.0f);
  p.c_lo = std::max(float(c - double(p.c)), p.c * 0x1p-60f);
  const KeyWeightPlan pl = key_weight_plan(H, KV, Tq, D, p.start, window);
  p.key0 = pl.key0; p.keys = pl.keys; p.nkb = pl.nkb; p.nparts = pl.nparts; p.len = pl.len;
  p.part = static_cast<float*>(workspace);
  // the keys a launch covers: those seen, or with a position in device memory as many as any position sees
  const int64_t keys = !q_start_dev ? pl.keys : window > 0 ? std::min(window - 1 + Tq, Tk) : Tk;
  if (D == 128)
    key_weight_launch<128>(p, pl, keys, stream);
  else if (D == 256)
    key_weight_launch<256>(p, pl, keys, stream);
  else
    key_weight_launch<512>(p, pl, keys, stream);
  return check_launch("attention_key_weights");
}
