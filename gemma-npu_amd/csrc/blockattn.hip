// Attention over the 8-bit key / value cache (blocks.h): the newest N of n tokens attend to it, causal, with a sliding
// window and the first tokens beside it if wanted.
//
//   o[h, i, :] = sum_j softmax_j(scale q[h, i] . k[g, j]) v[g, j],   g = h / (H / KV),
//
// over the rows j that the query at position p = n - N + i sees: j <= p and, with a window W, p - j < W or j < sinks.
// Row j is code x scale of its block, or the bf16 row of the ring for the n % 64 rows behind the last whole block.
//
// A key's scale leaves its product with q as a factor of the score.  A value's scale t enters the softmax weight as
// an exponent: P'_j = exp2(s_j + log2 t - ms), and sum_j exp2(s_j - ms) = sum P'_j / t is added up in fp32 beside it.
// ms lies 7 below a value that trails the maximum of s_j + log2 t by at most 8: P' is at most 2^15, and what contributes
// most has the most bits.  Codes become fp16 exactly (|code| <= 127, e4m3 lies within fp16), so both products are fp16
// MFMAs summed in fp32.  The roundings: P' to fp16 (2^-11; subnormal below 2^-14, off by 2^-32 of the row's largest, where
// the codes of the largest's block are off by 2^-8 of that block's values), and q, scaled by a power of two that brings its
// row's largest value to 2^10 (exact but for values below 2^-27 of that).  The rows of the ring go through bf16 MFMAs
// with P' in bf16 (2^-8).
//
// A block whose value scale is far below the largest so far, by more than 2^8, would have its P' among fp16's
// subnormals, and one value far out in a block leaves its other columns to such blocks alone.  So ms is lowered for it, by
// what its scale lies below the largest, 2^46 at most, or to 7 below its own maximum if that is higher; sums and outputs are
// rescaled in fp32, as where the maximum grows.  (Of 2^30 rows the sums stay below 2^(30 + 15 + 36 + 46), the outputs far
// below.)  Scales further apart than 2^46 cost the smaller one's weights a bit for every factor of two.
//
// Work split.  The rows (query, head) of one KV head, N G of them, are cut into tiles of 16 RT rows and their visible
// blocks into parts; a workgroup takes a tile and a part, and a second kernel joins the parts by their logsumexp.  In each
// group of four waves wave w makes S^T = K Q^T of the group's rows for a block's keys 16 w .. 16 w + 15; all waves split
// head_dim for O^T.  The softmax weights go through LDS, with one barrier a block.  Keys and values come straight from
// memory in fragment order into registers, one to four blocks ahead: no LDS, no transposing.
//
// One token of 8 KV heads of 128 over 65521 rows (134 MB of codes): 31 us, 4.8 TB/s once the blocks flow.  One of a head of 512
// over 3659 rows: 7.7 us, of which the queries' way into registers is 3, a block and its products 2.  5 queries of 8 heads of
// 512 over 32749 rows: 19.7 us.  509 queries of 8 heads of 256 over a window of 4096 (17 GFLOP): 47 us, 2.2 a block of 64 rows, whose
// S, softmax and P V follow one another in the two waves of a SIMD.
#include <algorithm>
#include <type_traits>

#include "attn_common.h"
#include "attn_parts.h"
#include "blocks.h"

namespace w8a8 {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

struct BlockAttnParams {
  BlockCache c;
  const uint16_t* q; int64_t qhs, qrs;  // bf16 [H, N, D] (element strides, last dim contiguous)
  PartParams out;                       // o, lse, parts, rows
  const int32_t* n_dev;                 // n in device memory, or null
  int n, N, window, sinks, capacity, ntiles;
  float cs;                             // scale * log2(e)
};

// The blocks that a tile's rows see: i < nb stands for block i, from `sb` on for block i + skip.
struct BlockGeom {
  int n, pmin, pmax, sb, skip, nb, np;
};
__device__ __forceinline__ BlockGeom block_geom(const BlockAttnParams& p, int tile, int R) {
  BlockGeom t;
  t.n = p.n_dev ? max(p.N, min(*p.n_dev, p.capacity)) : p.n;
  const int r0 = tile * R, r1 = min(r0 + R, p.out.rows) - 1;
  t.pmin = t.n - p.N + r0 / p.out.G;
  t.pmax = t.n - p.N + r1 / p.out.G;
  const int wb = p.window > 0 ? max(0, t.pmin - p.window + 1) / BLK : 0;
  t.sb = (min(p.sinks, t.n) + BLK - 1) / BLK;
  t.skip = max(0, wb - t.sb);
  t.nb = t.pmax / BLK + 1 - t.skip;
  t.np = min(p.out.nparts, t.nb);
  return t;
}

// Four codes as fp16: int8 through 1024 + code + 128, whose low byte is the code's with its sign bit turned.
template <bool E4M3>
__device__ __forceinline__ void codes_f16(uint32_t w, v2h& a, v2h& b) {
  if constexpr (E4M3) {
    a = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    b = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  } else {
    const uint32_t x = w ^ 0x80808080u;
    const v2h bias = {_Float16(1152.0f), _Float16(1152.0f)};
    a = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias;
    b = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias;
  }
}
template <bool E4M3>
__device__ __forceinline__ v8h codes8_f16(uint32_t lo, uint32_t hi) {
  v2h a, b, c, d;
  codes_f16<E4M3>(lo, a, b);
  codes_f16<E4M3>(hi, c, d);
  return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Row groups of a workgroup's waves (four waves each), workgroups of a CU, and blocks on their way in a wave's registers.
// From 32 rows on two groups hold half of the queries each and an eighth of head_dim of all rows' outputs.
constexpr int block_groups(int rt) { return rt == 1 ? 1 : 2; }
constexpr int block_occupancy(int rt, int d) { return rt > 1 ? 1 : d == 128 ? 3 : 2; }
constexpr int block_ahead(int rt, int d) { return d == 128 ? (rt <= 2 ? 4 : 2) : d == 256 && rt <= 4 ? 2 : 1; }

template <int D, int RT, bool E4M3>
__global__ __launch_bounds__(256 * block_groups(RT), block_groups(RT) * block_occupancy(RT, D)) void block_attn_kernel(BlockAttnParams p) {
  constexpr int R = 16 * RT, RG = block_groups(RT), NW = 4 * RG, RW = RT / RG;  // row tiles of a wave's S phase
  constexpr int NK = D / 64, NV = D / 16 / NW, NKK = D / 32;                    // a wave's fragments of keys, of values; k-steps
  constexpr int PLD = BLK + 8;                                                  // padded row of softmax weights
  __shared__ __attribute__((aligned(16))) uint16_t qs[R * D];  // the tile's queries, chunk c of row r at c ^ (r & 15)
  __shared__ __attribute__((aligned(16))) uint16_t pl[2][R * PLD];
  __shared__ float smax[2][4][R], alpha_s[2][R], lsum[4][R], cqs[R];
  __shared__ int flag_s[2][8];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 15, qq = lane >> 4;
  const int kt = wave & 3, r0 = 16 * RW * (wave >> 2);  // this wave's key tile and first row in the S phase
  const int G = p.out.G, rows = p.out.rows;
  const int lb = xcd_remap(blockIdx.x, gridDim.x);
  const int tile = lb % p.ntiles, pair = lb / p.ntiles, g = pair / p.out.nparts, part = pair % p.out.nparts;
  const BlockGeom geo = block_geom(p, tile, R);
  if (part >= geo.np) return;  // (the whole workgroup, before any barrier)
  const int i_lo = int(int64_t(part) * geo.nb / geo.np), i_hi = int(int64_t(part + 1) * geo.nb / geo.np);
  const int whole = geo.n / BLK;  // blocks with codes
  // Row r of the tile is query `first + t / G` and head t % G of the group, t = odd + r < 2^17: a quotient that fp32 has exactly
  // (an integer division is some forty instructions, which are waited for one cache line at a time).
  const int first = tile * R / G, odd = tile * R - first * G;
  const float per = 1.0f / float(G);
  auto query = [&](int r) __attribute__((always_inline)) { return int((float(odd + r) + 0.5f) * per); };  // less `first`
  auto block = [&](int i) __attribute__((always_inline)) { return i < geo.sb ? i : i + geo.skip; };
  const bool has_ring = block(i_hi - 1) >= whole;  // the part's last block is the unfinished one
  const int ncode = i_hi - i_lo - (has_ring ? 1 : 0);
  const int win = p.window, sinks = p.sinks;

  // Blocks' keys and values on their way in registers, PF of each, with their scales
  constexpr int PF = block_ahead(RT, D);
  const int64_t head = int64_t(g) * p.c.blocks;
  const uint8_t* const kc = p.c.k + head * BLK * D + kt * (16 * D) + lane * 16;
  const uint8_t* const vc = p.c.v + head * BLK * D + wave * (NV * 1024) + lane * 16;
  v4u kr[PF][NK], vr[PF][NV];
  float ksr[PF], vsr[PF];
  auto load_k = [&](int u, int i) __attribute__((always_inline)) {
    const int b = block(i);
    const uint8_t* at = kc + int64_t(b) * (BLK * D);
#pragma unroll
    for (int j = 0; j < NK; ++j) kr[u][j] = *reinterpret_cast<const v4u*>(at + j * 1024);
    // (vector loads, which are waited for in order: a scalar one would stall the block that needs it)
    ksr[u] = p.c.ks[head + b + (lane >> 6)];
    vsr[u] = p.c.vs[head + b + (lane >> 6)];
  };
  auto load_v = [&](int u, int i) __attribute__((always_inline)) {
    const uint8_t* at = vc + int64_t(block(i)) * (BLK * D);
#pragma unroll
    for (int j = 0; j < NV; ++j) vr[u][j] = *reinterpret_cast<const v4u*>(at + j * 1024);
  };

  // The tile's queries, asked for before the keys and values, whose arrival their conversion hides: a wave takes
  // R / NW rows, D / 8 lanes a row.
  constexpr int LPR = D / 8, RPI = 64 / LPR, NI = R / NW / RPI;  // lanes of a row, rows at a time, times
  auto staged = [&](int i) __attribute__((always_inline)) { return wave * (R / NW) + i * RPI + lane / LPR; };
  auto place = [&](int r) __attribute__((always_inline)) {
    return reinterpret_cast<v4u*>(qs + r * D + 8 * ((lane % LPR) ^ (r & 15)));
  };
  v4u qw[NI];
  auto ask_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = staged(i), x = query(r), h = odd + r - x * G;
      qw[i] = v4u{0u, 0u, 0u, 0u};
      if (tile * R + r < rows)
        qw[i] = *reinterpret_cast<const v4u*>(p.q + int64_t(g * G + h) * p.qhs + int64_t(first + x) * p.qrs + 8 * (lane % LPR));
    }
  };
  auto put_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NI; ++i) *place(staged(i)) = qw[i];
  };
  ask_q();
  __builtin_amdgcn_sched_barrier(0);
  if (ncode > 0) load_k(0, i_lo);
#pragma unroll
  for (int u = 0; u < PF; ++u) {  // in the order of their use
    if (u + 1 < PF && u + 1 < ncode) load_k(u + 1, i_lo + u + 1);
    if (u < ncode) load_v(u, i_lo + u);
  }
  __builtin_amdgcn_sched_barrier(0);
  int pos[RW];  // of this lane's rows r0 + 16 rt + qi
#pragma unroll
  for (int rt = 0; rt < RW; ++rt) {
    const int r = r0 + 16 * rt + qi;
    pos[rt] = tile * R + r < rows ? geo.n - p.N + first + query(r) : -1;  // (sees nothing)
  }
  put_q();
  // .. made fp16 in their places (a short loop: what such a kernel waits for first is its own instructions)
#pragma unroll 2
  for (int i = 0; i < NI; ++i) {
    const int r = staged(i);
    const v4u w = *place(r);
    uint32_t m2 = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) m2 = absmax_bf16x2(m2, w[e]);
    float top = absmax_pair(m2);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top = absmax2(top, __shfl_xor(top, o, 64));
    // 2^10 over the power of two at or below `top` (no smaller than 2^-87: zeros)
    const uint32_t e = max(__float_as_uint(top) >> 23, 40u);
    const float f = __uint_as_float((264u - e) << 23);
    v4u h;
#pragma unroll
    for (int j = 0; j < 4; ++j)  // (exact but for subnormals, whose rounding towards zero is below 2^-24 of 2^10)
      h[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(w[j] << 16) * f,
                                                                     __uint_as_float(w[j] & 0xffff0000u) * f));
    *place(r) = h;
    if (lane % LPR == 0) cqs[r] = p.cs * __uint_as_float((e - 10u) << 23);
  }
  __syncthreads();
  // .. and read as the B operand of k-step 2 j + h: q[64 j + 16 qq + 8 h .. + 7], which is how the codes lie
  // (where registers are short three quarters of them stay in LDS)
  constexpr int NQ = 4 * (RW * NKK + NV * RT) > 180 ? NKK / 4 : NKK;
  v8h qf[RW][NQ];
  auto frag = [&](int rt, int k) __attribute__((always_inline)) {
    return *reinterpret_cast<const v4u*>(qs + (r0 + 16 * rt + qi) * D + 8 * ((8 * (k >> 1) + 2 * qq + (k & 1)) ^ qi));
  };
  float cq[RW];  // what a score of the row is multiplied by
#pragma unroll
  for (int rt = 0; rt < RW; ++rt) {
#pragma unroll
    for (int k = 0; k < NQ; ++k) qf[rt][k] = __builtin_bit_cast(v8h, frag(rt, k));
    cq[rt] = cqs[r0 + 16 * rt + qi];
  }

  // A row's exponent that its weights and sums are held against, the largest score's that it follows, and its sum.
  float ms[RW], mt[RW], l[RW];
#pragma unroll
  for (int rt = 0; rt < RW; ++rt) ms[rt] = mt[rt] = -__builtin_inff(), l[rt] = 0.0f;
  v4f o[NV][RT];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) o[j][rt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

  v4f s[RW];
  float tb = 0.0f, tinv = 1.0f;  // log2 of the block's value scale, and one over the scale
  float tmax = -__builtin_inff(), low = 0.0f;  // the largest so far, and how far below it this one lies, if it is far
  const uint32_t near = win > 0 ? uint32_t(win) : 0x80000000u;
  auto seen = [&](int key, int at) __attribute__((always_inline)) {  // (compares alone: a branch here is one per score)
    return (uint32_t(at - key) < near) | ((key <= at) & (key < sinks));
  };
  auto inner = [&](int b) __attribute__((always_inline)) {  // every row sees the whole block
    const int kb = b * BLK;
    return kb + BLK - 1 <= geo.pmin && (win <= 0 || kb > geo.pmax - win || kb + BLK <= sinks) && tile * R + R <= rows;
  };
  // scores in exponents (log2), masked; this wave's row maxima into LDS
  auto finish_s = [&](int slot, int b, float ks, bool codes) __attribute__((always_inline)) {
    const bool all = inner(b);
#pragma unroll
    for (int rt = 0; rt < RW; ++rt) {
      const float f = codes ? ks * cq[rt] : p.cs;
#pragma unroll
      for (int i = 0; i < 4; ++i) s[rt][i] = __builtin_fmaf(s[rt][i], f, tb);
    }
    if (!all)
#pragma unroll
      for (int rt = 0; rt < RW; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[rt][i] = attn_mask(s[rt][i], seen(b * BLK + 16 * kt + 4 * qq + i, pos[rt]));
#pragma unroll
    for (int rt = 0; rt < RW; ++rt) {
      const float bm = lanes4_max(fmaxf(fmaxf(s[rt][0], s[rt][1]), fmaxf(s[rt][2], s[rt][3])));
      if (qq == 0) smax[slot][kt][r0 + 16 * rt + qi] = bm;
    }
  };
  auto s_phase = [&](int slot, int u, int i) __attribute__((always_inline)) {
    const float ks = ksr[u], vs = vsr[u];
    tb = __builtin_amdgcn_logf(vs);
    tinv = 1.0f / vs;
    low = tmax - tb > 8.0f ? fminf(tmax - tb, 46.0f) : 0.0f;  // (a block that reads NaN has no part in this)
    tmax = tb < __builtin_inff() ? fmaxf(tmax, tb) : tmax;
    constexpr int NS = RW == 1 ? 2 : 1;  // one row tile: two chains of products
    v4f acc[NS][RW];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int rt = 0; rt < RW; ++rt) acc[n][rt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const v8h a = codes8_f16<E4M3>(kr[u][j][2 * h], kr[u][j][2 * h + 1]);
#pragma unroll
        for (int rt = 0; rt < RW; ++rt) {
          const v8h q = 2 * j + h < NQ ? qf[rt][(2 * j + h) % NQ] : __builtin_bit_cast(v8h, frag(rt, 2 * j + h));
          acc[h % NS][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q, acc[h % NS][rt], 0, 0, 0);
        }
      }
#pragma unroll
    for (int rt = 0; rt < RW; ++rt) {
      s[rt] = acc[0][rt];
      if constexpr (NS == 2) s[rt] += acc[1][rt];
    }
    finish_s(slot, block(i), ks, true);
  };
  // after the barrier: the rows' new references and P' into LDS, with what O is rescaled by
  auto softmax = [&](int slot, auto half) __attribute__((always_inline)) {
    bool grew = false;
#pragma unroll
    for (int rt = 0; rt < RW; ++rt) {
      const int r = r0 + 16 * rt + qi;
      const float m = fmaxf(fmaxf(smax[slot][0][r], smax[slot][1][r]), fmaxf(smax[slot][2][r], smax[slot][3][r]));
      mt[rt] = m > mt[rt] + 8.0f ? m : mt[rt];  // (-inf while every key so far is masked)
      const float to = __builtin_amdgcn_fmed3f(mt[rt] - 7.0f - low, m - 7.0f, mt[rt] - 7.0f);
      const bool moved = to != ms[rt], had = ms[rt] != -__builtin_inff();
      const float alpha = !moved ? 1.0f : (had ? __builtin_amdgcn_exp2f(ms[rt] - to) : 0.0f);
      grew |= moved && had;
      ms[rt] = to;
      const float ref = ms[rt] == -__builtin_inff() ? 0.0f : ms[rt];
      float sum = 0.0f;
      uint16_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[rt][i] - ref);
        sum += e;
        if constexpr (decltype(half)::value)
          w[i] = __builtin_bit_cast(uint16_t, _Float16(e));
        else
          w[i] = f32_to_bf16(e);
      }
      // (a block that a row sees nothing of adds nothing, whatever its scale)
      l[rt] = __builtin_fmaf(sum, sum != 0.0f ? tinv : 0.0f, l[rt] * alpha);
      // key 16 kt + 4 qq + i is slot 4 (kt % 2) + i of lane group qq in k-step kt / 2
      *reinterpret_cast<v2u*>(&pl[slot][r * PLD + 32 * (kt >> 1) + 8 * qq + 4 * (kt & 1)]) =
          v2u{uint32_t(w[0]) | uint32_t(w[1]) << 16, uint32_t(w[2]) | uint32_t(w[3]) << 16};
      if (kt == 0 && qq == 0) alpha_s[slot][r] = alpha;
    }
    const bool any = __builtin_amdgcn_ballot_w64(grew) != 0;
    if (kt == 0 && lane == 0) flag_s[slot][wave >> 2] = any ? 1 : 0;
  };
  auto rescale = [&](int slot) __attribute__((always_inline)) {
    int f = flag_s[slot][0];
    if constexpr (RG == 2) f |= flag_s[slot][1];
    if (f != 0)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float a = alpha_s[slot][16 * rt + qi];
#pragma unroll
        for (int j = 0; j < NV; ++j) o[j][rt] *= a;
      }
  };
  auto weights = [&](int slot, int rt, int h) __attribute__((always_inline)) {
    return *reinterpret_cast<const v4u*>(&pl[slot][(16 * rt + qi) * PLD + 32 * h + 8 * qq]);
  };
  auto pv_phase = [&](int slot, int u) __attribute__((always_inline)) {
    rescale(slot);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      v8h a[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) a[j] = codes8_f16<E4M3>(vr[u][j][2 * h], vr[u][j][2 * h + 1]);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const v8h pb = __builtin_bit_cast(v8h, weights(slot, rt, h));
#pragma unroll
        for (int j = 0; j < NV; ++j) o[j][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], pb, o[j][rt], 0, 0, 0);
      }
    }
  };
  using Yes = std::true_type;
  using No = std::false_type;

  // Block i's scores and maxima are made one iteration ahead of its P V: the barrier between them makes the maxima of
  // block i + 1 and the weights of block i visible at once.
  if (ncode > 0) {
    s_phase(0, 0, i_lo);
    if (PF < ncode) load_k(0, i_lo + PF);
    __syncthreads();
    softmax(0, Yes{});
    for (int x0 = 0; x0 < ncode; x0 += PF)
#pragma unroll
      for (int u = 0; u < PF; ++u) {
        const int x = x0 + u, slot = x & 1;
        if (x >= ncode) break;
        const bool more = x + 1 < ncode;
        if (more) {
          s_phase(slot ^ 1, (u + 1) % PF, i_lo + x + 1);
          if (x + 1 + PF < ncode) load_k((u + 1) % PF, i_lo + x + 1 + PF);
        }
        __syncthreads();
        pv_phase(slot, u);
        if (x + PF < ncode) load_v(u, i_lo + x + PF);
        if (more) softmax(slot ^ 1, Yes{});
      }
  }

  if (has_ring) {
    // the unfinished block: bf16 rows, of which the first `live` are there, against the queries in bf16
    const int b = whole, live = geo.n - whole * BLK, slot = ncode & 1;
    const uint16_t* const rk = p.c.kt + (int64_t(g) * 2 + (b & 1)) * BLK * D + (kt * NKK * 64 + lane) * 8;
    const uint16_t* const rv = p.c.vt + (int64_t(g) * 2 + (b & 1)) * BLK * D + (wave * NV * 2 * 64 + lane) * 8;
    ask_q();
    v4u vw[NV][2];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) vw[j][h] = *reinterpret_cast<const v4u*>(rv + (2 * j + h) * 512);
    put_q();
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RW; ++rt) s[rt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (16 * kt < live) {
#pragma unroll 8
      for (int k = 0; k < NKK; ++k) {
        const v8bf a = *reinterpret_cast<const v8bf*>(rk + k * 512);
#pragma unroll
        for (int rt = 0; rt < RW; ++rt)
          s[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(v8bf, frag(rt, k)), s[rt], 0, 0, 0);
      }
    }
    tb = 0.0f;
    tinv = 1.0f;
    low = 0.0f;  // (weights in bf16, whose range is that of fp32)
    finish_s(slot, b, 1.0f, false);  // (rows from `live` on lie behind every position)
    // values of rows that aren't there are zero, infinities and NaN (0 x inf) leave the product and are added below to
    // the rows that see them
    uint32_t bad = 0u;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = 32 * h + 16 * (e >> 1) + 4 * qq + 2 * (e & 1);  // of the word's low half
        const uint32_t there = (key < live ? 0xffffu : 0u) | (key + 1 < live ? 0xffff0000u : 0u);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          vw[j][h][e] &= there;
          bad |= (vw[j][h][e] & 0x7f807f80u) + 0x00800080u;
        }
      }
    const bool any = __builtin_amdgcn_ballot_w64((bad & 0x80008000u) != 0u) != 0;
    if (any)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = ((vw[j][h][e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
            vw[j][h][e] &= ~((x >> 15) * 0xffffu);
          }
    __syncthreads();
    softmax(slot, No{});
    __syncthreads();
    rescale(slot);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const v8bf pb = __builtin_bit_cast(v8bf, weights(slot, rt, h));
#pragma unroll
        for (int j = 0; j < NV; ++j)
          o[j][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, vw[j][h]), pb, o[j][rt], 0, 0, 0);
      }
    if (any) {
      const uint16_t* const vt = p.c.vt + (int64_t(g) * 2 + (b & 1)) * BLK * D;
#pragma unroll 1
      for (int key = 0; key < live; ++key)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = uint32_t(vt[ring_value(key, 16 * (wave * NV + j) + 4 * qq + i)]) << 16;
            if ((x & 0x7f800000u) != 0x7f800000u) continue;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const int r = 16 * rt + qi;
              if (tile * R + r < rows && seen(b * BLK + key, geo.n - p.N + first + query(r))) o[j][rt][i] += __uint_as_float(x);
            }
          }
    }
  }

  // the rows' sums over the waves' keys
#pragma unroll
  for (int rt = 0; rt < RW; ++rt) {
    const float x = lanes4_sum(l[rt]);
    if (qq == 0) {
      lsum[kt][r0 + 16 * rt + qi] = x;
      if (kt == 0) cqs[r0 + 16 * rt + qi] = ms[rt];
    }
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = 16 * rt + qi, row = tile * R + r, d = wave * (16 * NV) + 4 * qq;  // + 16 j + i
    const float lt = (lsum[0][r] + lsum[1][r]) + (lsum[2][r] + lsum[3][r]);
    if (row >= rows) continue;
    if (geo.np > 1) {
      const int64_t at = (int64_t(g) * p.out.nparts + part) * rows + row;
#pragma unroll
      for (int j = 0; j < NV; ++j) *reinterpret_cast<v4f*>(p.out.part_o + at * D + d + 16 * j) = o[j][rt];
      if (wave == 0 && qq == 0) *reinterpret_cast<v2f*>(p.out.part_ml + at * 2) = v2f{cqs[r], lt};
      continue;
    }
    const float inv = lt > 0.0f ? 1.0f / lt : (lt == lt ? 0.0f : lt);  // (a NaN sum stays one)
    const int x = query(r), h = g * G + odd + r - x * G;
    uint16_t* const op = p.out.o + int64_t(h) * p.out.ohs + int64_t(first + x) * p.out.ors + d;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      *reinterpret_cast<v2u*>(op + 16 * j) =
          inv != 0.0f ? v2u{pack_bf16x2(o[j][rt][0] * inv, o[j][rt][1] * inv), pack_bf16x2(o[j][rt][2] * inv, o[j][rt][3] * inv)}
                      : v2u{0u, 0u};
    if (p.out.lse && wave == 0 && qq == 0) p.out.lse[int64_t(h) * p.N + first + x] = part_lse(cqs[r], lt);
  }
}

template <int D>
__global__ __launch_bounds__(256) void block_merge_kernel(BlockAttnParams p, int R) {
  const int row = blockIdx.x % p.out.rows;
  part_merge<D>(p.out, block_geom(p, row / R, R).np, p.N);
}
template <int D>
__global__ __launch_bounds__(256) void block_merge_few_kernel(BlockAttnParams p, int R) {
  part_merge_few<D>(p.out, [&](int row) { return block_geom(p, row / R, R).np; }, p.N);
}

// ---- host ----------------------------------------------------------------------------------------

struct BlockPlan {
  int rt, ntiles, nparts;
};

static BlockPlan block_plan(int64_t H, int64_t KV, int64_t N, int64_t n, int64_t D, int64_t window, int64_t sinks) {
  const int64_t rows = N * (H / KV);
  BlockPlan pl;
  pl.rt = rows <= 16 ? 1 : rows <= 32 ? 2 : D >= 256 || rows <= 64 ? 4 : 8;
  pl.ntiles = int((rows + 16 * pl.rt - 1) / (16 * pl.rt));
  // the blocks of a tile
  const int64_t span = window > 0 ? std::min<int64_t>(n, window + 16 * pl.rt / (H / KV) + 1 + BLK) / BLK + 1 + (std::min(sinks, n) + BLK - 1) / BLK
                                  : (n + BLK - 1) / BLK;
  const int64_t nb = std::min<int64_t>(span, (n + BLK - 1) / BLK);
  const int64_t cus = attn_cu_count();
  const int64_t want = std::max<int64_t>(1, cus * block_occupancy(pl.rt, int(D)) / (pl.ntiles * KV));
  pl.nparts = int(std::min<int64_t>({want, nb, PART_MAX}));
  return pl;
}

template <int D, bool E4M3>
static void block_launch(const BlockAttnParams& p, const BlockPlan& pl, hipStream_t stream) {
  const dim3 grid{unsigned(pl.ntiles) * unsigned(p.out.KV) * unsigned(p.out.nparts), 1, 1};
  switch (pl.rt) {
    case 1: block_attn_kernel<D, 1, E4M3><<<grid, 256, 0, stream>>>(p); break;
    case 2: block_attn_kernel<D, 2, E4M3><<<grid, 512, 0, stream>>>(p); break;
    case 4: block_attn_kernel<D, 4, E4M3><<<grid, 512, 0, stream>>>(p); break;
    default:
      if constexpr (D == 128) block_attn_kernel<D, 8, E4M3><<<grid, 512, 0, stream>>>(p);
  }
  if (p.out.nparts > PART_FEW)
    block_merge_kernel<D><<<dim3{unsigned(p.out.KV) * unsigned(p.out.rows), unsigned(D / 64), 1}, 256, 0, stream>>>(p, 16 * pl.rt);
  else if (p.out.nparts > 1)
    block_merge_few_kernel<D><<<part_few_grid<D>(p.out), 256, 0, stream>>>(p, 16 * pl.rt);
}

static bool block_attn_shape_ok(int64_t H, int64_t KV, int64_t N, int64_t capacity, int64_t D, int64_t window, int64_t sinks) {
  return block_shape_ok(KV, capacity, D) && H >= 1 && H <= (1 << 16) && H % KV == 0 && N >= 1 && N <= capacity && N * H < (int64_t(1) << 28) &&
         window >= 0 && window <= INT32_MAX / 2 && sinks >= 0 && sinks <= INT32_MAX / 2;
}

}  // namespace w8a8

using namespace w8a8;

extern "C" int64_t w8a8_block_attention_workspace_bytes(int64_t H, int64_t KV, int64_t N, int64_t capacity, int64_t D,
                                                        int64_t n, int64_t window, int64_t sinks) {
  if (!block_attn_shape_ok(H, KV, N, capacity, D, window, sinks) || n < -1 || n > capacity || (n >= 0 && n < N)) return -1;
  const BlockPlan pl = block_plan(H, KV, N, n < 0 ? capacity : n, D, window, sinks);
  return pl.nparts > 1 ? H * N * pl.nparts * (D + 2) * 4 : 0;
}

extern "C" int w8a8_block_attention(const uint16_t* q, int64_t q_head_stride, int64_t q_row_stride, const void* cache,
                                    int64_t H, int64_t KV, int64_t N, int64_t capacity, int64_t D, int e4m3, int64_t n,
                                    const int32_t* n_dev, int64_t window, int64_t sinks, float scale, uint16_t* o,
                                    int64_t o_head_stride, int64_t o_row_stride, float* lse, void* workspace,
                                    int64_t workspace_bytes, hipStream_t stream) {
  const char* what = "block_attention";
  if (D != 128 && D != 256 && D != 512)
    return fail(W8A8_ENOTSUP, "%s: head_dim %lld (supported: 128, 256, 512)", what, (long long)D);
  if (!block_attn_shape_ok(H, KV, N, capacity, D, window, sinks))
    return fail(W8A8_EINVAL, "%s: H=%lld KV=%lld N=%lld capacity=%lld window=%lld sinks=%lld", what, (long long)H, (long long)KV,
                (long long)N, (long long)capacity, (long long)window, (long long)sinks);
  if (n_dev ? n != -1 : (n < N || n > capacity))
    return fail(W8A8_EINVAL, "%s: n=%lld (N .. capacity, or -1 with a length in device memory)", what, (long long)n);
  if (!(scale > 0.0f) || scale == __builtin_inff()) return fail(W8A8_EINVAL, "%s: scale must be positive", what);
  if (!q || !cache || !o) return fail(W8A8_EINVAL, "%s: null pointer", what);
  const int64_t need = w8a8_block_attention_workspace_bytes(H, KV, N, capacity, D, n, window, sinks);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(W8A8_EINVAL, "%s: workspace of %lld bytes, %lld needed", what, (long long)(workspace ? workspace_bytes : 0),
                (long long)need);
  const int64_t rs[2] = {N > 1 ? q_row_stride : D, N > 1 ? o_row_stride : D};
  const int64_t hs[2] = {H > 1 ? q_head_stride : 0, H > 1 ? o_head_stride : 0};
  for (int i = 0; i < 2; ++i) {
    if (rs[i] < D || hs[i] < 0) return fail(W8A8_EINVAL, "%s: row strides smaller than head_dim, or negative", what);
    if (rs[i] % 8 != 0 || hs[i] % 8 != 0) return fail(W8A8_EALIGN, "%s: strides must be multiples of 8 elements", what);
  }
  if (H > 1 && o_head_stride < D) return fail(W8A8_EINVAL, "%s: o's heads overlap, stride %lld", what, (long long)o_head_stride);
  if ((uintptr_t)q % 16 || (uintptr_t)cache % 16 || (uintptr_t)o % 16 || (uintptr_t)workspace % 16 || (uintptr_t)n_dev % 4 ||
      (uintptr_t)lse % 4)
    return fail(W8A8_EALIGN, "%s: q, o, the cache and the workspace 16-byte, n and lse 4-byte aligned", what);
  const BlockPlan pl = block_plan(H, KV, N, n_dev ? capacity : n, D, window, sinks);
  BlockAttnParams p{};
  block_layout(const_cast<void*>(cache), KV, capacity, D, p.c);
  p.q = q; p.qhs = hs[0]; p.qrs = rs[0];
  p.out.o = o; p.out.ohs = hs[1]; p.out.ors = rs[1]; p.out.lse = lse; p.out.KV = int(KV); p.out.G = int(H / KV);
  p.out.rows = int(N * (H / KV)); p.out.nparts = pl.nparts;
  p.out.part_o = static_cast<float*>(workspace);
  p.out.part_ml = p.out.part_o + H * N * pl.nparts * D;
  p.n_dev = n_dev; p.n = int(std::max<int64_t>(n, 0)); p.N = int(N); p.window = int(window); p.sinks = window > 0 ? int(sinks) : 0;
  p.capacity = int(capacity); p.ntiles = pl.ntiles;
  p.cs = scale * 1.4426950408889634f;
  switch (int(D) + (e4m3 ? 1 : 0)) {
    case 128: block_launch<128, false>(p, pl, stream); break;
    case 129: block_launch<128, true>(p, pl, stream); break;
    case 256: block_launch<256, false>(p, pl, stream); break;
    case 257: block_launch<256, true>(p, pl, stream); break;
    case 512: block_launch<512, false>(p, pl, stream); break;
    default: block_launch<512, true>(p, pl, stream);
  }
  return check_launch(what);
}
