// Attention of drafted tokens over a cache: the queries are nodes of a tree whose keys and values stand
// behind the context's in the cache.
//
//   o[h, i, :] = sum_j softmax_j(scale * q[h, i] . k[g, j]) v[g, j],   g = h / (H / KV),
//
// over the rows j that node i sees: the context's n_past rows and, of the M nodes' rows n_past + m, its
// own and those above it in the tree (parents[m] in -1 .. m - 1, -1: the context's last token); with a
// window W only rows whose position is less than W before the node's, a node's position being n_past +
// its depth.  The queries are the last N of the M nodes, so a tree can be attended to level by level.
// A node with a parent outside -1 .. m - 1 is unused: it and the nodes below it see nothing, and their
// outputs are zero.  The reference decodes one token at a time (local_attn.py:44-83); this is that step
// for many candidate tokens at once.
//
// Work split.  The rows (node, head) of one KV head, N x G of them, are cut into tiles of 16 RT rows, and
// the keys into parts; a workgroup takes one tile and one part, so that few rows over a long cache still
// fill the chip, and attn_tree_merge_kernel joins the parts by their logsumexp.  The tiles of one part
// run next to each other on one XCD and share its L2's copy of the keys.
//
// Within a workgroup the key blocks pass through a two-slot LDS ring (buffer_load ... lds, K one block
// further ahead than V), one barrier per block: iteration n makes S^T = K Q^T and the softmax of block
// n + 1 and multiplies P V of block n.  The first RT waves own 16 rows' S phase each (the others wait: the
// keys' way through memory is what bounds small tiles), every wave D / NW columns of O^T in the P V phase,
// its V^T operand read from the row-major V rows with ds_read_b64_tr_b16.
// Scores, softmax and sums are fp32; the softmax weights are rounded to bf16 for the second product, at
// most 2^-8 of each weight, as the other attention kernels do.
//
// Values a row does not see never reach it: in the blocks that some row sees only in part (those at the
// window's edge and the tree's own) infinities and NaN in V are replaced by zeros before the MFMA, whose
// 0 * inf would be NaN, and added at the end to the rows that do see them.
#include <algorithm>
#include <type_traits>

#include "attn_common.h"

namespace w8a8 {

constexpr int TREE_MAX_NODES = 128;   // M, so that a node's view of the tree is four words
constexpr int TREE_WORDS = TREE_MAX_NODES / 32;
constexpr int TREE_MAX_PARTS = 512;

struct TreeParams {
  const uint16_t* q; int64_t qhs, qrs;  // bf16 [H, N, D] (element strides, last dim contiguous)
  const uint16_t* k; int64_t khs, krs;  // bf16 [KV, Tk, D]
  const uint16_t* v; int64_t vhs, vrs;
  uint16_t* o; int64_t ohs, ors;        // bf16 [H, N, D]
  float* lse;                           // fp32 [H, N], or null
  const int32_t* parents;               // [M]
  const int32_t* past_dev;              // n_past in device memory, or null: past
  int past;
  int KV, G, N, M, Tk, window;
  int rows, ntiles, nparts;             // N G rows, tiles of them, parts of the keys (at most)
  float* part_o;                        // [KV][nparts][rows][D] unnormalised sums
  float* part_ml;                       // [KV][nparts][rows][2] reference exponent and sum
  float c;                              // scale * log2(e)
};

// The call's context length, first key, key blocks and live parts.  A length in device memory outside
// 0 .. Tk - M is the caller's error: it is brought into that range, so nothing outside the cache is read.
struct TreeGeom {
  int past, klo, nblk, nparts;
};
template <int BN>
__device__ __forceinline__ TreeGeom tree_geom(const TreeParams& p) {
  TreeGeom t;
  t.past = p.past_dev ? max(0, min(*p.past_dev, p.Tk - p.M)) : p.past;
  t.klo = p.window > 0 ? max(0, t.past - p.window + 1) : 0;
  t.nblk = (t.past + p.M - t.klo + BN - 1) / BN;
  t.nparts = min(p.nparts, t.nblk);
  return t;
}

// Waves of a workgroup.  At head_dim 512 a tile of 64 rows has eight too, four of which have no rows of their own in
// the S phase: half of O^T per wave leaves the registers for a variable per slot (64 nodes over 32749 rows 91 -> 75 us).
constexpr int tree_waves(int rt, int d) { return rt > 4 || (d == 512 && rt == 4) ? 8 : 4; }

template <int D, int RT>
struct TreeShape {
  static constexpr int NW = tree_waves(RT, D);
  static constexpr int NT = NW * 64;
  static constexpr int BN = D == 128 ? 64 : 32;      // keys per block
  static constexpr int R = RT * 16;                  // rows per tile
  static constexpr int KCH = D / 8;                  // 16-byte chunks per K / V row
  static constexpr int ROW = D * 2;
  static constexpr int KV_SLOT = BN * ROW;
  static constexpr int PLD = BN + 8;                 // padded P row, elements
  static constexpr int P_SLOT = R * PLD * 2;
  static constexpr int A_OFF = 2 * P_SLOT;           // P [2]; ..
  static constexpr int F_OFF = A_OFF + 2 * R * 4;    // alpha [2][R]; flags [2][16], found [16]
  static constexpr int B_OFF = F_OFF + 3 * 16 * 4;   // the nodes' views [M][4]; depths [M]; chain ends [M]
  static constexpr int AUX = B_OFF + TREE_MAX_NODES * (TREE_WORDS + 2) * 4;
  static constexpr int NDW = D / NW / 16;            // 16-wide d tiles of O^T per wave
  static constexpr int KR = 3;                       // K fragments in flight
  static constexpr bool SPLIT = D < 512 || RT < 5;   // a variable per slot (the others would spill)
};

// The nodes' views of the tree into LDS: bits[m] = the nodes on m's chain (none: unused), depth[m].  Every
// chain's known length doubles each round (the bits of the node its known part ends at are added).
template <int NT>
__device__ __forceinline__ void tree_resolve(const int32_t* parents, int M, uint32_t* bits, int* depth, int* end) {
  const int m = threadIdx.x;
  const bool on = m < M;
  uint32_t b[TREE_WORDS] = {};
  int e = -1;
  if (on) {
    const int par = parents[m];
    e = par >= -1 && par < m ? par : -2;
#pragma unroll
    for (int w = 0; w < TREE_WORDS; ++w) {
      b[w] = (m >> 5) == w ? 1u << (m & 31) : 0u;
      bits[m * TREE_WORDS + w] = b[w];
    }
    end[m] = e;
  }
  __syncthreads();
  for (int known = 1; known < M; known *= 2) {
    int ne = e;
    if (on && e >= 0) {
#pragma unroll
      for (int w = 0; w < TREE_WORDS; ++w) b[w] |= bits[e * TREE_WORDS + w];
      ne = end[e];
    }
    __syncthreads();
    if (on && e >= 0) {
#pragma unroll
      for (int w = 0; w < TREE_WORDS; ++w) bits[m * TREE_WORDS + w] = b[w];
      end[m] = ne;
    }
    e = ne;
    __syncthreads();
  }
  if (on) {
    int n = -1;
#pragma unroll
    for (int w = 0; w < TREE_WORDS; ++w) {
      n += __popc(b[w]);
      if (e == -2) bits[m * TREE_WORDS + w] = 0u;
    }
    depth[m] = n;
  }
  __syncthreads();
}

template <int D, int RT>
__global__ __launch_bounds__(tree_waves(RT, D) * 64, 1) void attn_tree_kernel(TreeParams p) {
  using S = TreeShape<D, RT>;
  constexpr int NW = S::NW, NT = S::NT, BN = S::BN, R = S::R, KCH = S::KCH, ROW = S::ROW, PLD = S::PLD, NDW = S::NDW;
  constexpr int NKC = BN / 32;              // 32-key chunks per block
  constexpr int KU = BN * KCH / NT;         // DMA instructions per thread per K or V block
  constexpr int NKK = D / 32;               // k-steps of S^T
  static_assert(KU * NT == BN * KCH && NDW >= 1 && RT <= NW && NT >= TREE_MAX_NODES, "tiling");
  static_assert(4 * S::KV_SLOT + S::AUX <= 160 * 1024, "LDS");
  // With SPLIT every slot is a variable of its own: from one array the compiler has a read of V wait for all
  // the DMAs in flight, those into the other slot too, as it cannot tell the slots apart.
  constexpr bool SPLIT = S::SPLIT;
  __shared__ __attribute__((aligned(1024))) char k0[S::KV_SLOT], k1[S::KV_SLOT], v0[S::KV_SLOT], v1[S::KV_SLOT];
  __shared__ __attribute__((aligned(1024))) char aux_s[S::AUX];
  __shared__ __attribute__((aligned(1024))) char lds[4 * S::KV_SLOT + S::AUX];
  auto k_slot = [&](auto slot) __attribute__((always_inline)) -> char* {
    if constexpr (SPLIT) return slot ? k1 : k0;
    else return lds + slot * S::KV_SLOT;
  };
  auto v_slot = [&](auto slot) __attribute__((always_inline)) -> char* {
    if constexpr (SPLIT) return slot ? v1 : v0;
    else return lds + (2 + slot) * S::KV_SLOT;
  };
  char* aux;
  if constexpr (SPLIT) aux = aux_s;
  else aux = lds + 4 * S::KV_SLOT;
  float* const alpha_s = reinterpret_cast<float*>(aux + S::A_OFF);
  int* const flag_s = reinterpret_cast<int*>(aux + S::F_OFF);
  int* const found_s = flag_s + 32;
  uint32_t* const bits_s = reinterpret_cast<uint32_t*>(aux + S::B_OFF);
  int* const depth_s = reinterpret_cast<int*>(bits_s + TREE_MAX_NODES * TREE_WORDS);

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 15, qq = lane >> 4;

  // block b: XCD b % 8 runs the tiles of (KV head, part) pairs b % 8, b % 8 + 8, .. one after the other
  const TreeGeom geo = tree_geom<BN>(p);
  const int x = int(blockIdx.x) >> 3;
  const int pair = (x / p.ntiles) * 8 + (int(blockIdx.x) & 7), tile = x % p.ntiles;
  const int g = pair / p.nparts, part = pair % p.nparts;
  if (g >= p.KV || part >= geo.nparts) return;  // (the whole workgroup, before any barrier)
  const int past = geo.past, M = p.M, G = p.G, win = p.window;
  const int n_lo = int(int64_t(part) * geo.nblk / geo.nparts), n_hi = int(int64_t(part + 1) * geo.nblk / geo.nparts);
  const int kb0 = geo.klo + n_lo * BN, nblk = n_hi - n_lo;  // at least one block
  const bool last_part = part == geo.nparts - 1;

  // the part's keys as buffers of their own, so that a cache of any length has 32-bit offsets; rows past
  // the last node's read zero
  const int nkeys = min(nblk * BN, past + M - kb0);
  const uint32_t krs2 = uint32_t(p.krs) * 2u, vrs2 = uint32_t(p.vrs) * 2u;
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(p.k + int64_t(g) * p.khs + int64_t(kb0) * p.krs,
                                              uint32_t(nkeys - 1) * krs2 + uint32_t(ROW));
  const __amdgpu_buffer_rsrc_t rv = make_rsrc(p.v + int64_t(g) * p.vhs + int64_t(kb0) * p.vrs,
                                              uint32_t(nkeys - 1) * vrs2 + uint32_t(ROW));

  // K chunk x of row r lands at stored chunk x ^ swz(r), swz(r) = (r & 3) | ((r >> 1) & 12); V chunk x of
  // row r at x ^ 2 (r & 3)
  uint32_t koff[KU], voff[KU];
#pragma unroll
  for (int u = 0; u < KU; ++u) {
    const int xc = (u * NW + wave) * 64 + lane;
    const int row = xc / KCH, cs = xc % KCH;
    koff[u] = uint32_t(row) * krs2 + uint32_t(cs ^ ((row & 3) | ((row >> 1) & 12))) * 16u;
    voff[u] = uint32_t(row) * vrs2 + uint32_t(cs ^ (2 * (row & 3))) * 16u;
  }
  // block n goes to slot n % 2 (with SPLIT a type, so that each access names its slot's variable)
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 1>;
  auto issue_k = [&](auto slot, int n) __attribute__((always_inline)) {
    const uint32_t rowoff = uint32_t(n * BN) * krs2;
#pragma unroll
    for (int u = 0; u < KU; ++u) attn_dma16(rk, k_slot(slot) + (u * NW + wave) * 1024, rowoff + koff[u]);
  };
  auto issue_v = [&](auto slot, int n) __attribute__((always_inline)) {
    const uint32_t rowoff = uint32_t(n * BN) * vrs2;
#pragma unroll
    for (int u = 0; u < KU; ++u) attn_dma16(rv, v_slot(slot) + (u * NW + wave) * 1024, rowoff + voff[u]);
  };

  issue_k(Even{}, 0);
  issue_v(Even{}, 0);
  // Q (B operand: lane (qi, qq) holds q[row][32 kk + 8 qq .. + 7] of this wave's 16 rows)
  const int srow = 16 * (wave % RT) + qi;
  const int row = tile * R + srow;               // (node, head) row of the KV head
  const bool valid = row < p.rows;
  const int qnode = row / G, hl = row % G;
  v8bf qf[NKK];
  {
    const uint16_t* qp = p.q + int64_t(g * G + hl) * p.qhs + int64_t(qnode) * p.qrs + 8 * qq;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      v4i t = v4i{0, 0, 0, 0};
      if (valid) t = *reinterpret_cast<const v4i*>(qp + 32 * kk);
      qf[kk] = __builtin_bit_cast(v8bf, t);
    }
  }
  if (nblk > 1) issue_k(Odd{}, 1);

  // Block n is seen whole by every row when its keys are all context inside every node's window.
  auto inner = [&](int n) __attribute__((always_inline)) {
    const int kb = kb0 + n * BN;
    return kb + BN <= past && (win <= 0 || kb > past + M - 1 - win);
  };
  // A row's view of the tree's rows, where the part has blocks that are not seen whole: the nodes on its
  // chain, with a window those less than it deep below the node.
  auto view = [&](int r, uint32_t(&bits)[TREE_WORDS], int& depth) __attribute__((always_inline)) {
    const int m = M - p.N + r / G;
#pragma unroll
    for (int w = 0; w < TREE_WORDS; ++w) bits[w] = r < p.rows ? bits_s[m * TREE_WORDS + w] : 0u;
    depth = r < p.rows ? depth_s[m] : 0;
    if (win > 0 && win < M)
#pragma unroll
      for (int w = 0; w < TREE_WORDS; ++w)
        for (uint32_t left = bits[w]; left; left &= left - 1) {
          const int at = __builtin_ctz(left);
          if (depth - depth_s[32 * w + at] >= win) bits[w] &= ~(1u << at);
        }
  };
  uint32_t bits[TREE_WORDS] = {};
  int depth = 0;
  if (!inner(0) || !inner(nblk - 1)) {
    tree_resolve<NT>(p.parents, M, bits_s, depth_s, depth_s + TREE_MAX_NODES);
    view(row, bits, depth);
  }
  const bool live = (bits[0] | bits[1] | bits[2] | bits[3]) != 0u;
  // The keys kb .. kb + 31 that a row of this view and depth sees, as bits: its context rows (position below
  // `past`, within the window) and its nodes.
  auto seen = [&](const uint32_t(&b)[TREE_WORDS], int d, int kb) __attribute__((always_inline)) {
    auto word = [&](int w) { return w < 2 ? (w == 0 ? b[0] : b[1]) : w < 4 ? (w == 2 ? b[2] : b[3]) : 0u; };
    const int off = kb - past;  // the first key's node, or minus the context rows from it on
    uint32_t m = 0u;
    if (off >= 0)
      m = __builtin_amdgcn_alignbit(word((off >> 5) + 1), word(off >> 5), uint32_t(off & 31));
    else {
      const int n = -off;
      m = n < 32 ? (b[0] << n) | ((1u << n) - 1u) : ~0u;
      const int cut = win > 0 ? past + d - win + 1 - kb : 0;  // the first key inside the window
      if (cut > 0) m &= cut < n ? (cut < 32 ? ~0u << cut : 0u) : (n < 32 ? ~0u << n : 0u);
    }
    return (b[0] | b[1] | b[2] | b[3]) != 0u ? m : 0u;
  };

  const int krow = 8 * (qi >> 2) + (qi & 3);
  uint32_t kofs[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) kofs[j] = uint32_t(krow * KCH * 16 + (((4 * j + qq) ^ qi) * 16));

  // running softmax state of this lane's row: reference exponent ms (log2 units, trailing the maximum by
  // at most 8) and this lane group's share l of sum exp2(s c - ms)
  float ms = -__builtin_inff(), l = 0.0f;
  const float c = p.c;

  // S^T of block n, softmax, P rows and rescale factors into slot n % 2
  auto s_phase = [&](auto slot, int n) __attribute__((always_inline)) {
    if (wave >= RT) return;
    v4f s[2 * NKC];
    const char* kbase = k_slot(slot);
#pragma unroll
    for (int t = 0; t < 2 * NKC; ++t) s[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // K fragments through a ring of KR registers: fragment i + KR is read once fragment i has fed its
    // MFMA, so KR reads are in flight while the MFMAs run
    constexpr int NR = NKK * 2 * NKC, KR = S::KR;
    auto kfrag = [&](int i) __attribute__((always_inline)) {
      const int kk = i / (2 * NKC), t = i % (2 * NKC);
      const int row0 = 32 * (t >> 1) + 4 * (t & 1);
      return *reinterpret_cast<const v8bf*>(kbase + kofs[kk % 4] + row0 * (KCH * 16) + (kk / 4) * 256);
    };
    v8bf kf[KR];
#pragma unroll
    for (int i = 0; i < KR; ++i) kf[i] = kfrag(i);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int kk = i / (2 * NKC), t = i % (2 * NKC);
      s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i % KR], qf[kk], s[t], 0, 0, 0);
      if (i + KR < NR) kf[i % KR] = kfrag(i + KR);
    }
    if (!inner(n)) {
#pragma unroll
      for (int ch = 0; ch < NKC; ++ch) {
        const uint32_t m = seen(bits, depth, kb0 + n * BN + 32 * ch) >> (8 * qq);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[2 * ch + (e >> 2)][e & 3] = attn_mask(s[2 * ch + (e >> 2)][e & 3], ((m >> e) & 1u) != 0u);
      }
    }
    float bm = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < 2 * NKC; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) bm = fmaxf(bm, s[t][i]);
    bm = lanes4_max(bm);
    const float bmc = bm * c;
    const bool grow = bmc > ms + 8.0f;  // false while every key so far is masked (bmc = -inf)
    const bool had = ms != -__builtin_inff();
    const float alpha = !grow ? 1.0f : (had ? __builtin_amdgcn_exp2f(ms - bmc) : 0.0f);
    ms = grow ? bmc : ms;
    const float mref = ms == -__builtin_inff() ? 0.0f : ms;
    float bs = 0.0f;
    uint16_t* prow = reinterpret_cast<uint16_t*>(aux + slot * S::P_SLOT) + srow * PLD + 8 * qq;
#pragma unroll
    for (int ch = 0; ch < NKC; ++ch) {
      v8bf pb;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * ch + (e >> 2)][e & 3], c, -mref));
        bs += pe;
        pb[e] = (__bf16)pe;
      }
      *reinterpret_cast<v8bf*>(prow + 32 * ch) = pb;
    }
    l = l * alpha + bs;
    if (qq == 0) alpha_s[slot * R + srow] = alpha;
    // a row whose maximum grew past a finite one needs its O rescaled (a row that had none has O = 0)
    const bool any = __builtin_amdgcn_ballot_w64(grow && had) != 0;
    if (lane == 0) flag_s[slot * 16 + wave] = any ? 1 : 0;
  };

  // O^T for columns [wave D/NW, (wave+1) D/NW) of all rows: o[dt][rt] register i of lane (qi, qq) is
  // d = wave D/NW + 16 dt + 4 qq + i, row 16 rt + qi
  v4f o[NDW][RT];
#pragma unroll
  for (int dt = 0; dt < NDW; ++dt)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) o[dt][rt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const int vsrc = qq * 8 + (qi >> 2);  // this lane's V source row within a 32-key chunk (+4)
  int found = 0;                        // infinities or NaN were taken out of V (the same for the workgroup)
  auto pv_phase = [&](auto slot, int n) __attribute__((always_inline)) {
    int f = 0;
#pragma unroll
    for (int w = 0; w < RT; ++w) f |= flag_s[slot * 16 + w];
    if (f != 0) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float a = alpha_s[slot * R + rt * 16 + qi];
#pragma unroll
        for (int dt = 0; dt < NDW; ++dt) o[dt][rt] *= a;
      }
    }
    char* const vl = v_slot(slot);
    const uint16_t* pl = reinterpret_cast<const uint16_t*>(aux + slot * S::P_SLOT);
    if (!inner(n)) {
      // infinities and NaN in the block's V are taken out of the product (0 * inf would be NaN) and added
      // at the end to the rows that see them
      int bad = 0;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        v4u* const at = reinterpret_cast<v4u*>(vl + (u * NT + tid) * 16);
        v4u w = *at;
        int b = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u, b = 1;
          if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu, b = 1;
        }
        if (b) *at = w;
        bad |= b;
      }
      const bool any = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
      if (lane == 0) found_s[wave] = any ? 1 : 0;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) found |= found_s[w];
    }
#pragma unroll
    for (int ch = 0; ch < NKC; ++ch) {
      v8bf va[NDW];
#pragma unroll
      for (int dt = 0; dt < NDW; ++dt) {
        const int d = wave * (D / NW) + 16 * dt + 4 * (qi & 3);  // this lane's 4 source columns
        const int r0 = 32 * ch + vsrc, r1 = r0 + 4;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(
            vl + r0 * ROW + (((d >> 3) ^ (2 * (r0 & 3))) * 16) + (d & 7) * 2));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(
            vl + r1 * ROW + (((d >> 3) ^ (2 * (r1 & 3))) * 16) + (d & 7) * 2));
        va[dt] = __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const v8bf pb = *reinterpret_cast<const v8bf*>(pl + (rt * 16 + qi) * PLD + 32 * ch + 8 * qq);
#pragma unroll
        for (int dt = 0; dt < NDW; ++dt) o[dt][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[dt], pb, o[dt][rt], 0, 0, 0);
      }
    }
  };

  if (nblk > 1)
    attn_wait_vmcnt<KU>();  // K(0), V(0) and Q have landed; K(1) may be in flight
  else
    attn_wait_vmcnt<0>();
  __syncthreads();
  s_phase(Even{}, 0);
  auto step = [&](auto slot, auto other, int n) __attribute__((always_inline)) {
    attn_wait_vmcnt<0>();
    __syncthreads();  // P(n) of every row; K(n + 1) and V(n) in LDS; the other slots free
    if (n + 2 < nblk) issue_k(slot, n + 2);
    issue_v(other, n + 1);
    s_phase(other, n + 1);
    __builtin_amdgcn_sched_barrier(0);  // (the two phases' registers together spill)
    pv_phase(slot, n);
  };
  auto last = [&](auto slot, int n) __attribute__((always_inline)) {
    attn_wait_vmcnt<0>();
    __syncthreads();
    pv_phase(slot, n);
  };
  if constexpr (SPLIT) {
    int n = 0;
    for (; n + 2 < nblk; n += 2) {
      step(Even{}, Odd{}, n);
      step(Odd{}, Even{}, n + 1);
    }
    if (n + 1 < nblk) {
      step(Even{}, Odd{}, n);
      last(Odd{}, n + 1);
    } else {
      last(Even{}, n);
    }
  } else {
    for (int n = 0; n + 1 < nblk; ++n) step(n & 1, (n + 1) & 1, n);
    last((nblk - 1) & 1, nblk - 1);
  }

  const int d_lane = wave * (D / NW) + 4 * qq;  // + 16 dt + i
  if (found) {
#pragma unroll 1
    for (int rt = 0; rt < RT; ++rt) {
      const int r = tile * R + rt * 16 + qi;
      uint32_t b[TREE_WORDS];
      int d;
      view(r, b, d);
      v4f add[NDW];
#pragma unroll
      for (int dt = 0; dt < NDW; ++dt) add[dt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      for (int j = 0; j < nkeys; ++j) {
        if (inner(j / BN) || !((seen(b, d, kb0 + (j & ~31)) >> (j & 31)) & 1u)) continue;
        const uint16_t* vp = p.v + int64_t(g) * p.vhs + int64_t(kb0 + j) * p.vrs + d_lane;
#pragma unroll
        for (int dt = 0; dt < NDW; ++dt) {
          const v2u w = *reinterpret_cast<const v2u*>(vp + 16 * dt);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = (i & 1) ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16;
            if ((x & 0x7f800000u) == 0x7f800000u) add[dt][i] += __uint_as_float(x);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (t == rt) {
#pragma unroll
          for (int dt = 0; dt < NDW; ++dt) o[dt][t] += add[dt];
        }
    }
  }

  // An unused node's row: the last part, which holds the tree, marks it with a sum of -1.
  float lt = lanes4_sum(l);
  if (last_part && !live) {
    ms = -__builtin_inff();
    lt = -1.0f;
  }
  if (geo.nparts > 1) {
    const int64_t base = (int64_t(g) * p.nparts + part) * p.rows;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = tile * R + rt * 16 + qi;
      if (r < p.rows) {
        float* po = p.part_o + (base + r) * D + d_lane;
#pragma unroll
        for (int dt = 0; dt < NDW; ++dt) *reinterpret_cast<v4f*>(po + 16 * dt) = o[dt][rt];
      }
    }
    if (wave < RT && qq == 0 && valid) *reinterpret_cast<v2f*>(p.part_ml + (base + row) * 2) = v2f{ms, lt};
    return;
  }
  // one part: normalise and store (the row factors over the rescale factors, read for the last time)
  __syncthreads();
  if (wave < RT && qq == 0) {
    alpha_s[srow] = lt > 0.0f ? 1.0f / lt : (lt == lt ? 0.0f : lt);  // (a NaN sum stays one)
    if (valid && p.lse)
      p.lse[int64_t(g * G + hl) * p.N + qnode] =
          lt > 0.0f ? ms * 0.69314718055994531f + __logf(lt) : (lt == lt ? -__builtin_inff() : lt);
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = tile * R + rt * 16 + qi;
    if (r < p.rows) {
      const float inv = alpha_s[rt * 16 + qi];
      uint16_t* op = p.o + int64_t(g * G + r % G) * p.ohs + int64_t(r / G) * p.ors + d_lane;
#pragma unroll
      for (int dt = 0; dt < NDW; ++dt) {
        v2u w;
        w[0] = inv != 0.0f ? pack_bf16x2(o[dt][rt][0] * inv, o[dt][rt][1] * inv) : 0u;
        w[1] = inv != 0.0f ? pack_bf16x2(o[dt][rt][2] * inv, o[dt][rt][3] * inv) : 0u;
        *reinterpret_cast<v2u*>(op + 16 * dt) = w;
      }
    }
  }
}

// Joins the parts of each row: M = max m_s, w_s = exp2(m_s - M), o = sum_s w_s o_s / sum_s w_s l_s.  A
// workgroup takes one row's 64 columns: thread t sums column group t % 16 over parts t / 16, + 16, ..,
// eight loads in flight, and the 16 sums are added in order (the same result whatever the timing).
template <int D, int BN>
__global__ __launch_bounds__(256) void attn_tree_merge_kernel(TreeParams p) {
  __shared__ float wsh[TREE_MAX_PARTS];
  __shared__ v4f sums[256];
  __shared__ float red[4][2];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int g = blockIdx.x / p.rows, row = blockIdx.x % p.rows;
  const int np = tree_geom<BN>(p).nparts;
  if (np <= 1) return;  // the attention kernel wrote the row
  const int64_t base = int64_t(g) * p.nparts * p.rows + row;  // part s at base + s * rows
  const v2f* ml = reinterpret_cast<const v2f*>(p.part_ml) + base;
  float mx = -__builtin_inff();
  for (int s = t; s < np; s += 256) mx = fmaxf(mx, ml[int64_t(s) * p.rows][0]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (lane == 0) red[wave][0] = mx;
  const bool unused = ml[int64_t(np - 1) * p.rows][1] == -1.0f;
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
  const int node = row / p.G, h = g * p.G + row % p.G;
  const bool none = unused || L == 0.0f;
  v2u w = v2u{0u, 0u};
  if (!none) {
    const float inv = 1.0f / L;
    w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  }
  *reinterpret_cast<v2u*>(p.o + int64_t(h) * p.ohs + int64_t(node) * p.ors + col) = w;
  if (p.lse && col == 0)
    p.lse[int64_t(h) * p.N + node] = none ? -__builtin_inff() : mx * 0.69314718055994531f + __logf(L);
}

// ---- host ----------------------------------------------------------------------------------------

// Row tile (in 16 rows) and key parts of a call.
struct TreePlan {
  int rt, ntiles, nparts;
  int64_t nblk;  // key blocks of the longest span
};

static TreePlan tree_plan(int64_t H, int64_t KV, int64_t N, int64_t M, int64_t Tk, int64_t D, int64_t past,
                          int64_t window) {
  const int64_t rows = N * (H / KV);
  const int bn = D == 128 ? 64 : 32;
  const int64_t ctx = past >= 0 ? past : Tk - M;  // a length in device memory: the longest
  const int64_t span = (window > 0 && window - 1 < ctx ? window - 1 : ctx) + M;
  TreePlan best{}, pl;
  pl.nblk = best.nblk = (span + bn - 1) / bn;
  // Of the row tiles and part counts that put a quarter of a workgroup to two workgroups on every CU, the
  // one that a model of the call finishes first: each CU's key blocks, the start and the first block's way
  // through memory, the tile's store, and the parts written and read back.  The times of a block
  // (64 KiB of K and V at head_dim 512, 32 KiB else) are fitted to calls of 8 to 1024 rows over 700 to
  // 65521 keys; small tiles read the keys more often, large ones leave more to be joined.  us at 16 / 32 /
  // 64 / 80 / 96 / 128 rows a tile: 8 heads of 512, 16 nodes over 3658 rows 20 / 22 / 26 / 26 / 27 / 31, over
  // 32749 rows 57 / 42 / 36 / 39 / 39 / 45, 64 nodes over 32749 rows 194 / 121 / 75 / - / - / 72; 32 heads of
  // 128 on 8, 33 nodes over 65521 rows 163 / 114 / 131 / 96 / 103 / 112.
  static const int tiles[6] = {1, 2, 4, 5, 6, 8};
  static const double block[3][6] = {{0.63, 0.75, 1.2, 1.27, 1.4, 1.6}, {0.55, 0.8, 1.15, 1.3, 1.45, 1.75},
                                     {1.45, 1.7, 1.8, 2.4, 2.5, 2.9}};
  const int di = D == 128 ? 0 : D == 256 ? 1 : 2;
  const int64_t xcd_cus = std::max(1, attn_cu_count() / 8);
  double least = 0.0;
  for (int r = 0; r < 6; ++r) {
    pl.rt = tiles[r];
    if (r > 0 && rows <= 16 * tiles[r - 1]) break;  // the tile before holds them all
    pl.ntiles = int((rows + 16 * pl.rt - 1) / (16 * pl.rt));
    const bool two = di < 2 && pl.rt <= (di == 0 ? 2 : 4);  // two workgroups fit a CU's LDS
    for (int64_t quarters : {1, 2, 4, 8}) {
      const int64_t pairs = std::max<int64_t>(1, quarters * xcd_cus / (4 * pl.ntiles));  // (KV head, part)s on an XCD
      const int64_t want = std::max<int64_t>(1, pairs * 8 / KV);
      pl.nparts = int(std::min<int64_t>(std::min<int64_t>(want, pl.nblk), TREE_MAX_PARTS));
      const int64_t wgs = (KV * pl.nparts + 7) / 8 * pl.ntiles, per_cu = (wgs + xcd_cus - 1) / xcd_cus;
      const double t = double((pl.nblk + pl.nparts - 1) / pl.nparts) * double(per_cu) * block[di][r] *
                           (two && per_cu == 1 ? 1.25 : 1.0) +
                       double(16 * pl.rt * D * 4) / 60e3 +
                       (pl.nparts > 1 ? 1.5 + double(KV * rows * pl.nparts * D * 8) / 8e6 : 0.0);
      if (best.rt == 0 || t < least) least = t, best = pl;
    }
  }
  return best;
}

template <int D>
static void tree_launch(const TreeParams& p, int rt, hipStream_t stream) {
  const unsigned pairs = unsigned(p.KV) * unsigned(p.nparts);
  const dim3 grid{(pairs + 7) / 8 * 8 * unsigned(p.ntiles), 1, 1};
  switch (rt) {
    case 1: attn_tree_kernel<D, 1><<<grid, TreeShape<D, 1>::NT, 0, stream>>>(p); break;
    case 2: attn_tree_kernel<D, 2><<<grid, TreeShape<D, 2>::NT, 0, stream>>>(p); break;
    case 4: attn_tree_kernel<D, 4><<<grid, TreeShape<D, 4>::NT, 0, stream>>>(p); break;
    case 5: attn_tree_kernel<D, 5><<<grid, TreeShape<D, 5>::NT, 0, stream>>>(p); break;
    case 6: attn_tree_kernel<D, 6><<<grid, TreeShape<D, 6>::NT, 0, stream>>>(p); break;
    default: attn_tree_kernel<D, 8><<<grid, TreeShape<D, 8>::NT, 0, stream>>>(p);
  }
  if (p.nparts > 1)
    attn_tree_merge_kernel<D, TreeShape<D, 1>::BN>
        <<<dim3{unsigned(p.KV * p.rows), unsigned(D / 64), 1}, 256, 0, stream>>>(p);
}

static bool tree_shape_ok(int64_t H, int64_t KV, int64_t N, int64_t M, int64_t Tk, int64_t D, int64_t window) {
  return H >= 1 && KV >= 1 && H % KV == 0 && H <= (1 << 16) && N >= 1 && N <= M && M <= TREE_MAX_NODES && Tk >= M &&
         Tk <= INT32_MAX / 2 && window >= 0 && window <= INT32_MAX / 2 && (D == 128 || D == 256 || D == 512);
}

}  // namespace w8a8

using namespace w8a8;

extern "C" int64_t w8a8_attention_tree_workspace_bytes(int64_t H, int64_t KV, int64_t N, int64_t M, int64_t Tk,
                                                       int64_t D, int64_t n_past, int64_t window) {
  if (!tree_shape_ok(H, KV, N, M, Tk, D, window) || n_past < -1 || n_past > Tk - M) return -1;
  const TreePlan pl = tree_plan(H, KV, N, M, Tk, D, n_past, window);
  return pl.nparts > 1 ? int64_t(H) * N * pl.nparts * (D + 2) * 4 : 0;
}

extern "C" int w8a8_attention_tree_plan(int64_t H, int64_t KV, int64_t N, int64_t M, int64_t Tk, int64_t D,
                                        int64_t n_past, int64_t window, int* row_tile, int* parts) {
  if (!tree_shape_ok(H, KV, N, M, Tk, D, window) || n_past < -1 || n_past > Tk - M)
    return fail(W8A8_EINVAL, "attention_tree_plan: invalid arguments");
  const TreePlan pl = tree_plan(H, KV, N, M, Tk, D, n_past, window);
  if (row_tile) *row_tile = 16 * pl.rt;
  if (parts) *parts = pl.nparts;
  return W8A8_OK;
}

extern "C" int w8a8_attention_tree_bf16(const uint16_t* q, int64_t q_head_stride, int64_t q_row_stride,
                                        const uint16_t* k, int64_t k_head_stride, int64_t k_row_stride,
                                        const uint16_t* v, int64_t v_head_stride, int64_t v_row_stride, int64_t H,
                                        int64_t KV, int64_t N, int64_t M, int64_t Tk, int64_t D,
                                        const int32_t* parents, int64_t n_past, const int32_t* n_past_dev,
                                        int64_t window, float scale, uint16_t* o, int64_t o_head_stride,
                                        int64_t o_row_stride, float* lse, void* workspace, int64_t workspace_bytes,
                                        hipStream_t stream) {
  const char* what = "attention_tree";
  if (D != 128 && D != 256 && D != 512)
    return fail(W8A8_ENOTSUP, "%s: head_dim %lld (supported: 128, 256, 512)", what, (long long)D);
  if (M > TREE_MAX_NODES) return fail(W8A8_ENOTSUP, "%s: %lld nodes (at most %d)", what, (long long)M, TREE_MAX_NODES);
  if (!tree_shape_ok(H, KV, N, M, Tk, D, window))
    return fail(W8A8_EINVAL, "%s: H=%lld KV=%lld N=%lld M=%lld Tk=%lld window=%lld", what, (long long)H, (long long)KV,
                (long long)N, (long long)M, (long long)Tk, (long long)window);
  if (n_past_dev ? n_past != -1 : (n_past < 0 || n_past > Tk - M))
    return fail(W8A8_EINVAL, "%s: n_past=%lld (0 .. Tk - M = %lld, or -1 with n_past_dev)", what, (long long)n_past,
                (long long)(Tk - M));
  if (!(scale > 0.0f) || scale == __builtin_inff()) return fail(W8A8_EINVAL, "%s: scale must be positive", what);
  if (!q || !k || !v || !o || !parents) return fail(W8A8_EINVAL, "%s: null pointer", what);
  const TreePlan pl = tree_plan(H, KV, N, M, Tk, D, n_past, window);
  const int64_t need = w8a8_attention_tree_workspace_bytes(H, KV, N, M, Tk, D, n_past, window);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(W8A8_EINVAL, "%s: workspace of %lld bytes, %lld needed", what, (long long)(workspace ? workspace_bytes : 0),
                (long long)need);
  const int64_t rs[4] = {k_row_stride, v_row_stride, N > 1 ? q_row_stride : D, N > 1 ? o_row_stride : D};
  const int64_t hs[4] = {KV > 1 ? k_head_stride : 0, KV > 1 ? v_head_stride : 0, H > 1 ? q_head_stride : 0,
                         H > 1 ? o_head_stride : 0};
  for (int i = 0; i < 4; ++i) {
    if (rs[i] < D || hs[i] < 0) return fail(W8A8_EINVAL, "%s: row strides smaller than head_dim, or negative", what);
    if (rs[i] % 8 != 0 || hs[i] % 8 != 0) return fail(W8A8_EALIGN, "%s: strides must be multiples of 8 elements", what);
  }
  if (H > 1 && o_head_stride < D) return fail(W8A8_EINVAL, "%s: o's heads overlap, stride %lld", what, (long long)o_head_stride);
  if ((uintptr_t)q % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)o % 16 || (uintptr_t)workspace % 16 ||
      (uintptr_t)parents % 4 || (uintptr_t)n_past_dev % 4 || (uintptr_t)lse % 4)
    return fail(W8A8_EALIGN, "%s: q, k, v, o and the workspace 16-byte, parents, n_past and lse 4-byte aligned", what);
  // a part's rows are addressed by 32-bit offsets from its first one
  const int bn = D == 128 ? 64 : 32;
  const int64_t most = ((pl.nblk + pl.nparts - 1) / pl.nparts + 1) * bn;
  if (std::max(k_row_stride, v_row_stride) * 2 * most >= (int64_t(1) << 32))
    return fail(W8A8_ENOTSUP, "%s: %lld keys of %lld bytes each per workgroup pass 32-bit offsets", what, (long long)most,
                (long long)(std::max(k_row_stride, v_row_stride) * 2));
  TreeParams p{};
  p.q = q; p.qhs = hs[2]; p.qrs = rs[2]; p.k = k; p.khs = hs[0]; p.krs = rs[0]; p.v = v; p.vhs = hs[1]; p.vrs = rs[1];
  p.o = o; p.ohs = hs[3]; p.ors = rs[3]; p.lse = lse; p.parents = parents; p.past_dev = n_past_dev;
  p.past = int(std::max<int64_t>(n_past, 0)); p.KV = int(KV); p.G = int(H / KV); p.N = int(N); p.M = int(M);
  p.Tk = int(Tk); p.window = int(window); p.rows = int(N * (H / KV)); p.ntiles = pl.ntiles; p.nparts = pl.nparts;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + int64_t(H) * N * pl.nparts * D;
  p.c = scale * 1.4426950408889634f;
  if (D == 128)
    tree_launch<128>(p, pl.rt, stream);
  else if (D == 256)
    tree_launch<256>(p, pl.rt, stream);
  else
    tree_launch<512>(p, pl.rt, stream);
  return check_launch("attention_tree_bf16");
}
