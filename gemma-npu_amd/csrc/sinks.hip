// Attention with a sliding window and a few first tokens that stay visible.
//
//   o[h, i, :] = sum_j softmax_j(scale q[h, i] . k[g, j]) v[g, j],   g = h / (H / KV),
//
// over the keys j that the query at position p = q_start + i sees: j <= p and, with a window W, p - j < W or j < sinks.
// The reference's sliding layers have the window alone (pipeline.py:158-180); a conversation that runs far past it
// keeps its first tokens this way.  One kernel for prompts, drafted runs and single tokens.
//
// Work split.  The rows (query, head) of one KV head, Tq G of them, are cut into tiles of 16 RT rows.  A tile's key blocks
// are those of the sinks, then, without those between, those from its first query's window on to its last query;
// few tiles split theirs into parts, which a second kernel joins by their logsumexp.  Neighbouring tiles run on one
// XCD and share its L2's copy of the window.  In a kernel trace 3658 queries of 8 heads of 256,
// window 512: 40 us (tiles of 64 rows took 71 where those of 128 took 47: edge blocks' values were looked through in LDS then, a
// barrier more); 2048 of 32 heads of 128 on 8, window 4096: 239 us, untraced 203 a call, 681 TFLOP/s (four waves of 32 rows
// each 300); one token over a window of 1020: 5.3 us and 4 to join.
//
// Within a workgroup the key blocks pass through a two-slot LDS ring (buffer_load ... lds, K one block further ahead than
// V), one barrier per block: iteration n makes S^T = K Q^T and the softmax of block n + 1 and multiplies P V of block n.
// The first RT waves own 16 rows' S phase each, every wave D / NW columns of O^T, its V^T operand read from the
// row-major V rows with ds_read_b64_tr_b16.  Every block's buffer ends at the tile's last visible key, so whatever
// lies behind it is not read.  Scores, softmax and sums are fp32; the softmax weights are rounded to bf16 for the
// second product, at most 2^-8 of each weight, as the other attention kernels do.
#include <algorithm>
#include <type_traits>

#include "attn_common.h"
#include "attn_parts.h"

namespace w8a8 {

struct SinkParams {
  const uint16_t* q; int64_t qhs, qrs;  // bf16 [H, Tq, D] (element strides, last dim contiguous)
  const uint16_t* k; int64_t khs, krs;  // bf16 [KV, Tk, D]
  const uint16_t* v; int64_t vhs, vrs;
  PartParams out;                       // o, lse, parts, rows
  const int32_t* start_dev;             // q_start in device memory, or null
  int start, Tq, Tk, window, sinks, ntiles;
  float c;                              // scale * log2(e)
};

// The key blocks that a tile's rows see: n < nb stands for block n, from `sb` on for block n + skip.
struct SinkGeom {
  int start, pmin, pmax, sb, skip, nb, np;
};
template <int BN>
__device__ __forceinline__ SinkGeom sink_geom(const SinkParams& p, int tile, int R) {
  SinkGeom t;
  t.start = p.start_dev ? max(0, min(*p.start_dev, p.Tk - p.Tq)) : p.start;
  const int r0 = tile * R, r1 = min(r0 + R, p.out.rows) - 1;
  t.pmin = t.start + r0 / p.out.G;
  t.pmax = t.start + r1 / p.out.G;
  const int wb = p.window > 0 ? max(0, t.pmin - p.window + 1) / BN : 0;
  t.sb = (min(p.sinks, p.Tk) + BN - 1) / BN;
  t.skip = max(0, wb - t.sb);
  t.nb = t.pmax / BN + 1 - t.skip;
  t.np = min(p.out.nparts, t.nb);
  return t;
}

constexpr int sink_waves(int rt, int d) { return rt > 4 || (d == 512 && rt == 4) ? 8 : 4; }

template <int D, int RT>
struct SinkShape {
  static constexpr int NW = sink_waves(RT, D);
  static constexpr int NT = NW * 64;
  static constexpr int BN = D == 128 ? 64 : 32;      // keys per block
  static constexpr int R = RT * 16;                  // rows per tile
  static constexpr int KCH = D / 8;                  // 16-byte chunks per K / V row
  static constexpr int ROW = D * 2;
  static constexpr int KV_SLOT = BN * ROW;
  static constexpr int PLD = BN + 8;                 // padded P row, elements
  static constexpr int P_SLOT = R * PLD * 2;
  static constexpr int A_OFF = 2 * P_SLOT;           // P [2]; alpha [2][R]
  static constexpr int F_OFF = A_OFF + 2 * R * 4;    // flags [2][16]
  static constexpr int AUX = F_OFF + 2 * 16 * 4;
  static constexpr int NDW = D / NW / 16;            // 16-wide d tiles of O^T per wave
  static constexpr int KR = 3;                       // K fragments in flight
  static constexpr bool SPLIT = D < 512 || RT < 5;   // a variable per slot (the others would spill)
};

template <int D, int RT>
__global__ __launch_bounds__(sink_waves(RT, D) * 64, 1) void attn_sink_kernel(SinkParams p) {
  using S = SinkShape<D, RT>;
  constexpr int NW = S::NW, NT = S::NT, BN = S::BN, R = S::R, KCH = S::KCH, ROW = S::ROW, PLD = S::PLD, NDW = S::NDW;
  constexpr int NKC = BN / 32;              // 32-key chunks per block
  constexpr int KU = BN * KCH / NT;         // DMA instructions per thread per K or V block
  constexpr int NKK = D / 32;               // k-steps of S^T
  static_assert(KU * NT == BN * KCH && NDW >= 1 && RT <= NW, "tiling");
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

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 15, qq = lane >> 4;

  const int lb = xcd_remap(blockIdx.x, gridDim.x);
  const int tile = lb % p.ntiles, pair = lb / p.ntiles, g = pair / p.out.nparts, part = pair % p.out.nparts;
  const SinkGeom geo = sink_geom<BN>(p, tile, R);
  if (part >= geo.np) return;  // (the whole workgroup, before any barrier)
  const int G = p.out.G, rows = p.out.rows, win = p.window, sinks = p.sinks;
  const int n_lo = int(int64_t(part) * geo.nb / geo.np), n_hi = int(int64_t(part + 1) * geo.nb / geo.np);
  const int nblk = n_hi - n_lo;  // at least one block
  auto key_of = [&](int n) __attribute__((always_inline)) {  // first key of the part's block n
    const int i = n_lo + n;
    return (i < geo.sb ? i : i + geo.skip) * BN;
  };

  const uint32_t krs2 = uint32_t(p.krs) * 2u, vrs2 = uint32_t(p.vrs) * 2u;
  const uint16_t* const kg = p.k + int64_t(g) * p.khs;
  const uint16_t* const vg = p.v + int64_t(g) * p.vhs;

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
  // block n goes to slot n % 2 (with SPLIT a type, so that each access names its slot's variable).  A block is a buffer
  // of its own that ends at the tile's last key: caches of any length have 32-bit offsets, and rows behind it read zero.
  using Even = std::integral_constant<int, 0>;
  using Odd = std::integral_constant<int, 1>;
  auto issue_k = [&](auto slot, int n) __attribute__((always_inline)) {
    const int kb = key_of(n);
    const __amdgpu_buffer_rsrc_t r =
        make_rsrc(kg + int64_t(kb) * p.krs, uint32_t(min(BN, geo.pmax + 1 - kb) - 1) * krs2 + uint32_t(ROW));
#pragma unroll
    for (int u = 0; u < KU; ++u) attn_dma16(r, k_slot(slot) + (u * NW + wave) * 1024, koff[u]);
  };
  auto issue_v = [&](auto slot, int n) __attribute__((always_inline)) {
    const int kb = key_of(n);
    const __amdgpu_buffer_rsrc_t r =
        make_rsrc(vg + int64_t(kb) * p.vrs, uint32_t(min(BN, geo.pmax + 1 - kb) - 1) * vrs2 + uint32_t(ROW));
#pragma unroll
    for (int u = 0; u < KU; ++u) attn_dma16(r, v_slot(slot) + (u * NW + wave) * 1024, voff[u]);
  };

  issue_k(Even{}, 0);
  issue_v(Even{}, 0);
  // Q (B operand: lane (qi, qq) holds q[row][32 kk + 8 qq .. + 7] of this wave's 16 rows)
  const int srow = 16 * (wave % RT) + qi;
  const int row = tile * R + srow;               // (query, head) row of the KV head
  const bool valid = row < rows;
  const int qrow = row / G, hl = row % G;
  const int pos = valid ? geo.start + qrow : -1;  // (sees nothing)
  v8bf qf[NKK];
  {
    const uint16_t* qp = p.q + int64_t(g * G + hl) * p.qhs + int64_t(qrow) * p.qrs + 8 * qq;
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk) {
      v4i t = v4i{0, 0, 0, 0};
      if (valid) t = *reinterpret_cast<const v4i*>(qp + 32 * kk);
      qf[kk] = __builtin_bit_cast(v8bf, t);
    }
  }
  if (nblk > 1) issue_k(Odd{}, 1);

  const uint32_t near = win > 0 ? uint32_t(win) : 0x80000000u;
  auto seen = [&](int key, int at) __attribute__((always_inline)) {  // (compares alone: a branch here is one per score)
    return (uint32_t(at - key) < near) | ((key <= at) & (key < sinks));
  };
  // Block n is seen whole by every row.
  const bool full = tile * R + R <= rows;
  auto inner = [&](int n) __attribute__((always_inline)) {
    const int kb = key_of(n);
    return full && kb + BN - 1 <= geo.pmin && (win <= 0 || kb > geo.pmax - win || kb + BN <= sinks);
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
      const int kb = key_of(n) + 8 * qq;
#pragma unroll
      for (int t = 0; t < 2 * NKC; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] = attn_mask(s[t][i], seen(kb + 32 * (t >> 1) + 4 * (t & 1) + i, pos));
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
  bool found = false;                   // infinities or NaN were taken out of the wave's columns of V
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
    const char* const vl = v_slot(slot);
    const uint16_t* pl = reinterpret_cast<const uint16_t*>(aux + slot * S::P_SLOT);
    const bool edge = !inner(n);
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
      if (edge) {
        // infinities and NaN in the block's V are taken out of the product (0 * inf would be NaN) and added
        // at the end to the rows that see them
        uint32_t bad = 0u;
        auto odd = [](uint32_t w) __attribute__((always_inline)) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
#pragma unroll
        for (int dt = 0; dt < NDW; ++dt) {
          const v4u w = __builtin_bit_cast(v4u, va[dt]);
#pragma unroll
          for (int e = 0; e < 4; ++e) bad |= odd(w[e]);
        }
        if (__builtin_amdgcn_ballot_w64(bad != 0u) != 0) {
          found = true;
#pragma unroll
          for (int dt = 0; dt < NDW; ++dt) {
            v4u w = __builtin_bit_cast(v4u, va[dt]);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] &= ~((odd(w[e]) >> 15) * 0xffffu);
            va[dt] = __builtin_bit_cast(v8bf, w);
          }
        }
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
      const int at = r < rows ? geo.start + r / G : -1;
      v4f add[NDW];
#pragma unroll
      for (int dt = 0; dt < NDW; ++dt) add[dt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      for (int n = 0; n < nblk; ++n) {
        if (inner(n)) continue;
        for (int j = 0; j < BN; ++j) {
          const int key = key_of(n) + j;
          if (!seen(key, at)) continue;
          const uint16_t* vp = vg + int64_t(key) * p.vrs + d_lane;
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
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (t == rt) {
#pragma unroll
          for (int dt = 0; dt < NDW; ++dt) o[dt][t] += add[dt];
        }
    }
  }

  const float lt = lanes4_sum(l);
  if (geo.np > 1) {
    const int64_t base = (int64_t(g) * p.out.nparts + part) * rows;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = tile * R + rt * 16 + qi;
      if (r < rows) {
        float* po = p.out.part_o + (base + r) * D + d_lane;
#pragma unroll
        for (int dt = 0; dt < NDW; ++dt) *reinterpret_cast<v4f*>(po + 16 * dt) = o[dt][rt];
      }
    }
    if (wave < RT && qq == 0 && valid) *reinterpret_cast<v2f*>(p.out.part_ml + (base + row) * 2) = v2f{ms, lt};
    return;
  }
  // one part: normalise and store (the row factors over the rescale factors, read for the last time)
  __syncthreads();
  if (wave < RT && qq == 0) {
    alpha_s[srow] = lt > 0.0f ? 1.0f / lt : (lt == lt ? 0.0f : lt);  // (a NaN sum stays one)
    if (valid && p.out.lse) p.out.lse[int64_t(g * G + hl) * p.Tq + qrow] = part_lse(ms, lt);
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = tile * R + rt * 16 + qi;
    if (r < rows) {
      const float inv = alpha_s[rt * 16 + qi];
      uint16_t* op = p.out.o + int64_t(g * G + r % G) * p.out.ohs + int64_t(r / G) * p.out.ors + d_lane;
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

template <int D, int BN>
__global__ __launch_bounds__(256) void sink_merge_kernel(SinkParams p, int R) {
  const int row = blockIdx.x % p.out.rows;
  part_merge<D>(p.out, sink_geom<BN>(p, row / R, R).np, p.Tq);
}
template <int D, int BN>
__global__ __launch_bounds__(256) void sink_merge_few_kernel(SinkParams p, int R) {
  part_merge_few<D>(p.out, [&](int row) { return sink_geom<BN>(p, row / R, R).np; }, p.Tq);
}

// ---- host ----------------------------------------------------------------------------------------

// Row tile (in 16 rows) and key parts of a call.
struct SinkPlan {
  int rt, ntiles, nparts;
};

static SinkPlan sink_plan(int64_t H, int64_t KV, int64_t Tq, int64_t Tk, int64_t D, int64_t start, int64_t window,
                          int64_t sinks) {
  const int64_t G = H / KV, rows = Tq * G, bn = D == 128 ? 64 : 32;
  const int64_t keys = start >= 0 ? start + Tq : Tk;  // a position in device memory: the last
  SinkPlan best{}, pl;
  // As for attention of a tree of drafted tokens: of the row tiles and part counts, the one that a model of the call finishes
  // first.  Times of a block in us (64 KiB of K and V at head_dim 512, 32 KiB else).
  static const int tiles[4] = {1, 2, 4, 8};
  static const double block[3][4] = {{0.63, 0.75, 1.2, 1.6}, {0.55, 0.8, 1.15, 1.75}, {1.45, 1.7, 1.8, 2.9}};
  const int di = D == 128 ? 0 : D == 256 ? 1 : 2;
  const int64_t cus = attn_cu_count();
  double least = 0.0;
  for (int r = 0; r < 4; ++r) {
    pl.rt = tiles[r];
    if (r > 0 && rows <= 16 * tiles[r - 1]) break;  // the tile before holds them all
    pl.ntiles = int((rows + 16 * pl.rt - 1) / (16 * pl.rt));
    const bool two = di < 2 && pl.rt <= (di == 0 ? 2 : 4);  // two workgroups fit a CU's LDS
    // the longest tile's blocks, and their mean over the tiles (without a window the first ones have few)
    const int64_t span = (16 * pl.rt - 1) / G + 1, all = (keys + bn - 1) / bn;
    int64_t nb = all;
    if (window > 0) nb = std::min(all, (window + span) / bn + 1 + (std::min(sinks, keys) + bn - 1) / bn);
    const double mean = window > 0 || start < 0 ? double(nb) : std::max(1.0, double(nb) * (1.0 - 0.5 * double(Tq) / double(keys)));
    for (int64_t quarters : {1, 2, 4, 8}) {
      const int64_t want = std::max<int64_t>(1, quarters * cus / (4 * pl.ntiles * KV));
      pl.nparts = int(std::min<int64_t>({want, nb, PART_MAX}));
      const int64_t wgs = KV * pl.nparts * pl.ntiles, rounds = (wgs + cus - 1) / cus;
      const double per = mean / pl.nparts;
      const double t = std::max(double((nb + pl.nparts - 1) / pl.nparts), per * double(rounds)) * block[di][r] *
                           (two && rounds == 1 ? 1.25 : 1.0) +
                       double(16 * pl.rt * D * 4) / 60e3 * double(rounds) +
                       (pl.nparts > 1 ? 1.5 + double(KV * rows * pl.nparts * D * 8) / 8e6 : 0.0);
      if (best.rt == 0 || t < least) least = t, best = pl;
    }
  }
  return best;
}

template <int D>
static void sink_launch(const SinkParams& p, int rt, hipStream_t stream) {
  const dim3 grid{unsigned(p.out.KV) * unsigned(p.out.nparts) * unsigned(p.ntiles), 1, 1};
  switch (rt) {
    case 1: attn_sink_kernel<D, 1><<<grid, SinkShape<D, 1>::NT, 0, stream>>>(p); break;
    case 2: attn_sink_kernel<D, 2><<<grid, SinkShape<D, 2>::NT, 0, stream>>>(p); break;
    case 4: attn_sink_kernel<D, 4><<<grid, SinkShape<D, 4>::NT, 0, stream>>>(p); break;
    default: attn_sink_kernel<D, 8><<<grid, SinkShape<D, 8>::NT, 0, stream>>>(p);
  }
  if (p.out.nparts > PART_FEW)
    sink_merge_kernel<D, SinkShape<D, 1>::BN>
        <<<dim3{unsigned(p.out.KV) * unsigned(p.out.rows), unsigned(D / 64), 1}, 256, 0, stream>>>(p, 16 * rt);
  else if (p.out.nparts > 1)
    sink_merge_few_kernel<D, SinkShape<D, 1>::BN><<<part_few_grid<D>(p.out), 256, 0, stream>>>(p, 16 * rt);
}

static bool sink_shape_ok(int64_t H, int64_t KV, int64_t Tq, int64_t Tk, int64_t D, int64_t window, int64_t sinks) {
  return H >= 1 && KV >= 1 && H % KV == 0 && H <= (1 << 16) && Tq >= 1 && Tq <= Tk && Tk <= INT32_MAX / 2 &&
         Tq * H < (int64_t(1) << 28) && window >= 0 && window <= INT32_MAX / 2 && sinks >= 0 && sinks <= INT32_MAX / 2 &&
         (D == 128 || D == 256 || D == 512);
}

}  // namespace w8a8

using namespace w8a8;

extern "C" int64_t w8a8_attention_sinks_workspace_bytes(int64_t H, int64_t KV, int64_t Tq, int64_t Tk, int64_t D,
                                                        int64_t q_start, int64_t window, int64_t sinks) {
  if (!sink_shape_ok(H, KV, Tq, Tk, D, window, sinks) || q_start < -1 || q_start > Tk - Tq) return -1;
  const SinkPlan pl = sink_plan(H, KV, Tq, Tk, D, q_start, window, sinks);
  return pl.nparts > 1 ? H * Tq * pl.nparts * (D + 2) * 4 : 0;
}

extern "C" int w8a8_attention_sinks_plan(int64_t H, int64_t KV, int64_t Tq, int64_t Tk, int64_t D, int64_t q_start,
                                         int64_t window, int64_t sinks, int* row_tile, int* parts) {
  if (!sink_shape_ok(H, KV, Tq, Tk, D, window, sinks) || q_start < -1 || q_start > Tk - Tq)
    return fail(W8A8_EINVAL, "attention_sinks_plan: invalid arguments");
  const SinkPlan pl = sink_plan(H, KV, Tq, Tk, D, q_start, window, sinks);
  if (row_tile) *row_tile = 16 * pl.rt;
  if (parts) *parts = pl.nparts;
  return W8A8_OK;
}

extern "C" int w8a8_attention_sinks_bf16(const uint16_t* q, int64_t q_head_stride, int64_t q_row_stride, const uint16_t* k,
                                         int64_t k_head_stride, int64_t k_row_stride, const uint16_t* v,
                                         int64_t v_head_stride, int64_t v_row_stride, int64_t H, int64_t KV, int64_t Tq,
                                         int64_t Tk, int64_t D, int64_t q_start, const int32_t* q_start_dev,
                                         int64_t window, int64_t sinks, float scale, uint16_t* o, int64_t o_head_stride,
                                         int64_t o_row_stride, float* lse, void* workspace, int64_t workspace_bytes,
                                         hipStream_t stream) {
  const char* what = "attention_sinks";
  if (D != 128 && D != 256 && D != 512)
    return fail(W8A8_ENOTSUP, "%s: head_dim %lld (supported: 128, 256, 512)", what, (long long)D);
  if (!sink_shape_ok(H, KV, Tq, Tk, D, window, sinks))
    return fail(W8A8_EINVAL, "%s: H=%lld KV=%lld Tq=%lld Tk=%lld window=%lld sinks=%lld", what, (long long)H, (long long)KV,
                (long long)Tq, (long long)Tk, (long long)window, (long long)sinks);
  if (q_start_dev ? q_start != -1 : (q_start < 0 || q_start > Tk - Tq))
    return fail(W8A8_EINVAL, "%s: q_start=%lld (0 .. Tk - Tq = %lld, or -1 with a position in device memory)", what,
                (long long)q_start, (long long)(Tk - Tq));
  if (!(scale > 0.0f) || scale == __builtin_inff()) return fail(W8A8_EINVAL, "%s: scale must be positive", what);
  if (!q || !k || !v || !o) return fail(W8A8_EINVAL, "%s: null pointer", what);
  const int64_t need = w8a8_attention_sinks_workspace_bytes(H, KV, Tq, Tk, D, q_start, window, sinks);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(W8A8_EINVAL, "%s: workspace of %lld bytes, %lld needed", what, (long long)(workspace ? workspace_bytes : 0),
                (long long)need);
  const int64_t rs[4] = {Tk > 1 ? k_row_stride : D, Tk > 1 ? v_row_stride : D, Tq > 1 ? q_row_stride : D, Tq > 1 ? o_row_stride : D};
  const int64_t hs[4] = {KV > 1 ? k_head_stride : 0, KV > 1 ? v_head_stride : 0, H > 1 ? q_head_stride : 0,
                         H > 1 ? o_head_stride : 0};
  for (int i = 0; i < 4; ++i) {
    if (rs[i] < D || hs[i] < 0) return fail(W8A8_EINVAL, "%s: row strides smaller than head_dim, or negative", what);
    if (rs[i] % 8 != 0 || hs[i] % 8 != 0) return fail(W8A8_EALIGN, "%s: strides must be multiples of 8 elements", what);
  }
  if (H > 1 && o_head_stride < D) return fail(W8A8_EINVAL, "%s: o's heads overlap, stride %lld", what, (long long)o_head_stride);
  if (std::max(rs[0], rs[1]) >= (int64_t(1) << 24))
    return fail(W8A8_ENOTSUP, "%s: k or v rows %lld elements apart", what, (long long)std::max(rs[0], rs[1]));
  if ((uintptr_t)q % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)o % 16 || (uintptr_t)workspace % 16 ||
      (uintptr_t)q_start_dev % 4 || (uintptr_t)lse % 4)
    return fail(W8A8_EALIGN, "%s: q, k, v, o and the workspace 16-byte, q_start and lse 4-byte aligned", what);
  const SinkPlan pl = sink_plan(H, KV, Tq, Tk, D, q_start, window, sinks);
  SinkParams p{};
  p.q = q; p.qhs = hs[2]; p.qrs = rs[2]; p.k = k; p.khs = hs[0]; p.krs = rs[0]; p.v = v; p.vhs = hs[1]; p.vrs = rs[1];
  p.out.o = o; p.out.ohs = hs[3]; p.out.ors = rs[3]; p.out.lse = lse; p.out.KV = int(KV); p.out.G = int(H / KV);
  p.out.rows = int(Tq * (H / KV)); p.out.nparts = pl.nparts;
  p.out.part_o = static_cast<float*>(workspace);
  p.out.part_ml = p.out.part_o + H * Tq * pl.nparts * D;
  p.start_dev = q_start_dev; p.start = int(std::max<int64_t>(q_start, 0)); p.Tq = int(Tq); p.Tk = int(Tk);
  p.window = int(window); p.sinks = window > 0 ? int(sinks) : 0; p.ntiles = pl.ntiles;
  p.c = scale * 1.4426950408889634f;
  if (D == 128)
    sink_launch<128>(p, pl.rt, stream);
  else if (D == 256)
    sink_launch<256>(p, pl.rt, stream);
  else
    sink_launch<512>(p, pl.rt, stream);
  return check_launch(what);
}
