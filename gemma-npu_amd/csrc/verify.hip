// Drafted tokens tested against the target's probabilities, and the token that follows drawn, from given random
// numbers: what stands between a drafted run's attention and the next draft.
//
//   p_i = softmax(logits[i] / T): the target after the context (i = 0) and after node i - 1;
//   q_m = softmax(draft[m] / T): what node m's token was drawn from, or without draft logits that token with certainty.
//
// A chain accepts node m while u[m] q_m(t_m) < p_m(t_m).  A tree (parents as attention of a tree of drafted tokens
// takes them; no draft logits) is walked in the order of its nodes: the children of the node reached so far are
// tested one after the other, u[m] (1 - s) < p(t_m) with s the probability of the tokens refused beside it, which
// have none left.  The next token is the first whose running sum of r passes u[N] times the sum of all, with r = p of
// the row reached, less q of the chain's refused node where that is less (max(p - q, 0)), or without the refused
// siblings' tokens; where that leaves nothing, p.  Accepted tokens and the next one are then distributed as the target's own samples.  The
// reference decodes greedily, one token at a time (gemma_npu.py:292-295).
//
// verify_stat_kernel reads every row once: a workgroup takes tiles of 4096 logits of one row into registers, one or a few
// (verify_tiles), and leaves their sum of exponentials.  verify_draw_kernel, 2048 tokens a workgroup, joins those of the call's
// rows (each workgroup for itself: a few KiB), decides, and sums r over its tokens; the last workgroup of a request
// to arrive finds the chunk in which the running sum passes its bound, and the token in it.  Exponentials and sums are
// in 64 bits: of 262144 tokens two neighbours' running sums differ by a few 1e-6 of the whole, and sums of
// 32-bit terms would draw another token once in some hundred calls.  Every sum has a fixed order.  4 drafted tokens of
// 262144 (9 rows, 4.7 MB): 6 us and 13; a tree of 48 (49 rows, 26 MB): 16.4 and 19.5; 8 requests of up to 8, 4 on average, in
// fp32 (72 rows, 75 MB): 23 and 19.  The statistics take 1.2-1.3 ps a logit, where their 17 64-bit operations are issued in
// 0.58: a workgroup's tiles are few, and it begins with a load, a maximum over all of it and a barrier.
#include <algorithm>

#include "w8a8_common.h"

namespace w8a8 {

constexpr int VERIFY_MAX_NODES = 128;
constexpr int VERIFY_STAT_E = 16, VERIFY_STAT = 256 * VERIFY_STAT_E;  // logits of a thread, of a workgroup: statistics
constexpr int VERIFY_DRAW_E = 8, VERIFY_DRAW = 256 * VERIFY_DRAW_E;   // and the draw

// A difference p - q of less than this share of p is what rounding left of two equal ones: exponentials are off by 6e-14, a
// row's and those that join its chunks, and sums by some 1e-14, and a row that begins elsewhere in its 16-byte words is cut
// into other chunks.
constexpr double VERIFY_NONE = 0x1p-40;

constexpr int VERIFY_LINE = 32;                   // a request's arrival count has a cache line of its own

struct VerifyStat {
  double sum;  // of exponentials against `top`; NaN with a NaN or +inf among the logits
  float top;   // one of the largest logits
};

struct VerifyParams {
  const void* x; int64_t xgs, xrs;          // target logits [B, N + 1, V] (element strides of requests and rows)
  const void* d; int64_t dgs, drs;          // draft logits [B, N, V], or null
  const int64_t* tok; int64_t ts;           // [B, N] (request stride)
  const float* u; int64_t us;               // [B, N + 1]
  const int32_t* parents; int64_t ps;       // [B, N] of stride ps (0: the same for all), or null: a chain
  const int32_t* lengths;                   // [B], or null: N
  int B, N, V, nst, ndr;                    // chunks of a row: statistics, draw
  int tiles;                                // of 4096 logits in a chunk of the statistics
  double inv_t;
  VerifyStat* stat;                         // [B (N + 1) + B N][nst]
  double* sums;                             // [B][ndr] of r
  int* arrived;                             // [B][VERIFY_LINE], the first of each
  int32_t* count; int64_t* path; int64_t* next;  // [B], [B, N], [B]
};

__device__ __forceinline__ int verify_length(const VerifyParams& p, int b) {
  return p.lengths ? max(0, min(p.lengths[b], p.N)) : p.N;
}

// Elements of X in front of a row that bring it to 16 bytes: a row's chunks are cut at whole 16-byte words.
template <class X>
__device__ __forceinline__ int verify_lead(const X* row) {
  return int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(X));
}

__device__ __forceinline__ float verify_value(float x) { return x; }
__device__ __forceinline__ float verify_value(uint16_t x) { return bf16_to_f32(x); }

// Sixteen bytes of a row from element i on (may begin before the row or end behind it: -inf there), and their values.
template <class X>
__device__ __forceinline__ v4u verify_load(const X* row, int i, int V) {
  constexpr int E = 16 / sizeof(X);
  if (i >= 0 && i + E <= V) return *reinterpret_cast<const v4u*>(row + i);
  v4u w;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(X) == 4) {
      w[j] = i + j >= 0 && i + j < V ? __float_as_uint(row[i + j]) : 0xff800000u;
    } else {
      w[j] = i + 2 * j >= 0 && i + 2 * j < V ? uint32_t(row[i + 2 * j]) : 0xff80u;
      w[j] |= (i + 2 * j + 1 >= 0 && i + 2 * j + 1 < V ? uint32_t(row[i + 2 * j + 1]) : 0xff80u) << 16;
    }
  }
  return w;
}
template <class X>
__device__ __forceinline__ float verify_at(v4u w, int e) {
  if constexpr (sizeof(X) == 4) return __uint_as_float(w[e]);
  return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
}

// A workgroup's sum, in an order of its own, for every thread.
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <class X>
__global__ __launch_bounds__(256) void verify_stat_kernel(VerifyParams p) {
  constexpr int E = 16 / sizeof(X), NV = VERIFY_STAT_E / E;
  __shared__ float redm[4];
  __shared__ double red[4];
  const int t = threadIdx.x, ch = blockIdx.x % p.nst, row = blockIdx.x / p.nst;
  if (ch == 0 && row < p.B && t == 0) p.arrived[row * VERIFY_LINE] = 0;  // for the next kernel
  const int targets = p.B * (p.N + 1);
  const X* x;
  if (row < targets) {
    const int b = row / (p.N + 1), i = row % (p.N + 1);
    if (i > verify_length(p, b)) return;
    x = static_cast<const X*>(p.x) + int64_t(b) * p.xgs + int64_t(i) * p.xrs;
  } else {
    const int b = (row - targets) / p.N, i = (row - targets) % p.N;
    if (i >= verify_length(p, b)) return;
    x = static_cast<const X*>(p.d) + int64_t(b) * p.dgs + int64_t(i) * p.drs;
  }
  // Against the largest of the first tile's logits, which a thread whose own are far larger leaves (64 bits hold
  // e^600 of it); the next tile's logits are on their way while this one's exponentials are made.
  auto load = [&](int tile, v4u(&w)[NV]) __attribute__((always_inline)) {
    const int base = tile * VERIFY_STAT - verify_lead(x);
#pragma unroll
    for (int c = 0; c < NV; ++c) w[c] = verify_load(x, base + E * (t + 256 * c), p.V);
  };
  double s = 0.0;
  float m = -__builtin_inff();
  bool bad = false;
  v4u w[NV];
  const int first = ch * p.tiles, end = min(first + p.tiles, (p.V + VERIFY_STAT + 6) / VERIFY_STAT);
  load(first, w);
#pragma unroll 1
  for (int tile = first; tile < end; ++tile) {
    v4u ahead[NV];
    if (tile + 1 < end) load(tile + 1, ahead);
    float top = -__builtin_inff();
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = verify_at<X>(w[c], e);
        top = fmaxf(top, v);
        bad |= !(v < __builtin_inff());
      }
    if (tile == first) {
      m = top;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
      if ((t & 63) == 0) redm[t >> 6] = m;
      __syncthreads();
      m = fmaxf(fmaxf(redm[0], redm[1]), fmaxf(redm[2], redm[3]));
    } else if ((double(top) - double(m)) * p.inv_t > 300.0) {
      s *= exp_64((double(m) - double(top)) * p.inv_t);
      m = top;
    }
    if (m > -__builtin_inff())
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < E; ++e) s += exp_64((double(verify_at<X>(w[c], e)) - double(m)) * p.inv_t);
#pragma unroll
    for (int c = 0; c < NV; ++c) w[c] = ahead[c];
  }
  float top = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  __syncthreads();
  if ((t & 63) == 0) redm[t >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(redm[0], redm[1]), fmaxf(redm[2], redm[3]));
  if (m != top) s *= exp_64((double(m) - double(top)) * p.inv_t);
  if (bad) s = __builtin_nan("");
  s = block_sum(s, red);
  if (t == 0) p.stat[int64_t(row) * p.nst + ch] = VerifyStat{s, top};
}

// The kernel below runs each of its parts once, in one workgroup after the other: what it waits for is memory and its
// own instructions on their way to the CU, so exponentials stand in loops rather than side by side.
//
// Where among 256 threads' values v, in their order, the running sum passes `bound`: the first thread with
// v > 0 whose inclusive sum does (rounding may leave none: the last with v > 0; -1: none has), and the sum before it.
struct VerifyFound {
  int thread;
  double before, total;
};
__device__ __forceinline__ VerifyFound verify_find(double v, double share, bool relative, double* red, double* before, int (*at)[4]) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  double w = v;
#pragma unroll 1
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(w, o, 64);
    if (lane >= o) w += up;
  }
  const double ex = __shfl_up(w, 1, 64);
  __syncthreads();
  if (lane == 63) red[wave] = w;
  __syncthreads();
  const double r0 = red[0], r1 = r0 + red[1], r2 = r1 + red[2], total = r2 + red[3];
  const double off = wave == 0 ? 0.0 : wave == 1 ? r0 : wave == 2 ? r1 : r2;
  const double bound = relative ? share * total : share;
  const uint64_t has = __builtin_amdgcn_ballot_w64(v > 0.0), past = __builtin_amdgcn_ballot_w64(v > 0.0 && off + w > bound);
  if (lane == 0) {
    at[0][wave] = past ? 64 * wave + __builtin_ctzll(past) : 256;
    at[1][wave] = has ? 64 * wave + 63 - __builtin_clzll(has) : -1;
  }
  __syncthreads();
  int who = min(min(at[0][0], at[0][1]), min(at[0][2], at[0][3]));
  if (who == 256) who = max(max(at[1][0], at[1][1]), max(at[1][2], at[1][3]));
  if (t == who) *before = lane ? off + ex : off;
  __syncthreads();
  return VerifyFound{who, *before, total};
}

// What a request's rows and nodes come to.
struct VerifyState {
  float top[2 * VERIFY_MAX_NODES + 1];       // rows 0 .. N the target's, N + 1 .. 2 N the draft's
  double sum[2 * VERIFY_MAX_NODES + 1];
  double pt[VERIFY_MAX_NODES];
  int par[VERIFY_MAX_NODES];
  bool ok[VERIFY_MAX_NODES];
  float u[VERIFY_MAX_NODES + 1];
  int64_t tok[VERIFY_MAX_NODES];
  int64_t gone[VERIFY_MAX_NODES];            // tokens without probability
  int path[VERIFY_MAX_NODES];
  int count, row, ngone, qrow;               // accepted, the row that the next token is drawn from, its draft row or -1
};

constexpr int VERIFY_STAGE = 1536;           // chunks' statistics in LDS at a time, at least a row's

template <class X>
__global__ __launch_bounds__(256, 5) void verify_draw_kernel(VerifyParams p) {
  constexpr int E = 16 / sizeof(X), NV = VERIFY_DRAW_E / E, PAD = VERIFY_DRAW_E + 1;
  __shared__ VerifyState s;
  __shared__ double red[4], before_s;
  __shared__ int at_s[2][4];
  __shared__ uint32_t bits[VERIFY_DRAW / 32];
  __shared__ int last, chunk_s;
  // the rows' statistics; then the chunk's logits (the target's and the draft's), then r in their places
  __shared__ union {
    struct {
      double sum[VERIFY_STAGE];
      float top[VERIFY_STAGE];
    } st;
    v2f x[256 * PAD];
    double r[256 * PAD];
  } sh;
  const int t = threadIdx.x, lane = t & 63, ch = blockIdx.x % p.ndr, b = blockIdx.x / p.ndr;
  const int N = p.N, len = verify_length(p, b);
  const bool tree = p.parents != nullptr, drafts = p.d != nullptr;
  const X* const target = static_cast<const X*>(p.x) + int64_t(b) * p.xgs;
  const X* const draft = drafts ? static_cast<const X*>(p.d) + int64_t(b) * p.dgs : nullptr;

  // ---- what the nodes need from memory, asked for at once ------------------------------------------------------
  int64_t tok = -1;
  int par = -2;
  if (t <= N) s.u[t] = p.u[int64_t(b) * p.us + t];
  if (t < len) {
    tok = p.tok[int64_t(b) * p.ts + t];
    par = tree ? p.parents[int64_t(b) * p.ps + t] : t - 1;
    if (par < -1 || par >= t) par = -2;  // unused
  }
  const bool in = tok >= 0 && tok < p.V && par >= -1;
  X xt = X(0), xd = X(0);
  if (in) {
    xt = target[int64_t(par + 1) * p.xrs + tok];
    if (drafts) xd = draft[int64_t(t) * p.drs + tok];
  }
  // ---- the rows' maxima and sums: staged, then 16 lanes a row -------------------------------------------------
  const int rows = len + 1 + (drafts ? len : 0), group = VERIFY_STAGE / p.nst;
  for (int r0 = 0; r0 < rows; r0 += group) {
    const int n = min(group, rows - r0);
    // rows len + 1 .. are the draft's, behind the B (N + 1) of the target
    const int64_t shift = int64_t(p.B) * (N + 1) + int64_t(b) * N - (len + 1);
    if (r0) __syncthreads();
#pragma unroll 4
    for (int i = t >> 6; i < n; i += 4) {  // a wave a row
      const int r = r0 + i;
      const VerifyStat* const st = p.stat + (r <= len ? int64_t(b) * (N + 1) + r : shift + r) * p.nst;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // (at most 128 chunks)
        const int c = lane + 64 * h;
        const VerifyStat v = st[min(c, p.nst - 1)];
        if (c < p.nst) {
          sh.st.sum[i * p.nst + c] = v.sum;
          sh.st.top[i * p.nst + c] = v.top;
        }
      }
    }
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += 16) {
      const int i = min(i0 + (t >> 4), n - 1), base = i * p.nst;
      float m = -__builtin_inff();
      for (int c = t & 15; c < p.nst; c += 16) m = fmaxf(m, sh.st.top[base + c]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
      double z = 0.0;
#pragma unroll 1
      for (int c = t & 15; c < p.nst; c += 16) {
        const float top = sh.st.top[base + c];
        // (a chunk of -inf alone has a sum of 0, or NaN)
        z += sh.st.sum[base + c] * (top == m ? 1.0 : exp_64((double(top) - double(m)) * p.inv_t));
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
      if (i0 + (t >> 4) < n && (t & 15) == 0) {
        const int r = r0 + i, at = r <= len ? r : N - len + r;
        s.top[at] = m;
        s.sum[at] = z;
      }
    }
  }
  if (t < VERIFY_DRAW / 32) bits[t] = 0u;
  __syncthreads();
  // ---- the nodes' probabilities ------------------------------------------------------------------------------
  if (t < N) {
    double pq[2] = {0.0, tok >= 0 && tok < p.V ? 1.0 : 0.0};
    if (in) {
      double v = double(verify_value(xt)), keep = 0.0;
#pragma unroll 1
      for (int h = 0; h < (drafts ? 2 : 1); ++h) {
        const int r = h ? N + 1 + t : par + 1;
        const double e = exp_64((v - double(s.top[r])) * p.inv_t) / s.sum[r];
        if (h == 0) keep = e;
        else pq[1] = e;
        v = double(verify_value(xd));
      }
      pq[0] = keep;
    }
    s.pt[t] = pq[0];
    s.par[t] = par;
    s.tok[t] = tok;
    s.ok[t] = double(s.u[t]) * pq[1] < pq[0] && t < len;  // (a chain's test)
  }
  __syncthreads();
  // ---- the walk, in one wave -----------------------------------------------------------------------------------
  if (t < 64) {
    int at = -1, count = 0, ngone = 0;
    if (!tree) {  // as far as every test holds
      const uint64_t m0 = __builtin_amdgcn_ballot_w64(lane < len && !s.ok[lane]);
      const uint64_t m1 = __builtin_amdgcn_ballot_w64(lane + 64 < len && !s.ok[min(lane + 64, VERIFY_MAX_NODES - 1)]);
      count = m0 ? __builtin_ctzll(m0) : m1 ? 64 + __builtin_ctzll(m1) : len;
      at = count - 1;
      ngone = count < len ? 1 : 0;
      if (ngone && lane == 0) s.gone[0] = s.tok[count];
      if (lane < count) s.path[lane] = lane;
      if (lane + 64 < count) s.path[lane + 64] = lane + 64;
    } else {  // the children of the node reached, in order
      double gone = 0.0;
      for (int from = 0;;) {
        const int i0 = from + lane, i1 = from + 64 + lane;
        const uint64_t m0 = __builtin_amdgcn_ballot_w64(i0 < N && s.par[min(i0, VERIFY_MAX_NODES - 1)] == at);
        const uint64_t m1 = __builtin_amdgcn_ballot_w64(i1 < N && s.par[min(i1, VERIFY_MAX_NODES - 1)] == at);
        if ((m0 | m1) == 0) break;
        const int m = from + (m0 ? __builtin_ctzll(m0) : 64 + __builtin_ctzll(m1));
        const int64_t mt = s.tok[m];
        bool again = false;  // its token was refused beside it
        for (int j = lane; j < ngone; j += 64) again |= s.gone[j] == mt;
        const double pm = __builtin_amdgcn_ballot_w64(again) ? 0.0 : s.pt[m];
        if (double(s.u[m]) * (1.0 - gone) < pm) {
          if (lane == 0) s.path[count] = m;
          at = m;
          ++count;
          ngone = 0;
          gone = 0.0;
        } else {
          if (lane == 0) s.gone[ngone] = mt;
          ++ngone;
          gone += pm;
        }
        from = m + 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the refused tokens are read by the other lanes
        __builtin_amdgcn_wave_barrier();
      }
    }
    if (lane == 0) {
      s.count = count;
      s.row = at + 1;
      s.qrow = drafts && ngone ? at + 1 : -1;  // (a chain's refused node)
      s.ngone = drafts ? 0 : ngone;
    }
  }
  __syncthreads();
  const int row = s.row, qrow = s.qrow;
  if (ch == 0) {
    if (t < N) p.path[int64_t(b) * N + t] = t < s.count ? s.path[t] : -1;
    if (t == 0) p.count[b] = s.count;
  }
  // ---- r over a chunk's tokens, eight in a row a thread: this workgroup's, and for the last one to arrive then
  // those of the chunk in which the running sum passes its bound
  const X* const x = target + int64_t(row) * p.xrs;
  const X* const q = qrow >= 0 ? draft + int64_t(qrow) * p.drs : nullptr;
  const int lead = verify_lead(x);
  const bool alike = q && verify_lead(q) == lead;
  const double top = s.top[row], inv = 1.0 / s.sum[row];
  const double qtop = q ? double(s.top[N + 1 + qrow]) : 0.0, qinv = q ? 1.0 / s.sum[N + 1 + qrow] : 0.0;
  bool plain = false;  // nothing is left of p (where rounding took it all): p itself
  double bound = 0.0;
  int c = ch;
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    const int base = c * VERIFY_DRAW - lead;
    for (int j = t; j < s.ngone; j += 256) {  // the chunk's tokens without probability
      const int64_t at = s.gone[j] - base;
      if (at >= 0 && at < VERIFY_DRAW) atomicOr(&bits[at >> 5], 1u << (at & 31));
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int i = base + VERIFY_DRAW_E * t + E * v;
      const v4u y = verify_load(x, i, p.V);
      v4u z;
      if (alike && !plain) z = verify_load(q, i, p.V);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float d = -__builtin_inff();
        if (q && !plain) d = alike ? verify_at<X>(z, e) : (i + e >= 0 && i + e < p.V ? verify_value(q[i + e]) : d);
        sh.x[PAD * t + E * v + e] = v2f{verify_at<X>(y, e), d};
      }
    }
    __syncthreads();
    const uint32_t out = plain ? 0u : bits[t >> 2] >> (8 * (t & 3));
    double sum = 0.0;
#pragma unroll 2
    for (int e = 0; e < VERIFY_DRAW_E; ++e) {
      const v2f w = sh.x[PAD * t + e];
      double a = exp_64((double(w[0]) - top) * p.inv_t) * inv;
      if (q && !plain) {
        const double less = a - exp_64((double(w[1]) - qtop) * p.inv_t) * qinv;
        a = less > a * VERIFY_NONE ? less : 0.0;
      }
      a = a > 0.0 && !((out >> e) & 1u) ? a : 0.0;  // (false for NaN)
      sh.r[PAD * t + e] = a;
      sum += a;
    }
    if (pass) {  // the token
      const VerifyFound f = verify_find(sum, bound, false, red, &before_s, at_s);
      if (t == max(f.thread, 0)) {
        double at = f.before;
        int first = -1, any = 0;
        for (int e = 0; e < VERIFY_DRAW_E; ++e) {
          const double r = sh.r[PAD * t + e];
          at += r;
          if (r > 0.0) {
            any = e;
            if (first < 0 && at > bound) first = e;
          }
        }
        p.next[b] = max(0, base + VERIFY_DRAW_E * t + (first >= 0 ? first : any));
      }
      return;
    }
    sum = block_sum(sum, red);
    double* const sums = p.sums + int64_t(b) * p.ndr;
    if (t == 0) {
      // Write-through stores and a wait instead of a release and an acquire, which write back and invalidate the
      // XCD's L2 for every workgroup; what the last one reads of the others' is read past the L2 as well.
      __hip_atomic_store(sums + ch, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
      __builtin_amdgcn_s_waitcnt(0);
      last = __hip_atomic_fetch_add(p.arrived + b * VERIFY_LINE, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM) == p.ndr - 1;
    }
    __syncthreads();
    if (!last) return;
    // the chunk, among `per` of each thread
    const int per = (p.ndr + 255) / 256, c0 = t * per, c1 = min(c0 + per, p.ndr);
    auto chunk_sum = [&](int i) __attribute__((always_inline)) {
      if (!plain) return __hip_atomic_load(sums + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
      double r = 0.0;  // (rare)
#pragma unroll 1
      for (int j = max(0, i * VERIFY_DRAW - lead); j < min(p.V, (i + 1) * VERIFY_DRAW - lead); ++j) {
        const double a = exp_64((double(verify_value(x[j])) - top) * p.inv_t) * inv;
        r += a > 0.0 ? a : 0.0;
      }
      return r;
    };
    VerifyFound f;
#pragma unroll 1
    for (;;) {
      double mine = 0.0;
#pragma unroll 1
      for (int i = c0; i < c1; ++i) mine += chunk_sum(i);
      f = verify_find(mine, double(s.u[N]), true, red, &before_s, at_s);
      // (without a distribution, NaN or nothing, there is nothing to draw from)
      if (f.total > 0.0 || plain || !(s.sum[row] > 0.0)) break;
      plain = true;
    }
    if (!(f.total > 0.0) || !(f.total < __builtin_inf()) || !(s.sum[row] > 0.0)) {
      if (t == 0) p.next[b] = -1;
      return;
    }
    bound = double(s.u[N]) * f.total;
    if (t == f.thread) {
      double at = f.before, from = at;
      int got = -1;
#pragma unroll 1
      for (int i = c0; i < c1; ++i) {
        const double v = per == 1 ? 1.0 : chunk_sum(i);
        if (v > 0.0) {
          got = i;
          from = at;
          if (at + v > bound) break;
        }
        at += v;
      }
      chunk_s = got;
      before_s = from;
    }
    if (t < VERIFY_DRAW / 32) bits[t] = 0u;
    __syncthreads();
    c = chunk_s;
    bound -= before_s;
    __syncthreads();
  }
}

}  // namespace w8a8

using namespace w8a8;

// Chunks of a row, which begins up to 7 elements behind a whole 16-byte word.
static int64_t verify_chunks(int64_t V, int64_t chunk) { return (V + 7 + chunk - 1) / chunk; }
// Tiles of 4096 logits in a chunk of the statistics: as many as leave six workgroups for every CU (the fewer chunks, the
// fewer each workgroup of the draw joins; tree of 48 of 262144, 2 tiles a chunk for 1: draw 23.0 -> 19.5 us, statistics
// 16.8 -> 16.4), and a row at most 128 chunks.
static int64_t verify_tiles(int64_t rows, int64_t V) {
  const int64_t tiles = verify_chunks(V, VERIFY_STAT);
  return std::max((tiles + 127) / 128, std::min<int64_t>(8, rows * tiles / 1500));
}
static int64_t verify_stats(int64_t rows, int64_t V) { return verify_chunks(V, VERIFY_STAT * std::max<int64_t>(1, verify_tiles(rows, V))); }
// Workgroups of a launch: 2^32 threads are too many.
constexpr int64_t VERIFY_BLOCKS = (int64_t(1) << 24) - 1;
static bool verify_shape_ok(int64_t B, int64_t N, int64_t V) {
  return B >= 1 && N >= 0 && N <= VERIFY_MAX_NODES && V >= 1 && V < (int64_t(1) << 30) &&
         B <= (int64_t(1) << 22) && B * (2 * N + 1) * verify_chunks(V, VERIFY_STAT) < (int64_t(1) << 31) &&
         B * (N + 1) * verify_stats(B * (N + 1), V) <= VERIFY_BLOCKS && B * verify_chunks(V, VERIFY_DRAW) <= VERIFY_BLOCKS;
}

static int64_t verify_sums_at(int64_t B, int64_t N, int64_t V) { return B * (2 * N + 1) * verify_stats(B * (N + 1), V) * int64_t(sizeof(VerifyStat)); }

extern "C" int64_t w8a8_verify_drafts_workspace_bytes(int64_t B, int64_t N, int64_t V) {
  if (!verify_shape_ok(B, N, V)) return -1;
  return verify_sums_at(B, N, V) + B * verify_chunks(V, VERIFY_DRAW) * 8 + B * VERIFY_LINE * 4;
}

extern "C" int w8a8_verify_drafts(const void* logits, const void* draft, int logits_are_f32, int64_t group_stride,
                                  int64_t row_stride, int64_t draft_group_stride, int64_t draft_row_stride,
                                  const int64_t* tokens, int64_t token_stride, const float* uniforms,
                                  int64_t uniform_stride, const int32_t* parents, int64_t parent_stride,
                                  const int32_t* lengths, int64_t B, int64_t N, int64_t V, double temperature,
                                  int32_t* accepted, int64_t* path, int64_t* next, void* workspace,
                                  int64_t workspace_bytes, hipStream_t stream) {
  const char* what = "verify_drafts";
  if (N > VERIFY_MAX_NODES) return fail(W8A8_ENOTSUP, "%s: %lld drafted tokens (at most %d)", what, (long long)N, VERIFY_MAX_NODES);
  if (!verify_shape_ok(B, N, V))
    return fail(W8A8_EINVAL, "%s: B=%lld N=%lld V=%lld", what, (long long)B, (long long)N, (long long)V);
  if (!(temperature > 0.0) || temperature == __builtin_inf() || 1.0 / temperature == __builtin_inf())
    return fail(W8A8_EINVAL, "%s: the temperature must be positive", what);
  if (draft && parents) return fail(W8A8_ENOTSUP, "%s: a tree is verified without draft logits", what);
  const int64_t rows = B * (N + 1 + (draft ? N : 0));
  if (rows * verify_stats(B * (N + 1), V) > VERIFY_BLOCKS)
    return fail(W8A8_EINVAL, "%s: B=%lld N=%lld V=%lld with draft logits", what, (long long)B, (long long)N, (long long)V);
  if (!logits || !uniforms || !accepted || !next || (N > 0 && (!tokens || !path)))
    return fail(W8A8_EINVAL, "%s: null pointer", what);
  if ((N > 0 && row_stride < V) || (B > 1 && group_stride < 0) || (draft && N > 1 && draft_row_stride < V) ||
      (draft && B > 1 && draft_group_stride < 0) || (B > 1 && (token_stride < 0 || uniform_stride < 0 || parent_stride < 0)))
    return fail(W8A8_EINVAL, "%s: row strides smaller than V, or negative", what);
  const int64_t need = w8a8_verify_drafts_workspace_bytes(B, N, V);
  if (!workspace || workspace_bytes < need)
    return fail(W8A8_EINVAL, "%s: workspace of %lld bytes, %lld needed", what, (long long)(workspace ? workspace_bytes : 0),
                (long long)need);
  const uintptr_t es = logits_are_f32 ? 4 : 2;
  if ((uintptr_t)logits % es || (uintptr_t)draft % es || (uintptr_t)tokens % 8 || (uintptr_t)uniforms % 4 ||
      (uintptr_t)parents % 4 || (uintptr_t)lengths % 4 || (uintptr_t)accepted % 4 || (uintptr_t)path % 8 ||
      (uintptr_t)next % 8 || (uintptr_t)workspace % 8)
    return fail(W8A8_EALIGN, "%s: every operand aligned to its type, the workspace to 8 bytes", what);
  VerifyParams p{};
  p.x = logits; p.xgs = B > 1 ? group_stride : 0; p.xrs = N > 0 ? row_stride : 0;
  p.d = N > 0 ? draft : nullptr; p.dgs = B > 1 ? draft_group_stride : 0; p.drs = N > 1 ? draft_row_stride : 0;
  p.tok = tokens; p.ts = B > 1 ? token_stride : 0; p.u = uniforms; p.us = B > 1 ? uniform_stride : 0;
  p.parents = N > 0 ? parents : nullptr; p.ps = B > 1 ? parent_stride : 0; p.lengths = lengths;
  p.B = int(B); p.N = int(N); p.V = int(V); p.nst = int(verify_stats(B * (N + 1), V));
  p.tiles = int(std::max<int64_t>(1, verify_tiles(B * (N + 1), V))); p.ndr = int(verify_chunks(V, VERIFY_DRAW));
  p.inv_t = 1.0 / temperature;
  p.stat = static_cast<VerifyStat*>(workspace);
  p.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + verify_sums_at(B, N, V));
  p.arrived = reinterpret_cast<int*>(p.sums + B * p.ndr);
  p.count = accepted; p.path = path; p.next = next;
  const dim3 g1{unsigned(rows * p.nst), 1, 1}, g2{unsigned(B) * unsigned(p.ndr), 1, 1};
  if (logits_are_f32) {
    verify_stat_kernel<float><<<g1, 256, 0, stream>>>(p);
    verify_draw_kernel<float><<<g2, 256, 0, stream>>>(p);
  } else {
    verify_stat_kernel<uint16_t><<<g1, 256, 0, stream>>>(p);
    verify_draw_kernel<uint16_t><<<g2, 256, 0, stream>>>(p);
  }
  return check_launch("verify_drafts");
}
