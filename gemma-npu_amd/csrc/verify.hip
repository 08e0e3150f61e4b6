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
// siblings' tokens.  Accepted tokens and the next one are then distributed as the target's own samples.  The
// reference decodes greedily, one token at a time (gemma_npu.py:292-295).
//
// verify_stat_kernel reads every row once: a workgroup takes 8192 logits of one row into registers and leaves
// their maximum and sum of exponentials.  verify_draw_kernel, 8192 tokens a workgroup, joins those of the call's
// rows (each workgroup for itself: a few KiB), decides, and sums r over its tokens; the last workgroup of a request
// to arrive finds the chunk in which the running sum passes its bound, and the token in it.  Exponentials and sums are
// in 64 bits: of 262144 tokens two neighbours' running sums differ by a few 1e-6 of the whole, and sums of
// 32-bit terms would draw another token once in some hundred calls.  Every sum has a fixed order.
#include <algorithm>

#include "w8a8_common.h"

namespace w8a8 {

constexpr int VERIFY_MAX_NODES = 128;
constexpr int VERIFY_E = 32;                      // logits of a thread
constexpr int VERIFY_CHUNK = 256 * VERIFY_E;

struct VerifyStat {
  double sum;  // of exponentials against the maximum; NaN with a NaN or +inf among the logits
  float top;
};

struct VerifyParams {
  const void* x; int64_t xgs, xrs;          // target logits [B, N + 1, V] (element strides of requests and rows)
  const void* d; int64_t dgs, drs;          // draft logits [B, N, V], or null
  const int64_t* tok; int64_t ts;           // [B, N] (request stride)
  const float* u; int64_t us;               // [B, N + 1]
  const int32_t* parents; int64_t ps;       // [B, N] of stride ps (0: the same for all), or null: a chain
  const int32_t* lengths;                   // [B], or null: N
  int B, N, V, nch;
  double inv_t;
  VerifyStat* stat;                         // [B (N + 1) + B N][nch]
  double* sums;                             // [B][nch] of r
  int* arrived;                             // [B]
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

// Sixteen bytes of a row from element i on (may begin before the row or end behind it: -inf there).
template <class X>
__device__ __forceinline__ void verify_load(const X* row, int i, int V, float* v) {
  constexpr int E = 16 / sizeof(X);
  if (i >= 0 && i + E <= V) {
    const v4u w = *reinterpret_cast<const v4u*>(row + i);
#pragma unroll
    for (int e = 0; e < E; ++e)
      v[e] = sizeof(X) == 4 ? __uint_as_float(w[e & 3])
                            : __uint_as_float(e & 1 ? w[(e >> 1) & 3] & 0xffff0000u : w[(e >> 1) & 3] << 16);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = i + e >= 0 && i + e < V ? verify_value(row[i + e]) : -__builtin_inff();
  }
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
  constexpr int E = 16 / sizeof(X), NV = VERIFY_E / E;
  __shared__ float redm[4];
  __shared__ double red[4];
  const int t = threadIdx.x, ch = blockIdx.x % p.nch, row = blockIdx.x / p.nch;
  if (ch == 0 && row < p.B && t == 0) p.arrived[row] = 0;  // for the next kernel
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
  const int base = ch * VERIFY_CHUNK - verify_lead(x);
  float v[VERIFY_E];
#pragma unroll
  for (int c = 0; c < NV; ++c) verify_load(x, base + E * (t + 256 * c), p.V, v + E * c);
  float m = -__builtin_inff();
  bool bad = false;
#pragma unroll
  for (int e = 0; e < VERIFY_E; ++e) {
    m = fmaxf(m, v[e]);
    bad |= !(v[e] < __builtin_inff());
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((t & 63) == 0) redm[t >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(redm[0], redm[1]), fmaxf(redm[2], redm[3]));
  double s = bad ? __builtin_nan("") : 0.0;
  if (m > -__builtin_inff())
#pragma unroll
    for (int e = 0; e < VERIFY_E; ++e) s += exp_64((double(v[e]) - double(m)) * p.inv_t);
  s = block_sum(s, red);
  if (t == 0) p.stat[int64_t(row) * p.nch + ch] = VerifyStat{s, m};
}

// What a request's rows and nodes come to.
struct VerifyState {
  float top[2 * VERIFY_MAX_NODES + 1];       // rows 0 .. N the target's, N + 1 .. 2 N the draft's
  double sum[2 * VERIFY_MAX_NODES + 1];
  double pt[VERIFY_MAX_NODES], qt[VERIFY_MAX_NODES];
  int par[VERIFY_MAX_NODES];
  float u[VERIFY_MAX_NODES + 1];
  int64_t tok[VERIFY_MAX_NODES];
  int64_t gone[VERIFY_MAX_NODES];            // tokens without probability
  int path[VERIFY_MAX_NODES];
  int count, row, ngone, qrow;               // accepted, the row that the next token is drawn from, its draft row or -1
};

template <class X>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyParams p) {
  constexpr int E = 16 / sizeof(X), NV = VERIFY_E / E;
  __shared__ VerifyState s;
  __shared__ double red[4], scan[256];
  __shared__ uint32_t bits[VERIFY_CHUNK / 32];
  __shared__ int last, found;
  __shared__ double before_s;
  const int t = threadIdx.x, lane = t & 63, ch = blockIdx.x % p.nch, b = blockIdx.x / p.nch;
  const int N = p.N, len = verify_length(p, b);
  const bool tree = p.parents != nullptr, drafts = p.d != nullptr;
  const X* const target = static_cast<const X*>(p.x) + int64_t(b) * p.xgs;
  const X* const draft = drafts ? static_cast<const X*>(p.d) + int64_t(b) * p.dgs : nullptr;

  // ---- the rows' maxima and sums, eight lanes a row ---------------------------------------------------------
  {
    const int rows = len + 1 + (drafts ? len : 0);
    for (int r0 = 0; r0 < rows; r0 += 32) {
      const int i = r0 + (t >> 3);
      const bool on = i < rows, own = i <= len;
      const int64_t row = own ? int64_t(b) * (N + 1) + i : int64_t(p.B) * (N + 1) + int64_t(b) * N + (i - len - 1);
      const VerifyStat* st = p.stat + row * p.nch;
      float m = -__builtin_inff();
      double z = 0.0;
      if (on)
        for (int c = t & 7; c < p.nch; c += 8) m = fmaxf(m, st[c].top);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
      if (on)
        for (int c = t & 7; c < p.nch; c += 8) {
          const VerifyStat v = st[c];
          // (a chunk of -inf alone has a sum of 0, or NaN)
          z = __builtin_fma(v.sum, v.top == m ? 1.0 : exp_64((double(v.top) - double(m)) * p.inv_t), z);
        }
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
      if (on && (t & 7) == 0) {
        const int at = own ? i : N + 1 + (i - len - 1);
        s.top[at] = m;
        s.sum[at] = z;
      }
    }
  }
  for (int m = t; m < VERIFY_CHUNK / 32; m += 256) bits[m] = 0u;
  __syncthreads();
  // ---- the nodes' probabilities ------------------------------------------------------------------------------
  if (t <= N) s.u[t] = p.u[int64_t(b) * p.us + t];
  if (t < N) {
    const int64_t tok = p.tok[int64_t(b) * p.ts + t];
    int par = tree ? p.parents[int64_t(b) * p.ps + t] : t - 1;
    if (t >= len || par < -1 || par >= t) par = -2;  // unused
    const bool in = tok >= 0 && tok < p.V;
    double pt = 0.0, qt = in ? 1.0 : 0.0;
    if (in && par >= -1 && par < len) {
      pt = exp_64((double(verify_value(target[int64_t(par + 1) * p.xrs + tok])) - double(s.top[par + 1])) * p.inv_t) / s.sum[par + 1];
      if (drafts)
        qt = exp_64((double(verify_value(draft[int64_t(t) * p.drs + tok])) - double(s.top[N + 1 + t])) * p.inv_t) / s.sum[N + 1 + t];
    }
    s.pt[t] = pt;
    s.qt[t] = qt;
    s.par[t] = par;
    s.tok[t] = tok;
  }
  __syncthreads();
  // ---- the walk, in one wave: the children of the node reached, in order ---------------------------------------
  if (t < 64) {
    int at = -1, count = 0, ngone = 0, from = 0;
    double gone = 0.0;
    for (;;) {
      // the next child of `at` behind `from`
      const int i0 = from + lane, i1 = from + 64 + lane;
      const uint64_t m0 = __builtin_amdgcn_ballot_w64(i0 < N && s.par[min(i0, VERIFY_MAX_NODES - 1)] == at);
      const uint64_t m1 = __builtin_amdgcn_ballot_w64(i1 < N && s.par[min(i1, VERIFY_MAX_NODES - 1)] == at);
      if ((m0 | m1) == 0) break;
      const int m = from + (m0 ? __builtin_ctzll(m0) : 64 + __builtin_ctzll(m1));
      const int64_t tok = s.tok[m];
      bool again = false;  // its token was refused beside it
      for (int j = lane; j < ngone; j += 64) again |= s.gone[j] == tok;
      const double pm = __builtin_amdgcn_ballot_w64(again) ? 0.0 : s.pt[m];
      const double need = tree ? double(s.u[m]) * (1.0 - gone) : double(s.u[m]) * s.qt[m];
      if (need < pm) {
        if (lane == 0) s.path[count] = m;
        at = m;
        ++count;
        ngone = 0;
        gone = 0.0;
      } else {
        if (lane == 0) s.gone[ngone] = tok;
        ++ngone;
        gone += pm;
        if (!tree) break;
      }
      from = m + 1;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the refused tokens are read by the other lanes
      __builtin_amdgcn_wave_barrier();
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
  // ---- r over this chunk's tokens -----------------------------------------------------------------------------
  const X* const x = target + int64_t(row) * p.xrs;
  const X* const q = qrow >= 0 ? draft + int64_t(qrow) * p.drs : nullptr;
  const int lead = verify_lead(x);
  const bool alike = q && verify_lead(q) == lead;
  const double top = s.top[row], inv = 1.0 / s.sum[row];
  const double qtop = q ? double(s.top[N + 1 + qrow]) : 0.0, qinv = q ? 1.0 / s.sum[N + 1 + qrow] : 0.0;
  auto mark = [&](int base) __attribute__((always_inline)) {  // the chunk's tokens without probability
    for (int j = t; j < s.ngone; j += 256) {
      const int64_t at = s.gone[j] - base;
      if (at >= 0 && at < VERIFY_CHUNK) atomicOr(&bits[at >> 5], 1u << (at & 31));
    }
  };
  // r of the 16 bytes of tokens from chunk element `off` on
  auto rest = [&](int base, int off, bool plain, double (&r)[E]) __attribute__((always_inline)) {
    float v[E], w[E];
    verify_load(x, base + off, p.V, v);
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = -__builtin_inff();
    if (q && !plain) {
      if (alike)
        verify_load(q, base + off, p.V, w);
      else
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (base + off + e >= 0 && base + off + e < p.V) w[e] = verify_value(q[base + off + e]);
    }
    const uint32_t out = plain ? 0u : bits[off >> 5] >> (off & 31);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      double a = exp_64((double(v[e]) - top) * p.inv_t) * inv;
      if (q && !plain) a -= exp_64((double(w[e]) - qtop) * p.inv_t) * qinv;
      r[e] = a > 0.0 && !((out >> e) & 1u) ? a : 0.0;  // (false for NaN)
    }
  };
  {
    const int base = ch * VERIFY_CHUNK - lead;
    mark(base);
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      double r[E];
      rest(base, E * (t + 256 * c), false, r);
#pragma unroll
      for (int e = 0; e < E; ++e) sum += r[e];
    }
    sum = block_sum(sum, red);
    if (t == 0) {
      double* at = p.sums + int64_t(b) * p.nch;
      __hip_atomic_store(at + ch, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = __hip_atomic_fetch_add(p.arrived + b, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == p.nch - 1;
    }
    __syncthreads();
    if (!last) return;
  }
  // ---- the last workgroup: the chunk, then the token in it ---------------------------------------------------
  const double* sums = p.sums + int64_t(b) * p.nch;
  const VerifyStat* st = p.stat + (int64_t(b) * (N + 1) + row) * p.nch;
  const int per = (p.nch + 255) / 256;
  bool plain = false;
  double mine = 0.0, total;
  auto chunk_sum = [&](int c) __attribute__((always_inline)) {
    if (!plain) return __hip_atomic_load(sums + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double r = st[c].sum * exp_64((double(st[c].top) - top) * p.inv_t) * inv;
    return r > 0.0 ? r : 0.0;
  };
  for (int pass = 0;; ++pass) {
    mine = 0.0;
    for (int c = t * per; c < min((t + 1) * per, p.nch); ++c) mine += chunk_sum(c);
    total = block_sum(mine, red);
    if (total > 0.0 || pass == 1) break;
    plain = true;  // nothing is left of p (where rounding took it all): p itself
  }
  if (!(total > 0.0) || !(total < __builtin_inf()) || !(s.sum[row] > 0.0)) {
    if (t == 0) p.next[b] = -1;  // no distribution
    return;
  }
  // exclusive running sums over the threads, in order
  auto running = [&](double v) __attribute__((always_inline)) {
    __syncthreads();
    scan[t] = v;
    __syncthreads();
    if (t < 64) {  // four in a row a lane
      const double a = scan[4 * t], c1 = a + scan[4 * t + 1], c2 = c1 + scan[4 * t + 2], c3 = c2 + scan[4 * t + 3];
      double w = c3;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(w, o, 64);
        if (lane >= o) w += up;
      }
      double ex = __shfl_up(w, 1, 64);
      if (lane == 0) ex = 0.0;
      scan[4 * t] = ex;
      scan[4 * t + 1] = ex + a;
      scan[4 * t + 2] = ex + c1;
      scan[4 * t + 3] = ex + c2;
    }
    __syncthreads();
    return scan[t];
  };
  const double bound = double(s.u[N]) * total;
  if (t == 0) found = p.nch, before_s = 0.0;
  double ex = running(mine);
  // the first chunk whose running sum passes the bound (its predecessors' does not); rounding may leave none: then
  // the last one that has any
  {
    int c0 = -1, cl = -1;
    double at = ex, bl = 0.0, b0 = 0.0;
    for (int c = t * per; c < min((t + 1) * per, p.nch); ++c) {
      const double v = chunk_sum(c);
      if (v > 0.0) cl = c, bl = at;
      if (c0 < 0 && at + v > bound && v > 0.0) c0 = c, b0 = at;
      at += v;
    }
    if (c0 >= 0) atomicMin(&found, c0);
    __syncthreads();
    const bool none = found == p.nch;
    __syncthreads();
    if (none && cl >= 0) atomicMax(&last, (cl << 1) | 1);  // (last is 1 now)
    __syncthreads();
    const int c = none ? last >> 1 : found;
    if (none ? cl == c : c0 == c) before_s = none ? bl : b0;
    __syncthreads();
    if (t == 0) found = c, last = 0;
    __syncthreads();
  }
  const int c = found, base = c * VERIFY_CHUNK - lead;
  const double left = bound - before_s;
  for (int m = t; m < VERIFY_CHUNK / 32; m += 256) bits[m] = 0u;
  __syncthreads();
  mark(base);
  __syncthreads();
  // 32 tokens in a row a thread
  double r[NV][E], sum = 0.0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    rest(base, VERIFY_E * t + E * v, plain, r[v]);
#pragma unroll
    for (int e = 0; e < E; ++e) sum += r[v][e];
  }
  double at = running(sum);
  int first = -1, final_ = -1;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      at += r[v][e];
      if (r[v][e] > 0.0) {
        final_ = VERIFY_E * t + E * v + e;
        if (first < 0 && at > left) first = final_;
      }
    }
  if (t == 0) found = VERIFY_CHUNK;
  __syncthreads();
  if (first >= 0) atomicMin(&found, first);
  if (final_ >= 0) atomicMax(&last, final_);
  __syncthreads();
  if (t == 0) p.next[b] = max(0, base + (found < VERIFY_CHUNK ? found : last));
}

}  // namespace w8a8

using namespace w8a8;

static int64_t verify_chunks(int64_t V) { return (V + 7 + VERIFY_CHUNK - 1) / VERIFY_CHUNK; }

static bool verify_shape_ok(int64_t B, int64_t N, int64_t V) {
  return B >= 1 && N >= 0 && N <= VERIFY_MAX_NODES && V >= 1 && V < (int64_t(1) << 30) &&
         B <= (int64_t(1) << 22) && B * (2 * N + 1) * verify_chunks(V) < (int64_t(1) << 31);
}

static int64_t verify_sums_at(int64_t B, int64_t N, int64_t V) { return B * (2 * N + 1) * verify_chunks(V) * int64_t(sizeof(VerifyStat)); }

extern "C" int64_t w8a8_verify_drafts_workspace_bytes(int64_t B, int64_t N, int64_t V) {
  if (!verify_shape_ok(B, N, V)) return -1;
  return verify_sums_at(B, N, V) + B * verify_chunks(V) * 8 + (B * 4 + 7) / 8 * 8;
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
  p.B = int(B); p.N = int(N); p.V = int(V); p.nch = int(verify_chunks(V));
  p.inv_t = 1.0 / temperature;
  p.stat = static_cast<VerifyStat*>(workspace);
  p.sums = reinterpret_cast<double*>(static_cast<char*>(workspace) + verify_sums_at(B, N, V));
  p.arrived = reinterpret_cast<int*>(p.sums + B * p.nch);
  p.count = accepted; p.path = path; p.next = next;
  const unsigned rows = unsigned(B * (N + 1 + (p.d ? N : 0)));
  const dim3 g1{rows * unsigned(p.nch), 1, 1}, g2{unsigned(B) * unsigned(p.nch), 1, 1};
  if (logits_are_f32) {
    verify_stat_kernel<float><<<g1, 256, 0, stream>>>(p);
    verify_draw_kernel<float><<<g2, 256, 0, stream>>>(p);
  } else {
    verify_stat_kernel<uint16_t><<<g1, 256, 0, stream>>>(p);
    verify_draw_kernel<uint16_t><<<g2, 256, 0, stream>>>(p);
  }
  return check_launch("verify_drafts");
}
