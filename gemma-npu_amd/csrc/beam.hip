// A beam search step's choice: of the nb beams' V continuations each, the k of the largest
//
//   score[i] + log_softmax(logits[i])[v],
//
// sorted, ties to the lowest i V + v.  Decode's greedy tail (the reference's loop, gemma_npu.py:292-295, takes
// the argmax) for several sequences that are weighed against each other.
//
// beam_chunk_kernel reads the logits once.  A workgroup takes a run of 256 E logits of one beam into registers,
// makes their maximum and sum of exponentials, and finds its k largest: the k-th largest of the maxima of 64
// lane groups is a bound that at least k logits reach and few more do, so those are listed and ranked by
// counting.  Where too many reach it (equal logits), or there is a NaN, the k are taken one by one instead.
// Within a beam the order of logits is the order of scores, so nothing else can be among the k best.
// beam_join_kernel, one workgroup per group of beams, makes the beams' logsumexp and takes the k best of those
// lists the same way.  Exponentials, sums and scores are in 64 bits, off by less than 1e-13 before the result is
// rounded: beams may differ by less than 32 bits resolve, and the choice between them has to be right.  Where too
// many reach its bound (k near 64, beams far apart) the listed ones give a tighter one: 64 of 64 beams of 32000 one
// by one 1189 us, so 135.  The logits' way through memory and their exponentials bound large calls (64 beams of
// 262144 fp32 logits, 67 MB: 34 us, with exponentials of 32 bits 28), two kernels' starts and barriers small ones
// (4 beams of bf16: 14.6 us, with 32 bits 13.3).
#include <algorithm>

#include "w8a8_common.h"

namespace w8a8 {

constexpr int BEAM_MAX_K = 64;
constexpr int BEAM_MAX_BEAMS = 256;
constexpr int BEAM_LIST = 1024;             // most candidates that are ranked by counting
constexpr int BEAM_ROUNDS = 8;              // most times that the join tightens its bound
constexpr int BEAM_HELD = 8;                // candidates that a thread of the join keeps in registers

struct BeamStat {
  double sum;  // of exponentials against the maximum
  float top;
};

struct BeamParams {
  const void* x; int64_t gs, rs;            // logits [B, nb, V] bf16 or fp32 (element strides of groups and beams)
  const float* score; int64_t ss;           // fp32 [B, nb]
  int nb, V, k, nch;
  BeamStat* stat;                           // [B nb][nch]
  uint2* cand;                              // [B nb][nch][k] logit's bits and token
  float* out_score; int64_t *out_beam, *out_tok;  // [B, k]
};

// Order-preserving bits: larger for larger values, NaN above +inf, -0 and +0 alike.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((b & 0x7fffffffu) == 0u) return 0x80000000u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_bits(double x) {
  const uint64_t b = uint64_t(__double_as_longlong(x)), m = b & 0x7fffffffffffffffull;
  if (m > 0x7ff0000000000000ull) return ~0ull;
  if (m == 0) return 0x8000000000000000ull;
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ uint32_t lane_value(uint32_t v, int j) { return uint32_t(__builtin_amdgcn_readlane(int(v), j)); }
__device__ __forceinline__ float lane_value(float v, int j) { return __uint_as_float(lane_value(__float_as_uint(v), j)); }

// The k-th largest of 64 lanes' values (k <= 64, none of them NaN): the value whose rank, ties by lane, is k - 1.
template <class T>
__device__ __forceinline__ T wave_kth(T v, int k) {
  const int lane = threadIdx.x & 63;
  int rank = 0;
#pragma unroll 16
  for (int j = 0; j < 64; ++j) {
    const T o = lane_value(v, j);
    rank += (o > v || (o == v && j < lane)) ? 1 : 0;
  }
  const uint64_t at = __builtin_amdgcn_ballot_w64(rank == k - 1);
  return lane_value(v, __builtin_ctzll(at));
}

// A candidate before another: larger, or equal and of the lower index.
template <class T>
__device__ __forceinline__ bool before(T a, uint32_t ai, T b, uint32_t bi) {
  return (a > b) | ((a == b) & (ai < bi));  // (no branch: both are read at once)
}

// The best of a workgroup's candidates, given to every thread.
template <class T, int NW>
__device__ __forceinline__ void block_first(T& v, uint32_t& i, T* sv, uint32_t* si) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const T ov = __shfl_xor(v, o, 64);
    const uint32_t oi = __shfl_xor(i, o, 64);
    if (before(ov, oi, v, i)) v = ov, i = oi;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sv[threadIdx.x >> 6] = v, si[threadIdx.x >> 6] = i;
  __syncthreads();
  v = sv[0], i = si[0];
#pragma unroll
  for (int w = 1; w < NW; ++w)
    if (before(sv[w], si[w], v, i)) v = sv[w], i = si[w];
}

template <class X, int E>
__global__ __launch_bounds__(256) void beam_chunk_kernel(BeamParams p) {
  constexpr int CHUNK = 256 * E;
  __shared__ uint32_t lv[BEAM_LIST], li[BEAM_LIST];
  __shared__ float gmax[64];
  __shared__ float red[4], bound_s;
  __shared__ double red2[4];
  __shared__ int count;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int row = blockIdx.x / p.nch, ch = blockIdx.x % p.nch;
  const X* xp = static_cast<const X*>(p.x) + int64_t(row / p.nb) * p.gs + int64_t(row % p.nb) * p.rs;
  const int base = ch * CHUNK, n = min(CHUNK, p.V - base);
  // element e of thread t is logit base + 8 (t + 256 (e / 8)) + e % 8, or where that leaves lane groups without
  // any base + t + 256 e; past the last one -inf
  float v[E];
  const bool thin = n <= 2048;
  const bool wide = (reinterpret_cast<uintptr_t>(xp) & 15) == 0;
  auto local = [&](int e) __attribute__((always_inline)) { return thin ? t + 256 * e : 8 * (t + 256 * (e >> 3)) + (e & 7); };
#pragma unroll
  for (int c = 0; c < E / 8; ++c) {
    const int at = 8 * (t + 256 * c);
    const X* src = xp + base + at;
    if (!thin && wide && at + 8 <= n) {
      if constexpr (sizeof(X) == 2) {
        float f[8];
        unpack8(*reinterpret_cast<const v4u*>(src), f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * c + e] = f[e];
      } else {
        const v4f a = *reinterpret_cast<const v4f*>(src), b = *reinterpret_cast<const v4f*>(src + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[8 * c + e] = a[e], v[8 * c + 4 + e] = b[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float f = -__builtin_inff();
        const int i = local(8 * c + e);
        if (i < n) {
          if constexpr (sizeof(X) == 2)
            f = bf16_to_f32(xp[base + i]);
          else
            f = xp[base + i];
        }
        v[8 * c + e] = f;
      }
    }
  }
  auto valid = [&](int e) __attribute__((always_inline)) { return local(e) < n; };
  auto index = [&](int e) __attribute__((always_inline)) { return uint32_t(base + local(e)); };

  // the maximum (fmaxf passes NaN over), and those of groups of four lanes
  float m = -__builtin_inff();
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
  float mw = fmaxf(m, __shfl_xor(m, 1, 64));
  mw = fmaxf(mw, __shfl_xor(mw, 2, 64));
  if ((t & 3) == 0) gmax[t >> 2] = mw;
#pragma unroll
  for (int o = 32; o >= 4; o >>= 1) mw = fmaxf(mw, __shfl_xor(mw, o, 64));
  if (lane == 0) red[wave] = mw;
  if (t == 0) count = 0;
  __syncthreads();
  const float top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  if (wave == 0) {
    const float b = wave_kth(gmax[lane], p.k);
    if (lane == 0) bound_s = b;
  }
  // e^(v - top): subtracted in 64 bits, so that a term is 1 at the maximum and never above, however far out the logits
  // are (a mask of the type's lowest value over the whole chunk)
  const double ref = top == -__builtin_inff() ? 0.0 : double(top);
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) s += exp_64(double(v[e]) - ref);  // NaN with a NaN or +inf among the logits
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) red2[wave] = s;
  __syncthreads();
  s = (red2[0] + red2[1]) + (red2[2] + red2[3]);
  const float bound = bound_s;
  const bool plain = s == s;
  auto list = [&](int e) __attribute__((always_inline)) {
    const int at = atomicAdd(&count, 1);
    if (at < BEAM_LIST) lv[at] = order_bits(v[e]), li[at] = index(e);
  };
  if (plain && bound > -__builtin_inff()) {
    if (m >= bound)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v[e] >= bound) list(e);
  } else if (plain) {
    // fewer than k groups hold more than -inf (a grammar's mask, a short vocabulary): all that is above it, and
    // of the rest the first k logits hold as many as can be among the best
    if (m > -__builtin_inff() || t < p.k)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (v[e] > -__builtin_inff() || (valid(e) && local(e) < p.k)) list(e);
  }
  __syncthreads();
  if (t == 0) p.stat[int64_t(row) * p.nch + ch] = BeamStat{s, top};
  uint2* out = p.cand + (int64_t(row) * p.nch + ch) * p.k;
  const int nc = count;
  auto value = [&](uint32_t o) __attribute__((always_inline)) {  // the logit's bits again (NaN: the quiet one)
    return o == 0xffffffffu ? 0x7fc00000u : (o & 0x80000000u ? o & 0x7fffffffu : ~o);
  };
  if (plain && nc <= BEAM_LIST) {
    for (int j = t; j < nc; j += 256) {
      int rank = 0;
      const uint32_t a = lv[j], ai = li[j];
#pragma unroll 8
      for (int c = 0; c < nc; ++c) {
        const uint32_t o = lv[c], oi = li[c];
        rank += before(o, oi, a, ai) ? 1 : 0;
      }
      if (rank < p.k) out[rank] = make_uint2(value(a), ai);
    }
    for (int j = nc + t; j < p.k; j += 256) out[j] = make_uint2(0x7fc00000u, 0xffffffffu);  // (none left)
    return;
  }
  // one by one: the best after the last one taken
  uint32_t last = 0xffffffffu, lasti = 0;
  bool any = false;
  for (int j = 0; j < p.k; ++j) {
    uint32_t b = 0, bi = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t o = order_bits(v[e]), i = index(e);
      if (valid(e) && (!any || before(last, lasti, o, i)) && before(o, i, b, bi)) b = o, bi = i;
    }
    block_first<uint32_t, 4>(b, bi, lv, li);
    if (t == 0) out[j] = make_uint2(value(b), bi);  // (none left: token 0xffffffff)
    last = b, lasti = bi, any = true;
  }
}

__global__ __launch_bounds__(1024) void beam_join_kernel(BeamParams p) {
  __shared__ double log_s[BEAM_MAX_BEAMS], score_s[BEAM_MAX_BEAMS];
  __shared__ float max_s[BEAM_MAX_BEAMS];
  __shared__ uint64_t lv[BEAM_LIST], la[BEAM_LIST];  // candidates: score's order bits, beam << 32 | token
  __shared__ uint32_t gmax[64], bound_s;
  __shared__ int count;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int grp = blockIdx.x;
  const int per = p.nch * p.k, total = p.nb * per;
  const uint2* cand = p.cand + int64_t(grp) * total;
  // the first candidates are asked for before the beams' sums are made
  uint2 held[BEAM_HELD];
#pragma unroll
  for (int u = 0; u < BEAM_HELD; ++u) held[u] = t + 1024 * u < total ? cand[t + 1024 * u] : make_uint2(0u, 0xffffffffu);
  if (t == 0) count = 0;
  // Each beam's maximum, the logarithm of its sum against that, and its score, one wave per beam.  They are kept apart:
  // a logit is taken from the maximum first, as log_softmax has it, and logits of any size leave the rest its bits.
  for (int i = wave; i < p.nb; i += 16) {
    const BeamStat* st = p.stat + (int64_t(grp) * p.nb + i) * p.nch;
    float m = -__builtin_inff();
    for (int c = lane; c < p.nch; c += 64) m = fmaxf(m, st[c].top);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    double s = 0.0;
    for (int c = lane; c < p.nch; c += 64) {
      const BeamStat a = st[c];
      // a chunk of -inf only has the sum 0 of its reference 0
      s += a.top == -__builtin_inff() ? a.sum : a.sum * exp(double(a.top) - double(m));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    const double sc = double(p.score[int64_t(grp) * p.ss + i]);
    // no token can follow where all logits are -inf; +inf and NaN make NaN, as log_softmax does
    const double b = m == -__builtin_inff() && s == 0.0 ? (sc != sc ? sc : -__builtin_inf()) : sc - (double(m) + log(s));
    const bool finite = b - b == 0.0;
    if (lane == 0) max_s[i] = m, log_s[i] = finite ? log(s) : 0.0, score_s[i] = finite ? sc : b;
  }
  __syncthreads();
  // A candidate's score's order bits and place; false where there is none.  A beam whose score or logsumexp is not
  // finite has that score for every token: its first tokens stand for it.  (j / per, less than 256, from a product
  // that is off by at most one: an integer division is most of the work otherwise.)
  const float rper = 1.0f / float(per);
  auto score = [&](int j, uint2 a, uint64_t& o, uint64_t& at) __attribute__((always_inline)) {
    int i = int(float(j) * rper), c = j - i * per;
    if (c < 0) --i, c += per;
    if (c >= per) ++i, c -= per;
    const double b = score_s[i];
    uint32_t tok = a.y;
    double sc = double(__uint_as_float(a.x)) - double(max_s[i]) - log_s[i] + b;
    if (!(b - b == 0.0)) {
      sc = b;
      tok = c < p.k && c < p.V ? uint32_t(c) : 0xffffffffu;
    }
    o = order_bits(sc);
    at = uint64_t(uint32_t(i)) << 32 | tok;
    return tok != 0xffffffffu;
  };
  uint64_t bits[BEAM_HELD], place[BEAM_HELD], top = 0;  // (0, below every score: none)
#pragma unroll
  for (int u = 0; u < BEAM_HELD; ++u) {
    bits[u] = 0;
    if (1024 * u >= total) break;
    const int j = t + 1024 * u;
    if (j < total && !score(j, held[u], bits[u], place[u])) bits[u] = 0;
    top = max(top, bits[u]);
  }
  for (int j = t + 1024 * BEAM_HELD; j < total; j += 1024) {
    uint64_t o, at;
    if (score(j, cand[j], o, at)) top = max(top, o);
  }
  // the bound: of the upper halves of the best scores of 64 groups
  uint32_t high = uint32_t(top >> 32);
#pragma unroll
  for (int x = 8; x > 0; x >>= 1) high = max(high, uint32_t(__shfl_xor(high, x, 64)));
  if ((t & 15) == 0) gmax[t >> 4] = high;
  __syncthreads();
  if (wave == 0) {
    const uint32_t b = wave_kth(gmax[lane], p.k);
    if (lane == 0) bound_s = b;
  }
  __syncthreads();
  uint64_t bound = max(uint64_t(bound_s) << 32, uint64_t(1));
  auto list = [&](uint64_t o, uint64_t at) __attribute__((always_inline)) {
    const int c = atomicAdd(&count, 1);
    if (c < BEAM_LIST) lv[c] = o, la[c] = at;
  };
  int nc;
  for (int round = 0;; ++round) {
#pragma unroll
    for (int u = 0; u < BEAM_HELD; ++u) {
      if (1024 * u >= total) break;
      if (bits[u] >= bound) list(bits[u], place[u]);
    }
    for (int j = t + 1024 * BEAM_HELD; j < total; j += 1024) {
      uint64_t o, at;
      if (score(j, cand[j], o, at) && o >= bound) list(o, at);
    }
    __syncthreads();
    nc = count;
    if (nc <= BEAM_LIST || round == BEAM_ROUNDS) break;
    // too many (a group without any of the best beams): the same bound of those that were listed
    __syncthreads();  // (every wave has read the count that is cleared)
    if (wave == 0) {
      uint32_t high = 0;
      for (int c = lane; c < BEAM_LIST; c += 64) high = max(high, uint32_t(lv[c] >> 32));
      const uint32_t b = wave_kth(high, p.k);
      if (lane == 0) bound_s = b, count = 0;
    }
    __syncthreads();
    const uint64_t tighter = uint64_t(bound_s) << 32;
    if (tighter <= bound) break;  // (equal scores)
    bound = tighter;
  }
  auto store = [&](int r, uint64_t o, uint64_t at) __attribute__((always_inline)) {
    const uint64_t b = o == ~0ull ? 0x7ff8000000000000ull : (o >> 63 ? o & 0x7fffffffffffffffull : ~o);
    p.out_score[int64_t(grp) * p.k + r] = float(__longlong_as_double((long long)b));
    p.out_beam[int64_t(grp) * p.k + r] = int64_t(at >> 32);
    p.out_tok[int64_t(grp) * p.k + r] = int64_t(uint32_t(at));
  };
  if (nc <= BEAM_LIST) {
    for (int a = t; a < nc; a += 1024) {
      const uint64_t o = lv[a], at = la[a];
      int rank = 0;
#pragma unroll 8
      for (int c = 0; c < nc; ++c) {
        const uint64_t oc = lv[c], ac = la[c];
        rank += (oc > o) | ((oc == o) & (ac < at)) ? 1 : 0;
      }
      if (rank < p.k) store(rank, o, at);
    }
    return;
  }
  // one by one: the best after the last one taken
  __shared__ uint64_t sv[16], sa[16];
  uint64_t last = 0, lastat = 0;
  for (int r = 0; r < p.k; ++r) {
    uint64_t b = 0, ba = ~0ull;  // (below every candidate)
    for (int j = t; j < total; j += 1024) {
      uint64_t o, at;
      if (!score(j, cand[j], o, at)) continue;
      if (r > 0 && !(o < last || (o == last && at > lastat))) continue;
      if (o > b || (o == b && at < ba)) b = o, ba = at;
    }
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) {
      const uint64_t ob = __shfl_xor(b, x, 64), oa = __shfl_xor(ba, x, 64);
      if (ob > b || (ob == b && oa < ba)) b = ob, ba = oa;
    }
    __syncthreads();
    if (lane == 0) sv[wave] = b, sa[wave] = ba;
    __syncthreads();
    b = sv[0], ba = sa[0];
    for (int w = 1; w < 16; ++w)
      if (sv[w] > b || (sv[w] == b && sa[w] < ba)) b = sv[w], ba = sa[w];
    if (t == 0) store(r, b, ba);
    last = b, lastat = ba;
  }
}

}  // namespace w8a8

using namespace w8a8;

// Logits per thread of the chunk kernel: 32, or 16 where that leaves CUs without a workgroup.
static int beam_e(int64_t rows, int64_t V) { return rows * ((V + 8191) / 8192) < 2 * 256 ? 16 : 32; }
static int64_t beam_chunks(int64_t rows, int64_t V) {
  const int64_t chunk = 256 * beam_e(rows, V);
  return (V + chunk - 1) / chunk;
}

// (Launches of less than 2^32 threads.)
static bool beam_shape_ok(int64_t B, int64_t nb, int64_t V, int64_t k) {
  return B >= 1 && B < (1 << 22) && nb >= 1 && nb <= BEAM_MAX_BEAMS && V >= 1 && V <= INT32_MAX / 2 && k >= 1 &&
         k <= BEAM_MAX_K && k <= nb * V && B * nb * beam_chunks(B * nb, V) < (1 << 24);
}

extern "C" int64_t w8a8_beam_select_workspace_bytes(int64_t B, int64_t nb, int64_t V, int64_t k) {
  if (!beam_shape_ok(B, nb, V, k)) return -1;
  return B * nb * beam_chunks(B * nb, V) * (int64_t(sizeof(BeamStat)) + 8 * k);
}

extern "C" int w8a8_beam_select(const void* logits, int logits_are_f32, int64_t group_stride, int64_t row_stride,
                                const float* scores, int64_t score_stride, int64_t B, int64_t nb, int64_t V, int64_t k,
                                float* out_scores, int64_t* out_beams, int64_t* out_tokens, void* workspace,
                                int64_t workspace_bytes, hipStream_t stream) {
  const char* what = "beam_select";
  if (!beam_shape_ok(B, nb, V, k))
    return fail(W8A8_EINVAL, "%s: B=%lld nb=%lld V=%lld k=%lld (at most %d beams, k at most %d and nb V)", what, (long long)B,
                (long long)nb, (long long)V, (long long)k, BEAM_MAX_BEAMS, BEAM_MAX_K);
  if (!logits || !scores || !out_scores || !out_beams || !out_tokens || !workspace)
    return fail(W8A8_EINVAL, "%s: null pointer", what);
  if ((nb > 1 && row_stride < V) || (B > 1 && (group_stride < V || score_stride < nb)))
    return fail(W8A8_EINVAL, "%s: strides smaller than the rows", what);
  const int64_t need = w8a8_beam_select_workspace_bytes(B, nb, V, k);
  if (workspace_bytes < need)
    return fail(W8A8_EINVAL, "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  if ((uintptr_t)logits % (logits_are_f32 ? 4 : 2) || (uintptr_t)scores % 4 || (uintptr_t)out_scores % 4 ||
      (uintptr_t)out_beams % 8 || (uintptr_t)out_tokens % 8 || (uintptr_t)workspace % 8)
    return fail(W8A8_EALIGN, "%s: operands naturally, the workspace 8-byte aligned", what);
  BeamParams p{};
  p.x = logits; p.gs = B > 1 ? group_stride : 0; p.rs = nb > 1 ? row_stride : 0;
  p.score = scores; p.ss = B > 1 ? score_stride : 0;
  p.nb = int(nb); p.V = int(V); p.k = int(k); p.nch = int(beam_chunks(B * nb, V));
  p.stat = static_cast<BeamStat*>(workspace);
  p.cand = reinterpret_cast<uint2*>(p.stat + B * nb * p.nch);
  p.out_score = out_scores; p.out_beam = out_beams; p.out_tok = out_tokens;
  const unsigned grid = unsigned(B * nb * p.nch);
  const bool e16 = beam_e(B * nb, V) == 16;
  if (logits_are_f32)
    e16 ? beam_chunk_kernel<float, 16><<<grid, 256, 0, stream>>>(p) : beam_chunk_kernel<float, 32><<<grid, 256, 0, stream>>>(p);
  else
    e16 ? beam_chunk_kernel<uint16_t, 16><<<grid, 256, 0, stream>>>(p)
        : beam_chunk_kernel<uint16_t, 32><<<grid, 256, 0, stream>>>(p);
  beam_join_kernel<<<unsigned(B), 1024, 0, stream>>>(p);
  return check_launch("beam_select");
}
