// Rows of the key / value cache put elsewhere: the beams' states in the order a beam search step chose, an
// accepted path of drafted tokens moved up to the context, and a cache cut to a budget of rows.  The
// reference's cache only grows (HF's DynamicCache, gemma_npu.py:278-300).
#include <algorithm>

#include "w8a8_common.h"

namespace w8a8 {

// ---- t[i] = t[index[i]] in place ----------------------------------------------------------------------
//
// A thread owns one column (16 bytes) of every row of the axis: it reads the rows that others take before
// it writes any, so rows can be exchanged and copied at will without a second buffer, and rows that stay
// are neither read nor written.  All tensors of a call, a layer's or a whole model's keys and values, go in
// one launch.

constexpr int REORDER_MAX = 64;       // rows of the axis that change
constexpr int REORDER_TENSORS = 48;   // tensors of a launch
constexpr int64_t REORDER_BLOCKS = (int64_t(1) << 24) - 1;  // workgroups of a launch's x: 2^32 threads are too many

struct ReorderTensor {
  char* base;
  int64_t axis, outer, inner;         // byte strides: of the axis, of the entries before it, of the runs behind it
  int64_t run;                        // columns (of the launch's width) per run
  int32_t ninner, block0;             // runs per entry; the tensor's first workgroup
};
struct ReorderParams {
  const int64_t* index; int64_t is;   // [n], or [entries before the axis][n] with is = n
  int n, size, ntensors, nouter;      // n rows change; rows 0 .. size - 1 can be taken
  ReorderTensor t[REORDER_TENSORS];
};
static_assert(sizeof(ReorderParams) <= 4096, "kernel arguments");

template <class C, int N>
__global__ __launch_bounds__(256) void reorder_kernel(ReorderParams p) {
  int x = 0;
  while (x + 1 < p.ntensors && int(blockIdx.x) >= p.t[x + 1].block0) ++x;
  const ReorderTensor& d = p.t[x];
  const uint32_t run = uint32_t(d.run), per = run * uint32_t(d.ninner);
  const uint32_t col = uint32_t(int(blockIdx.x) - d.block0) * 256u + threadIdx.x;
  if (col >= per) return;
  const int o = blockIdx.y;
  const uint32_t in = d.ninner > 1 ? col / run : 0u;
  char* base = d.base + int64_t(o) * d.outer + int64_t(in) * d.inner + int64_t(col - in * run) * int64_t(sizeof(C));
  const int64_t* index = p.index + int64_t(o) * p.is;
  C v[N];
  int src[N];  // (the same for the workgroup)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    src[i] = i;
    if (i < p.n) {
      const int64_t s = index[i];
      if (s >= 0 && s < p.size) src[i] = int(s);  // an index outside the axis leaves the row as it is
    }
    src[i] = __builtin_amdgcn_readfirstlane(src[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (src[i] != i) v[i] = *reinterpret_cast<const C*>(base + int64_t(src[i]) * d.axis);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (src[i] != i) *reinterpret_cast<C*>(base + int64_t(i) * d.axis) = v[i];
}

// ---- a cache cut to its budget ---------------------------------------------------------------------------
//
// Per KV head, of n rows `budget` are kept: those whose position is within `recent` of the newest one, then
// those of the largest weight (NaN the largest; ties: the lower row).  Attention does not depend on the order
// of the rows, so the kept rows below the budget stay where they are and the others move, in order, into
// the places that became free: the least that can be moved, in place, and no row is both read and written.
//
// The budget-th largest key is found by a radix select over digits of 11, 11 and 10 bits.  What comes before a
// row in row order (equal keys, free places, moving rows) is a sum over the waves or chunks before it and
// ballots within, so ranks come out in row order.  Up to EVICT_ONE rows one workgroup per KV head does it all
// from keys in LDS (evict_select_kernel).  Above that the rows are read by a workgroup per chunk of 4096:
//   evict_newest_kernel  each chunk's newest position
//   evict_digit_kernel   the keys' first digits counted per chunk
//   evict_split_kernel   the first digit of the budget-th key from those counts; rows of larger digits are
//                        counted, the keys of that digit listed, in row order
//   evict_least_kernel   one workgroup per KV head finds the key among those, and what is before each chunk
//   evict_list_kernel    the lists of free places and moving rows, chunk by chunk
// and evict_move_kernel copies the rows.  A cache that is cut by a few rows (EVICT_FEW, as at every step of a
// cache that is full) goes without that: the rows that go are taken one by one (evict_few_kernel).  Loops are not
// unrolled over a thread's rows: a workgroup runs through such code once, and fetching it took longer than the
// work (65521 rows of 8 heads with the keys in registers 84 us for the select alone, 242 us reading them again at
// each step; in chunks 33).

constexpr int EVICT_NW = 16;
constexpr int EVICT_ONE = 16384;           // most rows of evict_select_kernel
constexpr int EVICT_CHUNK = 4096;          // rows per workgroup of the others
constexpr int EVICT_INFO = 6;              // words of a chunk's counts
constexpr int EVICT_FEW = 6;               // most rows that evict_few_kernel takes out
constexpr int EVICT_FEW_COLS = 2048;       // and most 16-byte columns of k (and of v) that its workgroup moves

struct EvictParams {
  const float* w; int64_t whs;          // fp32 [KV, n]
  const int32_t* pos; int64_t phs;      // int32 [KV, n]
  int n, budget, recent;
  int32_t* kept; int64_t khs;           // int32 [KV, budget]
  float* w_out; int64_t wos;            // fp32 [KV, budget]
  int32_t* pos_out; int64_t pos_os;     // int32 [KV, budget]
  int32_t* hole;                        // [KV][most] free places, ascending
  int32_t* mover;                       // [KV][most] rows that fill them, ascending
  int32_t* count;                       // [KV]
  int32_t* least;                       // [KV][2] the least key kept, how many rows of it
  int32_t* info;                        // [KV][nch][EVICT_INFO] a chunk's newest position; rows of larger digits below the
                                        // budget and from it on, of the digit likewise; then what is before it
  uint32_t* digit;                      // [KV][nch][1024] counts of two first digits each
  uint32_t* open;                       // [KV][nch][4096] keys of the budget-th key's first digit
  int most, nch;                        // min(budget, n - budget); chunks
  char* k; int64_t kh, kr;              // the cache's bytes: strides of heads and rows
  char* v; int64_t vh, vr;
  int row_cols;                         // 16-byte columns per row
};

// Order of the rows: larger is kept first; 0, below every row's, stands for no row.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t pos, int64_t old) {
  const uint32_t b = __float_as_uint(w), m = b & 0x7fffffffu;
  uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
  k = m > 0x7f800000u ? 0xfffffffeu : m == 0u ? 0x80000000u : k;
  return int64_t(pos) > old ? 0xffffffffu : k;
}

__device__ __forceinline__ int evict_count(bool b) { return __popcll(__builtin_amdgcn_ballot_w64(b)); }
__device__ __forceinline__ int evict_rank(bool b) {  // lanes before this one with b
  return __popcll(__builtin_amdgcn_ballot_w64(b) & ((1ull << (threadIdx.x & 63)) - 1ull));
}

// v summed over the 16 waves before this one (buf [16], not in use by others until the next barrier after).
__device__ __forceinline__ int evict_before(int v, int* buf) {
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) buf[wave] = v;
  __syncthreads();
  int s = 0;
  for (int x = 0; x < EVICT_NW; ++x) s += x < wave ? buf[x] : 0;
  return s;
}

// The digit that holds the need-th largest of the counted rows, and how many of its rows that leaves: thread t
// of 1024 gives the counts c0 and c1 of digits 2047 - 2 t and 2046 - 2 t.
__device__ __forceinline__ void evict_pick(int c0, int c1, int* red, uint32_t* digit_s, int* need_s, uint32_t& digit,
                                           int& need) {
  const int t = threadIdx.x, lane = t & 63, hi = 2047 - 2 * t;
  int sum = c0 + c1;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(sum, o, 64);
    if (lane >= o) sum += v;
  }
  const int total = __shfl(sum, 63, 64);
  const int above = evict_before(total, red) + sum - c0 - c1;  // rows of larger digits
  if (above < need && above + c0 >= need) *digit_s = uint32_t(hi), *need_s = need - above;
  if (above + c0 < need && above + c0 + c1 >= need) *digit_s = uint32_t(hi - 1), *need_s = need - above - c0;
  __syncthreads();
  digit = *digit_s;
  need = *need_s;
}

// The largest of v over the workgroup's 1024 threads.
__device__ __forceinline__ int evict_max(int v, int* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int x = 0; x < EVICT_NW; ++x) v = max(v, red[x]);
  return v;
}

__global__ __launch_bounds__(1024) void evict_select_kernel(EvictParams p) {
  __shared__ uint32_t key[EVICT_ONE];
  __shared__ int32_t ps[EVICT_ONE];
  __shared__ uint32_t hist[2048];
  __shared__ int red[EVICT_NW], red2[EVICT_NW], red3[EVICT_NW];
  __shared__ uint32_t digit_s;
  __shared__ int need_s;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = blockIdx.x;
  const float* w = p.w + int64_t(g) * p.whs;
  const int32_t* pos = p.pos + int64_t(g) * p.phs;
  const int n = p.n, budget = p.budget;
  hist[t] = 0u;
  hist[t + 1024] = 0u;
  // the weights' bits and the positions into LDS while the newest is found
  int newest = INT32_MIN;
  for (int r0 = t; r0 < n; r0 += 4096) {
    float x[4];
    int32_t y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + 1024 * u;
      x[u] = r < n ? w[r] : 0.0f;
      y[u] = r < n ? pos[r] : INT32_MIN;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (r0 + 1024 * u < n) key[r0 + 1024 * u] = __float_as_uint(x[u]), ps[r0 + 1024 * u] = y[u];
      newest = max(newest, y[u]);
    }
  }
  newest = evict_max(newest, red);  // (its barrier: hist is cleared)
  const int64_t old = int64_t(newest) - p.recent;
#pragma unroll 2
  for (int r = t; r < n; r += 1024) {
    const uint32_t k = evict_key(__uint_as_float(key[r]), ps[r], old);
    key[r] = k;
    atomicAdd(&hist[k >> 21], 1u);
  }
  uint32_t prefix = 0, digit;
  int need = budget;
#pragma unroll 1
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    if (d > 0) {
      const uint32_t mask = d == 1 ? 0xffe00000u : 0xfffffc00u, digits = d == 1 ? 2047u : 1023u;
#pragma unroll 4
      for (int r = t; r < n; r += 1024)
        if ((key[r] & mask) == prefix) atomicAdd(&hist[(key[r] >> shift) & digits], 1u);
    }
    __syncthreads();
    const int hi = 2047 - 2 * t, c0 = int(hist[hi]), c1 = int(hist[hi - 1]);
    hist[hi] = 0u;
    hist[hi - 1] = 0u;
    evict_pick(c0, c1, red2, &digit_s, &need_s, digit, need);
    prefix |= digit << shift;
  }

  // wave w's rows: steps of 64 from w * steps * 64 on
  const int steps = (n + 64 * EVICT_NW - 1) / (64 * EVICT_NW), row0 = wave * steps * 64 + lane;
  int neq = 0;
#pragma unroll 4
  for (int e = 0; e < steps; ++e) {
    const int r = row0 + 64 * e;
    neq += evict_count(r < n && key[r] == prefix);
  }
  int seen = evict_before(neq, red3);
  const int seen0 = seen;
  int nhole = 0, nmove = 0;
#pragma unroll 2
  for (int e = 0; e < steps; ++e) {
    const int r = row0 + 64 * e;
    const uint32_t k = r < n ? key[r] : 0u;
    const bool eq = r < n && k == prefix, low = r < budget;
    const bool keep = r < n && (k > prefix || (eq && seen + evict_rank(eq) < need));
    seen += evict_count(eq);
    nhole += evict_count(low && !keep);
    nmove += evict_count(!low && keep);
  }
  __syncthreads();
  int hole = evict_before(nhole, red), move = evict_before(nmove, red2);
  seen = seen0;
  int32_t* const holes = p.hole + int64_t(g) * p.most;
  int32_t* const movers = p.mover + int64_t(g) * p.most;
  int32_t* const ko = p.kept + int64_t(g) * p.khs;
  float* const wo = p.w_out + int64_t(g) * p.wos;
  int32_t* const po = p.pos_out + int64_t(g) * p.pos_os;
  for (int e0 = 0; e0 < steps; e0 += 4) {
    float x[4];  // (the keys are not the weights' bits)
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = row0 + 64 * (e0 + u) < budget ? w[row0 + 64 * (e0 + u)] : 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (e0 + u >= steps) break;
      const int r = row0 + 64 * (e0 + u);
      const uint32_t k = r < n ? key[r] : 0u;
      const bool eq = r < n && k == prefix, low = r < budget;
      const bool keep = r < n && (k > prefix || (eq && seen + evict_rank(eq) < need));
      seen += evict_count(eq);
      if (low && !keep) holes[hole + evict_rank(low && !keep)] = r;
      hole += evict_count(low && !keep);
      if (!low && keep) movers[move + evict_rank(!low && keep)] = r;
      move += evict_count(!low && keep);
      if (low && keep) ko[r] = r, wo[r] = x[u], po[r] = ps[r];
    }
  }
  if (wave == EVICT_NW - 1 && lane == 0) p.count[g] = hole;
}

// A row's key and, less for higher rows, its place: of equal keys the highest row goes first.
__device__ __forceinline__ uint64_t evict_place(uint32_t key, int row) { return uint64_t(key) << 32 | uint32_t(~row); }

// The least of v over the workgroup's 1024 threads (buf [16], not in use by others until the next barrier after).
__device__ __forceinline__ uint64_t evict_min(uint64_t v, uint64_t* buf) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, uint64_t(__shfl_xor(v, o, 64)));
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EVICT_NW; ++i) v = min(v, buf[i]);
  return v;
}

// With the rows that go (out [n - budget] in LDS): the rows that move, and where to.  Called by 1024 threads.
__device__ __forceinline__ void evict_few_move(const EvictParams& p, int g, const int* out, int* hole, int* mover) {
  const int t = threadIdx.x, budget = p.budget, drop = p.n - budget;
  // free places and the rows that fill them, both in row order: thread j < drop ranks out[j] and row budget + j
  int nhole = 0;
  for (int j = 0; j < drop; ++j) nhole += out[j] < budget ? 1 : 0;
  if (t < drop) {
    int before = 0, moves = 0;
    bool stays = true;  // row budget + t
    for (int i = 0; i < drop; ++i) {
      before += out[i] < out[t] ? 1 : 0;
      moves += out[i] >= budget && out[i] < budget + t ? 1 : 0;
      stays = stays && out[i] != budget + t;
    }
    if (out[t] < budget) hole[before] = out[t];
    if (stays) mover[t - moves] = budget + t;
  }
  __syncthreads();
  char* const k = p.k + int64_t(g) * p.kh;
  char* const v = p.v + int64_t(g) * p.vh;
  for (int i = t; i < nhole * p.row_cols; i += 1024) {
    const int m = i / p.row_cols, col = i % p.row_cols;
    const int64_t dst = hole[m], src = mover[m], c = int64_t(col) * 16;
    const v4u a = *reinterpret_cast<const v4u*>(k + src * p.kr + c);
    const v4u b = *reinterpret_cast<const v4u*>(v + src * p.vr + c);
    *reinterpret_cast<v4u*>(k + dst * p.kr + c) = a;
    *reinterpret_cast<v4u*>(v + dst * p.vr + c) = b;
    if (col == 0) {
      p.kept[int64_t(g) * p.khs + dst] = int32_t(src);
      p.w_out[int64_t(g) * p.wos + dst] = p.w[int64_t(g) * p.whs + src];
      p.pos_out[int64_t(g) * p.pos_os + dst] = p.pos[int64_t(g) * p.phs + src];
    }
  }
}

// One workgroup per KV head and a launch for everything, where at most EVICT_FEW rows go.  A thread holds E rows
// in registers; the row of the least key (ties: the highest) goes, as often as rows have to.  Each choice is a
// minimum over the workgroup, which bounds it (1.2 us): of 4097 rows of head_dim 512 one goes in 5.3 us, four in
// 9.1, eight would in 13.9; the radix select and the launch that moves the rows take 13.8 whatever goes (of 512
// rows 9.4 against 7.7 for four and 11.8 for eight, of 16384 28 against 13 and 19).
template <int E>
__global__ __launch_bounds__(1024) void evict_few_kernel(EvictParams p) {
  __shared__ uint64_t least[2][EVICT_NW];
  __shared__ int red[EVICT_NW], out[EVICT_FEW], hole[EVICT_FEW], mover[EVICT_FEW];
  const int t = threadIdx.x, g = blockIdx.x, n = p.n, budget = p.budget, drop = n - budget;
  const float* w = p.w + int64_t(g) * p.whs;
  const int32_t* pos = p.pos + int64_t(g) * p.phs;
  float x[E];
  int32_t y[E];
  int newest = INT32_MIN;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int r = t + 1024 * e;
    x[e] = r < n ? w[r] : 0.0f;
    y[e] = r < n ? pos[r] : INT32_MIN;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) newest = max(newest, y[e]);
  const int64_t old = int64_t(evict_max(newest, red)) - p.recent;
  uint32_t key[E], gone = 0;  // (this thread's rows that are not there)
#pragma unroll
  for (int e = 0; e < E; ++e) {
    key[e] = evict_key(x[e], y[e], old);
    gone |= t + 1024 * e < n ? 0u : 1u << e;
  }
#pragma unroll 1
  for (int j = 0; j < drop; ++j) {
    uint64_t m = ~0ull;  // (at least two rows are left: none is ~0 but the last)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (!(gone >> e & 1u)) m = min(m, evict_place(key[e], t + 1024 * e));
    const int r = int(~uint32_t(evict_min(m, least[j & 1])));
    if ((r & 1023) == t) gone |= 1u << (r >> 10);
    if (t == 0) out[j] = r;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int r = t + 1024 * e;
    if (r < budget && !(gone >> e & 1u)) {
      p.kept[int64_t(g) * p.khs + r] = r;
      p.w_out[int64_t(g) * p.wos + r] = x[e];
      p.pos_out[int64_t(g) * p.pos_os + r] = y[e];
    }
  }
  __syncthreads();
  evict_few_move(p, g, out, hole, mover);
}

// A chunk's rows of thread t: chunk * 4096 + 256 (t / 64) + t % 64, + 64, + 128, + 192.
struct EvictRows {
  float w[4];
  int32_t pos[4];
  int row0;
};
__device__ __forceinline__ EvictRows evict_rows(const EvictParams& p, int g, int c) {
  EvictRows x;
  x.row0 = c * EVICT_CHUNK + 256 * int(threadIdx.x >> 6) + int(threadIdx.x & 63);
  const float* w = p.w + int64_t(g) * p.whs;
  const int32_t* pos = p.pos + int64_t(g) * p.phs;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = x.row0 + 64 * e;
    x.w[e] = r < p.n ? w[r] : 0.0f;
    x.pos[e] = r < p.n ? pos[r] : INT32_MIN;
  }
  return x;
}
// Rows of a position up to this one are not `recent`: from the chunks' newest.
__device__ __forceinline__ int64_t evict_old(const EvictParams& p, int g, int* red) {
  int newest = INT32_MIN;
  for (int c = threadIdx.x; c < p.nch; c += 1024) newest = max(newest, p.info[(int64_t(g) * p.nch + c) * EVICT_INFO]);
  return int64_t(evict_max(newest, red)) - p.recent;
}

__global__ __launch_bounds__(1024) void evict_newest_kernel(EvictParams p) {
  __shared__ int red[EVICT_NW];
  const int c = blockIdx.x, g = blockIdx.y;
  const int32_t* pos = p.pos + int64_t(g) * p.phs;
  int newest = INT32_MIN;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = c * EVICT_CHUNK + 1024 * e + int(threadIdx.x);
    if (r < p.n) newest = max(newest, pos[r]);
  }
  newest = evict_max(newest, red);
  if (threadIdx.x == 0) p.info[(int64_t(g) * p.nch + c) * EVICT_INFO] = newest;
}

__global__ __launch_bounds__(1024) void evict_digit_kernel(EvictParams p) {
  __shared__ uint32_t hist[2048];
  __shared__ int red[EVICT_NW];
  const int t = threadIdx.x, c = blockIdx.x, g = blockIdx.y;
  const EvictRows x = evict_rows(p, g, c);
  hist[t] = 0u;
  hist[t + 1024] = 0u;
  const int64_t old = evict_old(p, g, red);  // (its barrier: hist is cleared)
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (x.row0 + 64 * e < p.n) atomicAdd(&hist[evict_key(x.w[e], x.pos[e], old) >> 21], 1u);
  __syncthreads();
  // word t: digits 2047 - 2 t (low half) and 2046 - 2 t
  p.digit[(int64_t(g) * p.nch + c) * 1024 + t] = hist[2047 - 2 * t] | (hist[2046 - 2 * t] << 16);
}

__global__ __launch_bounds__(1024) void evict_split_kernel(EvictParams p) {
  __shared__ int red[EVICT_NW], red2[EVICT_NW], sums[4];
  __shared__ uint32_t digit_s;
  __shared__ int need_s;
  const int t = threadIdx.x, lane = t & 63, c = blockIdx.x, g = blockIdx.y;
  const EvictRows x = evict_rows(p, g, c);
  const int64_t old = evict_old(p, g, red);
  int c0 = 0, c1 = 0;
  const uint32_t* dg = p.digit + int64_t(g) * p.nch * 1024 + t;
#pragma unroll 8
  for (int i = 0; i < p.nch; ++i) {
    const uint32_t v = dg[int64_t(i) * 1024];
    c0 += int(v & 0xffffu);
    c1 += int(v >> 16);
  }
  if (t < 4) sums[t] = 0;
  uint32_t digit;
  int need = p.budget;
  evict_pick(c0, c1, red2, &digit_s, &need_s, digit, need);
  // rows of larger digits are kept; those of the digit are left open, listed in row order
  uint32_t key[4];
  int nopen = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool ok = x.row0 + 64 * e < p.n;
    key[e] = ok ? evict_key(x.w[e], x.pos[e], old) : 0u;
    nopen += evict_count(ok && key[e] >> 21 == digit);
  }
  __syncthreads();  // (red2 has been read)
  int at = evict_before(nopen, red2);
  uint32_t* const open = p.open + (int64_t(g) * p.nch + c) * EVICT_CHUNK;
  int cnt[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool ok = x.row0 + 64 * e < p.n, low = x.row0 + 64 * e < p.budget;
    const bool is_open = ok && key[e] >> 21 == digit, above = ok && key[e] >> 21 > digit;
    if (is_open) open[at + evict_rank(is_open)] = key[e];
    at += evict_count(is_open);
    cnt[0] += evict_count(above && low);
    cnt[1] += evict_count(above && !low);
    cnt[2] += evict_count(is_open && low);
    cnt[3] += evict_count(is_open && !low);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane == 0) atomicAdd(&sums[i], cnt[i]);
  __syncthreads();
  int32_t* const info = p.info + (int64_t(g) * p.nch + c) * EVICT_INFO;
  if (t < 4) info[1 + t] = sums[t];
  if (c == 0 && t == 0) {
    p.least[2 * g] = int32_t(digit);
    p.least[2 * g + 1] = need;
  }
}

__global__ __launch_bounds__(1024) void evict_least_kernel(EvictParams p) {
  __shared__ uint32_t hist[2048];
  __shared__ int red[EVICT_NW];
  __shared__ uint32_t digit_s;
  __shared__ int need_s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, g = blockIdx.x;
  int32_t* const info = p.info + int64_t(g) * p.nch * EVICT_INFO;
  const uint32_t* const open = p.open + int64_t(g) * p.nch * EVICT_CHUNK;
  uint32_t prefix = uint32_t(p.least[2 * g]) << 21, digit;
  int need = p.least[2 * g + 1];
  hist[t] = 0u;
  hist[t + 1024] = 0u;
  __syncthreads();
#pragma unroll 1
  for (int d = 1; d < 3; ++d) {
    const int shift = d == 1 ? 10 : 0;
    const uint32_t mask = d == 1 ? 0u : 0x001ffc00u, digits = d == 1 ? 2047u : 1023u;
    for (int c = wave; c < p.nch; c += EVICT_NW) {  // a wave per chunk
      const int m = info[c * EVICT_INFO + 3] + info[c * EVICT_INFO + 4];
#pragma unroll 4
      for (int i = lane; i < m; i += 64) {
        const uint32_t k = open[int64_t(c) * EVICT_CHUNK + i];
        if ((k & mask) == (prefix & mask)) atomicAdd(&hist[(k >> shift) & digits], 1u);
      }
    }
    __syncthreads();
    const int hi = 2047 - 2 * t, c0 = int(hist[hi]), c1 = int(hist[hi - 1]);
    hist[hi] = 0u;
    hist[hi - 1] = 0u;
    evict_pick(c0, c1, red, &digit_s, &need_s, digit, need);
    prefix |= digit << shift;
    __syncthreads();
  }
  // of each chunk: kept rows below the budget and from it on but for the equal ones, and those
  for (int c = wave; c < p.nch; c += EVICT_NW) {
    int32_t* const x = info + c * EVICT_INFO;
    const int nlow = x[3], m = nlow + x[4];
    int gl = 0, gh = 0, el = 0, eh = 0;
#pragma unroll 4
    for (int i0 = 0; i0 < m; i0 += 64) {
      const int i = i0 + lane;
      const uint32_t k = i < m ? open[int64_t(c) * EVICT_CHUNK + i] : 0u;
      const bool low = i < nlow, gt = i < m && k > prefix, eq = i < m && k == prefix;
      gl += evict_count(gt && low);
      gh += evict_count(gt && !low);
      el += evict_count(eq && low);
      eh += evict_count(eq && !low);
    }
    if (lane == 0) x[1] += gl, x[2] += gh, x[3] = el, x[4] = eh;
  }
  __threadfence_block();
  __syncthreads();
  // what is before each chunk: one thread, over the chunks (their counts asked for eight at a time)
  if (t != 0) return;
  int eq = 0, hole = 0, move = 0;
  for (int c0 = 0; c0 < p.nch; c0 += 8) {
    int x[8][4];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][i] = c0 + u < p.nch ? info[(c0 + u) * EVICT_INFO + 1 + i] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int c = c0 + u;
      if (c >= p.nch) break;
      const int first = c * EVICT_CHUNK, rows = min(EVICT_CHUNK, p.n - first), low = max(0, min(rows, p.budget - first));
      int32_t* const o = info + c * EVICT_INFO;
      o[3] = eq;
      o[4] = hole;
      o[5] = move;
      const int take_low = max(0, min(x[u][2], need - eq));
      eq += x[u][2];
      const int take_high = max(0, min(x[u][3], need - eq));
      eq += x[u][3];
      hole += low - x[u][0] - take_low;
      move += x[u][1] + take_high;
    }
  }
  p.least[2 * g] = int32_t(prefix);
  p.least[2 * g + 1] = need;
  p.count[g] = hole;
}

__global__ __launch_bounds__(1024) void evict_list_kernel(EvictParams p) {
  __shared__ int red[EVICT_NW], red2[EVICT_NW], red3[EVICT_NW], red4[EVICT_NW];
  const int c = blockIdx.x, g = blockIdx.y, budget = p.budget;
  const EvictRows x = evict_rows(p, g, c);
  const int64_t old = evict_old(p, g, red);
  const uint32_t least = uint32_t(p.least[2 * g]);
  const int need = p.least[2 * g + 1];
  const int32_t* const info = p.info + (int64_t(g) * p.nch + c) * EVICT_INFO;
  uint32_t key[4];
  int neq = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool ok = x.row0 + 64 * e < p.n;
    key[e] = ok ? evict_key(x.w[e], x.pos[e], old) : 0u;
    neq += evict_count(ok && key[e] == least);
  }
  int seen = info[3] + evict_before(neq, red2);
  bool keep[4];
  int nhole = 0, nmove = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = x.row0 + 64 * e;
    const bool ok = r < p.n, eq = ok && key[e] == least, low = r < budget;
    keep[e] = ok && (key[e] > least || (eq && seen + evict_rank(eq) < need));
    seen += evict_count(eq);
    nhole += evict_count(low && !keep[e]);
    nmove += evict_count(!low && keep[e]);
  }
  int hole = info[4] + evict_before(nhole, red3), move = info[5] + evict_before(nmove, red4);
  int32_t* const holes = p.hole + int64_t(g) * p.most;
  int32_t* const movers = p.mover + int64_t(g) * p.most;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = x.row0 + 64 * e;
    const bool low = r < budget, is_hole = low && !keep[e], is_move = !low && keep[e];
    if (is_hole) holes[hole + evict_rank(is_hole)] = r;
    if (is_move) movers[move + evict_rank(is_move)] = r;
    hole += evict_count(is_hole);
    move += evict_count(is_move);
    if (low && keep[e]) {
      p.kept[int64_t(g) * p.khs + r] = r;
      p.w_out[int64_t(g) * p.wos + r] = x.w[e];
      p.pos_out[int64_t(g) * p.pos_os + r] = x.pos[e];
    }
  }
}

// Long caches of which a few rows go: each chunk's least rows, then the least of those (of 65521 rows of 8 heads of
// 128 one in 10.6 us, six in 21.5, seven by the digits in 32.9).
__global__ __launch_bounds__(1024) void evict_few_chunk_kernel(EvictParams p) {
  __shared__ uint64_t least[2][EVICT_NW];
  __shared__ int red[EVICT_NW];
  const int c = blockIdx.x, g = blockIdx.y, drop = p.n - p.budget;
  const EvictRows x = evict_rows(p, g, c);
  const int64_t old = evict_old(p, g, red);
  uint64_t place[4], from = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = x.row0 + 64 * e;
    place[e] = r < p.n ? evict_place(evict_key(x.w[e], x.pos[e], old), r) : ~0ull;
    if (r < p.budget) {  // (the rows that go are overwritten by the next kernel)
      p.kept[int64_t(g) * p.khs + r] = r;
      p.w_out[int64_t(g) * p.wos + r] = x.w[e];
      p.pos_out[int64_t(g) * p.pos_os + r] = x.pos[e];
    }
  }
  uint32_t* const open = p.open + (int64_t(g) * p.nch + c) * EVICT_CHUNK;
#pragma unroll 1
  for (int j = 0; j < drop; ++j) {
    uint64_t m = ~0ull;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (place[e] >= from) m = min(m, place[e]);
    m = evict_min(m, least[j & 1]);
    if (threadIdx.x == 0) open[2 * j] = uint32_t(m), open[2 * j + 1] = uint32_t(m >> 32);
    from = m == ~0ull ? m : m + 1;  // (no two are alike; ~0: none is left)
  }
}

__global__ __launch_bounds__(1024) void evict_few_last_kernel(EvictParams p) {
  __shared__ uint64_t least[2][EVICT_NW];
  __shared__ int out[EVICT_FEW], hole[EVICT_FEW], mover[EVICT_FEW];
  const int t = threadIdx.x, g = blockIdx.x, drop = p.n - p.budget;
  const uint32_t* const open = p.open + int64_t(g) * p.nch * EVICT_CHUNK;
  uint64_t from = 0;
#pragma unroll 1
  for (int j = 0; j < drop; ++j) {
    uint64_t m = ~0ull;
    for (int i = t; i < p.nch * drop; i += 1024) {
      const uint32_t* const o = open + int64_t(i / drop) * EVICT_CHUNK + 2 * (i % drop);
      const uint64_t v = uint64_t(o[1]) << 32 | o[0];
      if (v >= from) m = min(m, v);
    }
    m = evict_min(m, least[j & 1]);
    if (t == 0) out[j] = int(~uint32_t(m));
    from = m + 1;
  }
  __syncthreads();
  evict_few_move(p, g, out, hole, mover);
}

__global__ __launch_bounds__(256) void evict_move_kernel(EvictParams p) {
  const int g = blockIdx.y;
  const int64_t total = int64_t(p.count[g]) * p.row_cols;
  const int32_t* const holes = p.hole + int64_t(g) * p.most;
  const int32_t* const movers = p.mover + int64_t(g) * p.most;
  char* const k = p.k + int64_t(g) * p.kh;
  char* const v = p.v + int64_t(g) * p.vh;
  for (int64_t x = int64_t(blockIdx.x) * 256 + threadIdx.x; x < total; x += int64_t(gridDim.x) * 256) {
    const int m = int(x / p.row_cols);
    const int col = int(x % p.row_cols);
    const int64_t dst = holes[m], src = movers[m], c = int64_t(col) * 16;
    const v4u a = *reinterpret_cast<const v4u*>(k + src * p.kr + c);
    const v4u b = *reinterpret_cast<const v4u*>(v + src * p.vr + c);
    *reinterpret_cast<v4u*>(k + dst * p.kr + c) = a;
    *reinterpret_cast<v4u*>(v + dst * p.vr + c) = b;
    if (col == 0) {
      p.kept[int64_t(g) * p.khs + dst] = int32_t(src);
      p.w_out[int64_t(g) * p.wos + dst] = p.w[int64_t(g) * p.whs + src];
      p.pos_out[int64_t(g) * p.pos_os + dst] = p.pos[int64_t(g) * p.phs + src];
    }
  }
}

}  // namespace w8a8

using namespace w8a8;

// (No kernel of 8 rows: the compiler makes a path for every set of rows that move, at 222 registers, and the 16
// rows' kernel is faster: 8 beams of 8191 rows, four layers, 204 -> 158 us.)
template <class C>
static void reorder_launch(const ReorderParams& p, int64_t blocks, hipStream_t stream) {
  const dim3 grid{unsigned(blocks), unsigned(p.nouter), 1};
  if (p.n <= 4)
    reorder_kernel<C, 4><<<grid, 256, 0, stream>>>(p);
  else if (p.n <= 16)
    reorder_kernel<C, 16><<<grid, 256, 0, stream>>>(p);
  else if (p.n <= 32)
    reorder_kernel<C, 32><<<grid, 256, 0, stream>>>(p);
  else
    reorder_kernel<C, 64><<<grid, 256, 0, stream>>>(p);
}

extern "C" int w8a8_reorder_rows(const w8a8_rows *tensors, int64_t count, const int64_t* index, int64_t index_stride,
                                 int64_t n, int64_t size, int64_t outer, hipStream_t stream) {
  const char* what = "reorder_rows";
  if (count < 0 || n < 0 || size < 1 || outer < 1 || outer > 65535 || size > INT32_MAX)
    return fail(W8A8_EINVAL, "%s: count=%lld n=%lld size=%lld outer=%lld", what, (long long)count, (long long)n,
                (long long)size, (long long)outer);
  if (n > REORDER_MAX || n > size)
    return fail(W8A8_ENOTSUP, "%s: %lld rows of %lld (at most %d)", what, (long long)n, (long long)size, REORDER_MAX);
  if (count == 0 || n == 0) return W8A8_OK;
  if (!tensors || !index) return fail(W8A8_EINVAL, "%s: null pointer", what);
  if ((uintptr_t)index % 8) return fail(W8A8_EALIGN, "%s: index must be 8-byte aligned", what);
  if (outer > 1 && index_stride != 0 && index_stride < n) return fail(W8A8_EINVAL, "%s: index stride", what);
  int64_t align = 16;
  for (int64_t i = 0; i < count; ++i) {
    const w8a8_rows& r = tensors[i];
    if (r.runs < 0 || r.run_bytes < 0 || r.runs > INT32_MAX || (r.runs > 0 && r.run_bytes > 0 && !r.data))
      return fail(W8A8_EINVAL, "%s: tensor %lld", what, (long long)i);
    if (r.runs == 0 || r.run_bytes == 0) continue;
    // rows that share bytes cannot be put in order
    if ((size > 1 && r.axis_stride <= 0) || (outer > 1 && r.outer_stride <= 0) || (r.runs > 1 && r.run_stride < r.run_bytes) ||
        (size > 1 && r.axis_stride < r.run_bytes))
      return fail(W8A8_EINVAL, "%s: tensor %lld: strides must be positive and rows must not overlap", what, (long long)i);
    // the same memory twice (a cache that two layers share) would be read and written by two workgroups
    for (int64_t j = 0; j < i; ++j)
      if (tensors[j].data == r.data && tensors[j].runs > 0 && tensors[j].run_bytes > 0)
        return fail(W8A8_EINVAL, "%s: tensors %lld and %lld are the same memory", what, (long long)j, (long long)i);
    for (int64_t x : {int64_t(reinterpret_cast<uintptr_t>(r.data)), size > 1 ? r.axis_stride : 0, outer > 1 ? r.outer_stride : 0,
                      r.runs > 1 ? r.run_stride : 0, r.run_bytes})
      while (x % align != 0) align = align == 16 ? 4 : 1;
  }
  // an index among the rows that change would be read and written at once
  const uintptr_t at = reinterpret_cast<uintptr_t>(index), behind = at + ((outer > 1 ? (outer - 1) * index_stride : 0) + n) * 8;
  for (int64_t i = 0; i < count; ++i) {
    const w8a8_rows& r = tensors[i];
    if (r.runs == 0 || r.run_bytes == 0) continue;
    const uintptr_t first = reinterpret_cast<uintptr_t>(r.data);
    const int64_t bytes = (outer > 1 ? (outer - 1) * r.outer_stride : 0) + (n > 1 ? (n - 1) * r.axis_stride : 0) +
                          (r.runs > 1 ? (r.runs - 1) * r.run_stride : 0) + r.run_bytes;
    if (at < first + bytes && first < behind) return fail(W8A8_EINVAL, "%s: the index lies in tensor %lld", what, (long long)i);
  }
  // (the last refusal: from here on tensors change)
  for (int64_t i = 0; i < count; ++i)
    if (tensors[i].runs > 0 && tensors[i].run_bytes / align > INT32_MAX / tensors[i].runs)
      return fail(W8A8_ENOTSUP, "%s: tensor %lld too large", what, (long long)i);
  for (int64_t i0 = 0; i0 < count;) {
    ReorderParams p{};
    p.index = index; p.is = outer > 1 ? index_stride : 0; p.n = int(n); p.size = int(size); p.nouter = int(outer);
    int64_t blocks = 0;
    for (; i0 < count && p.ntensors < REORDER_TENSORS; ++i0) {
      const w8a8_rows& r = tensors[i0];
      if (r.runs == 0 || r.run_bytes == 0) continue;
      ReorderTensor& d = p.t[p.ntensors];
      d.base = static_cast<char*>(r.data);
      d.axis = r.axis_stride; d.outer = r.outer_stride; d.inner = r.run_stride;
      d.run = r.run_bytes / align; d.ninner = int(r.runs);
      const int64_t b = (d.run * d.ninner + 255) / 256;
      if (blocks + b > REORDER_BLOCKS) break;  // (one tensor never has so many)
      d.block0 = int(blocks);
      blocks += b;
      ++p.ntensors;
    }
    if (p.ntensors == 0) return W8A8_OK;  // (only empty tensors were left)
    if (align == 16)
      reorder_launch<v4u>(p, blocks, stream);
    else if (align == 4)
      reorder_launch<uint32_t>(p, blocks, stream);
    else
      reorder_launch<uint8_t>(p, blocks, stream);
  }
  return check_launch(what);
}

// Chunks of a head's rows (0: one workgroup chooses).
static int64_t evict_chunks(int64_t n) { return n <= EVICT_ONE ? 0 : (n + EVICT_CHUNK - 1) / EVICT_CHUNK; }

extern "C" int64_t w8a8_evict_workspace_bytes(int64_t KV, int64_t n, int64_t budget) {
  if (KV < 1 || KV > 65535 || n < 1 || n > INT32_MAX / 2 || budget < 1 || budget > n) return -1;
  return KV * (3 + 2 * std::min(budget, n - budget) + evict_chunks(n) * (EVICT_INFO + 1024 + EVICT_CHUNK)) * 4;
}

extern "C" int w8a8_evict(void* k, int64_t k_head_stride, int64_t k_row_stride, void* v, int64_t v_head_stride,
                          int64_t v_row_stride, int64_t row_bytes, int64_t KV, int64_t n, const float* weights,
                          int64_t weights_stride, const int32_t* positions, int64_t positions_stride, int64_t budget,
                          int64_t recent, int32_t* kept, int64_t kept_stride, float* weights_out,
                          int64_t weights_out_stride, int32_t* positions_out, int64_t positions_out_stride,
                          void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const char* what = "evict";
  const int64_t need = w8a8_evict_workspace_bytes(KV, n, budget);
  if (need < 0 || recent < 0 || recent > budget)
    return fail(W8A8_EINVAL, "%s: KV=%lld n=%lld budget=%lld recent=%lld (1 <= budget <= n, recent <= budget)", what,
                (long long)KV, (long long)n, (long long)budget, (long long)recent);
  if (!k || !v || !weights || !positions || !kept || !weights_out || !positions_out || !workspace)
    return fail(W8A8_EINVAL, "%s: null pointer", what);
  if (workspace_bytes < need)
    return fail(W8A8_EINVAL, "%s: workspace of %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  if (row_bytes < 16 || row_bytes > (1 << 20)) return fail(W8A8_EINVAL, "%s: rows of %lld bytes", what, (long long)row_bytes);
  if (KV == 1) k_head_stride = v_head_stride = 0;
  if ((n > 1 && (k_row_stride < row_bytes || v_row_stride < row_bytes)) || k_head_stride < 0 || v_head_stride < 0 ||
      (KV > 1 && (k_head_stride < row_bytes || v_head_stride < row_bytes)))
    return fail(W8A8_EINVAL, "%s: strides smaller than the rows", what);
  if (KV > 1 && (weights_stride < n || positions_stride < n || kept_stride < budget || weights_out_stride < budget ||
                 positions_out_stride < budget))
    return fail(W8A8_EINVAL, "%s: strides of weights, positions or the outputs smaller than their rows", what);
  for (int64_t x : {int64_t(uintptr_t(k)), int64_t(uintptr_t(v)), k_head_stride, v_head_stride, n > 1 ? k_row_stride : 0,
                    n > 1 ? v_row_stride : 0, row_bytes})
    if (x % 16 != 0) return fail(W8A8_EALIGN, "%s: k, v, their strides and rows must be multiples of 16 bytes", what);
  for (const void* x : {(const void*)weights, (const void*)positions, (const void*)kept, (const void*)weights_out,
                        (const void*)positions_out, (const void*)workspace})
    if (uintptr_t(x) % 4 != 0) return fail(W8A8_EALIGN, "%s: weights, positions, outputs and workspace 4-byte aligned", what);
  EvictParams p{};
  p.w = weights; p.whs = KV > 1 ? weights_stride : 0; p.pos = positions; p.phs = KV > 1 ? positions_stride : 0;
  p.n = int(n); p.budget = int(budget); p.recent = int(recent);
  p.kept = kept; p.khs = KV > 1 ? kept_stride : 0; p.w_out = weights_out; p.wos = KV > 1 ? weights_out_stride : 0;
  p.pos_out = positions_out; p.pos_os = KV > 1 ? positions_out_stride : 0;
  p.most = int(std::min(budget, n - budget));
  p.nch = int(evict_chunks(n));
  p.count = static_cast<int32_t*>(workspace);
  p.least = p.count + KV;
  p.hole = p.least + 2 * KV;
  p.mover = p.hole + KV * p.most;
  p.info = p.mover + KV * p.most;
  p.digit = reinterpret_cast<uint32_t*>(p.info + KV * p.nch * EVICT_INFO);
  p.open = p.digit + KV * p.nch * 1024;
  p.k = static_cast<char*>(k); p.kh = k_head_stride; p.kr = k_row_stride;
  p.v = static_cast<char*>(v); p.vh = v_head_stride; p.vr = v_row_stride;
  p.row_cols = int(row_bytes / 16);
  if (n > budget && n - budget <= EVICT_FEW && (n - budget) * p.row_cols <= EVICT_FEW_COLS) {
    if (p.nch > 0) {
      const dim3 grid{unsigned(p.nch), unsigned(KV), 1};
      evict_newest_kernel<<<grid, 1024, 0, stream>>>(p);
      evict_few_chunk_kernel<<<grid, 1024, 0, stream>>>(p);
      evict_few_last_kernel<<<unsigned(KV), 1024, 0, stream>>>(p);
    } else if (n <= 4 * 1024) {
      evict_few_kernel<4><<<unsigned(KV), 1024, 0, stream>>>(p);
    } else if (n <= 8 * 1024) {
      evict_few_kernel<8><<<unsigned(KV), 1024, 0, stream>>>(p);
    } else {
      evict_few_kernel<16><<<unsigned(KV), 1024, 0, stream>>>(p);
    }
    return check_launch(what);
  }
  if (p.nch == 0) {
    evict_select_kernel<<<unsigned(KV), 1024, 0, stream>>>(p);
  } else {
    const dim3 grid{unsigned(p.nch), unsigned(KV), 1};
    evict_newest_kernel<<<grid, 1024, 0, stream>>>(p);
    evict_digit_kernel<<<grid, 1024, 0, stream>>>(p);
    evict_split_kernel<<<grid, 1024, 0, stream>>>(p);
    evict_least_kernel<<<unsigned(KV), 1024, 0, stream>>>(p);
    evict_list_kernel<<<grid, 1024, 0, stream>>>(p);
  }
  if (p.most > 0) {
    const int64_t blocks = std::min<int64_t>((int64_t(p.most) * p.row_cols + 255) / 256, 2048);
    evict_move_kernel<<<dim3{unsigned(blocks), unsigned(KV), 1}, 256, 0, stream>>>(p);
  }
  return check_launch(what);
}
