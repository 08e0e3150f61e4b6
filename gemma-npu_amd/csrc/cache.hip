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
  const int64_t col = int64_t(int(blockIdx.x) - d.block0) * 256 + threadIdx.x;
  const int64_t per = d.run * d.ninner;
  const int o = blockIdx.y;
  const bool on = col < per;
  char* base = d.base + int64_t(o) * d.outer + (on ? (col / d.run) * d.inner + (col % d.run) * int64_t(sizeof(C)) : 0);
  const int64_t* index = p.index + int64_t(o) * p.is;
  C v[N];
  int64_t src[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    src[i] = i;
    if (i < p.n) {
      const int64_t s = index[i];
      if (s >= 0 && s < p.size) src[i] = s;  // an index outside the axis leaves the row as it is
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (src[i] != i && on) v[i] = *reinterpret_cast<const C*>(base + src[i] * d.axis);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (src[i] != i && on) *reinterpret_cast<C*>(base + int64_t(i) * d.axis) = v[i];
}

// ---- a cache cut to its budget ---------------------------------------------------------------------------
//
// Per KV head, of n rows `budget` are kept: those whose position is within `recent` of the newest one, then
// those of the largest weight (NaN the largest; ties: the lower row).  Attention does not depend on the order
// of the rows, so the kept rows below the budget stay where they are and the others move, in order, into
// the places that became free: the least that can be moved, in place, and no row is both read and written.
//
// evict_select_kernel: one workgroup per KV head reads the weights and positions once into registers and
// finds the budget-th largest key by a radix select over digits of 11, 11 and 10 bits; the first digit's
// counting is the only one that all rows take part in.  Every wave owns a run of rows, so what comes before
// it in row order is a sum over the waves before.  Up to EVICT_FUSED rows the waves then walk their rows with
// ballots and list the free places and the moving rows; above that one workgroup per KV head would be walking
// alone for long, so it leaves the sums before each segment of 1024 rows, and evict_list_kernel lists them
// from a workgroup per segment.  evict_move_kernel copies the rows.  In all the keys are read by
// one CU per head, which bounds the choice: 64 KiB rows of 8 heads 242 us reading them again at each step,
// @SEL@

constexpr int EVICT_NW = 16;
constexpr int EVICT_SEG = 1024;            // rows per workgroup of evict_list_kernel
constexpr int EVICT_FUSED = 1024 * 16;

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
  int32_t* head;                        // [KV][4] newest position - recent as two words, the least key kept, how many of it
  int32_t* before;                      // [KV][nseg][3] equal keys, free places and moving rows before a segment
  int most;                             // min(budget, n - budget)
  int steps, nsub, nseg;                // steps of 64 rows per wave; segments per wave and per head
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

// E rows per thread in registers (n <= 1024 E), or with E = 0 read again at each step.
template <int E>
__global__ __launch_bounds__(1024) void evict_select_kernel(EvictParams p) {
  constexpr bool LISTS = E > 0 && E <= 16;
  constexpr int SEG_STEPS = EVICT_SEG / 64;
  __shared__ uint32_t hist[2048];
  __shared__ int red[EVICT_NW], red2[EVICT_NW];
  __shared__ uint32_t digit_s;
  __shared__ int need_s;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = blockIdx.x;
  const float* w = p.w + int64_t(g) * p.whs;
  const int32_t* pos = p.pos + int64_t(g) * p.phs;
  const int n = p.n, budget = p.budget, steps = p.steps;
  const int wave0 = wave * steps * 64, row0 = wave0 + lane;  // this wave's rows: steps of 64 from wave0 on

  uint32_t key[E > 0 ? E : 1];
  int32_t ps[LISTS ? E : 1];
  int newest = INT32_MIN;
  if constexpr (LISTS) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int r = row0 + 64 * e;
      const bool ok = e < steps && r < n;
      ps[e] = ok ? pos[r] : INT32_MIN;
      key[e] = ok ? __float_as_uint(w[r]) : 0u;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) newest = max(newest, ps[e]);
  } else {
    for (int r = t; r < n; r += 8192) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (r + 1024 * u < n) newest = max(newest, pos[r + 1024 * u]);
    }
  }
  hist[t] = 0u;
  hist[t + 1024] = 0u;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) newest = max(newest, __shfl_xor(newest, o, 64));
  if (lane == 0) red[wave] = newest;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < EVICT_NW; ++x) newest = max(newest, red[x]);
  const int64_t old = int64_t(newest) - p.recent;
  if constexpr (LISTS) {
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = evict_key(__uint_as_float(key[e]), ps[e], old);
  } else if constexpr (E > 0) {
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(w, uint32_t(n) * 4u), rp = make_rsrc(pos, uint32_t(n) * 4u);
    const int left = min(n, wave0 + steps * 64) - row0;  // this lane's rows are those of 64 e below it
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t off = uint32_t(row0 + 64 * e) * 4u;
      const float x = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rw, off, 0, 0));
      const int32_t y = int32_t(__builtin_amdgcn_raw_buffer_load_b32(rp, off, 0, 0));
      key[e] = 64 * e < left ? evict_key(x, y, old) : 0u;
      if (e % 16 == 15) __builtin_amdgcn_sched_barrier(0);  // (all 128 loads at once would spill)
    }
  }
  // f(key, step) for each of this thread's rows, in order; the whole wave takes part in each step
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < steps) f(key[e], e);
    } else {
      for (int e0 = 0; e0 < steps; e0 += 8) {
        uint32_t k[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int r = row0 + 64 * (e0 + u);
          k[u] = e0 + u < steps && r < n ? evict_key(w[r], pos[r], old) : 0u;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (e0 + u < steps) f(k[u], e0 + u);
      }
    }
  };

  // the budget-th largest key: its digits from the top, and how many of the rows with that key are kept
  uint32_t prefix = 0;
  int need = budget;
#pragma unroll 1
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    const uint32_t digits = d == 2 ? 1023u : 2047u, mask = d == 0 ? 0u : d == 1 ? 0xffe00000u : 0xfffffc00u;
    // (keys of no row are the smallest: they count in digits that are never reached)
    each([&](uint32_t k, int) {
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digits], 1u);
    });
    __syncthreads();
    // thread t: digits hi and hi - 1; larger digits are with the threads before it
    const int hi = 2047 - 2 * t;
    const int c0 = int(hist[hi]), c1 = int(hist[hi - 1]);
    hist[hi] = 0u;
    hist[hi - 1] = 0u;
    int above = c0 + c1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(above, o, 64);
      if (lane >= o) above += v;
    }
    if (lane == 63) red[wave] = above;
    __syncthreads();
    for (int x = 0; x < wave; ++x) above += red[x];
    above -= c0 + c1;  // rows of larger digits
    if (above < need && above + c0 >= need) digit_s = uint32_t(hi), need_s = need - above;
    if (above + c0 < need && above + c0 + c1 >= need) digit_s = uint32_t(hi - 1), need_s = need - above - c0;
    __syncthreads();
    prefix |= digit_s << shift;
    need = need_s;
  }

  // sum over the waves before this one
  auto scan = [&](int v, int* buf) __attribute__((always_inline)) {
    if (lane == 0) buf[wave] = v;
    __syncthreads();
    int s = 0;
    for (int x = 0; x < wave; ++x) s += buf[x];
    return s;
  };
  if constexpr (LISTS) {
    int neq = 0;
    each([&](uint32_t k, int) { neq += __popcll(__builtin_amdgcn_ballot_w64(k == prefix)); });
    int seen = scan(neq, red2);
    const uint64_t below = (1ull << lane) - 1ull;
    uint32_t keep_bits = 0;
    int nhole = 0, nmove = 0;
    each([&](uint32_t k, int e) {
      const uint64_t b = __builtin_amdgcn_ballot_w64(k == prefix);
      const bool keep = k > prefix || (k == prefix && seen + __popcll(b & below) < need);
      seen += __popcll(b);
      keep_bits |= keep ? 1u << e : 0u;
      const bool low = row0 + 64 * e < budget;
      nhole += __popcll(__builtin_amdgcn_ballot_w64(low && !keep));
      nmove += __popcll(__builtin_amdgcn_ballot_w64(!low && keep));
    });
    __syncthreads();
    int hole = scan(nhole, red), move = scan(nmove, red2);
    int32_t* const holes = p.hole + int64_t(g) * p.most;
    int32_t* const movers = p.mover + int64_t(g) * p.most;
    int32_t* const ko = p.kept + int64_t(g) * p.khs;
    float* const wo = p.w_out + int64_t(g) * p.wos;
    int32_t* const po = p.pos_out + int64_t(g) * p.pos_os;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < steps) {
        const int r = row0 + 64 * e;
        const bool keep = (keep_bits >> e) & 1u, low = r < budget;
        const uint64_t bh = __builtin_amdgcn_ballot_w64(low && !keep), bm = __builtin_amdgcn_ballot_w64(!low && keep);
        if (low && !keep) holes[hole + __popcll(bh & below)] = r;
        if (!low && keep) movers[move + __popcll(bm & below)] = r;
        hole += __popcll(bh);
        move += __popcll(bm);
        if (low && keep) ko[r] = r, wo[r] = w[r], po[r] = ps[e];
      }
    if (wave == EVICT_NW - 1 && lane == 0) p.count[g] = hole;
  } else {
    // per segment of this wave: rows of larger keys and of equal ones, below the budget and from it on
    int32_t* const bf = p.before + (int64_t(g) * p.nseg + wave * p.nsub) * 3;
    int gt = 0, eq = 0, gt_low = 0, eq_low = 0;           // this lane's, of the segment so far
    int all_eq = 0;                                       // the wave's
    auto flush = [&](int j) __attribute__((always_inline)) {
      int v[4] = {gt, eq, gt_low, eq_low};
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v[x] += __shfl_xor(v[x], o, 64);
      // packed for the second round: (larger, equal) counts of the segment and of its part below the budget
      if (lane == 0) bf[3 * j] = v[0] | (v[1] << 16), bf[3 * j + 1] = v[2] | (v[3] << 16);
      all_eq += v[1];
      gt = eq = gt_low = eq_low = 0;
    };
    each([&](uint32_t k, int e) {
      const bool low = row0 + 64 * e < budget, a = k > prefix, b = k == prefix;
      gt += a ? 1 : 0;
      eq += b ? 1 : 0;
      gt_low += a && low ? 1 : 0;
      eq_low += b && low ? 1 : 0;
      if (e % SEG_STEPS == SEG_STEPS - 1 || e == steps - 1) flush(e / SEG_STEPS);
    });
    int seen = scan(all_eq, red2);
    // lane 0 turns the counts into the sums before each segment
    int nhole = 0, nmove = 0;
    if (lane == 0) {
      int s = seen;
      for (int j = 0; j < p.nsub; ++j) {
        const int a = bf[3 * j], b = bf[3 * j + 1];
        const int eqs = a >> 16, eql = b >> 16, first = wave0 + j * EVICT_SEG;
        const int rows = max(0, min(min(EVICT_SEG, steps * 64 - j * EVICT_SEG), n - first));
        const int low = max(0, min(rows, budget - first));
        const int kept_low = (b & 0xffff) + max(0, min(eql, need - s));
        const int kept = (a & 0xffff) + max(0, min(eqs, need - s));
        bf[3 * j] = s;
        bf[3 * j + 1] = nhole;
        bf[3 * j + 2] = nmove;
        s += eqs;
        nhole += low - kept_low;
        nmove += kept - kept_low;
      }
    }
    nhole = __builtin_amdgcn_readfirstlane(nhole);
    nmove = __builtin_amdgcn_readfirstlane(nmove);
    __syncthreads();
    const int hole = scan(nhole, red), move = scan(nmove, red2);
    if (lane == 0)
      for (int j = 0; j < p.nsub; ++j) bf[3 * j + 1] += hole, bf[3 * j + 2] += move;
    if (t == 0) {
      int32_t* const h = p.head + 4 * g;
      h[0] = int32_t(uint32_t(uint64_t(old)));
      h[1] = int32_t(old >> 32);
      h[2] = int32_t(prefix);
      h[3] = need;
    }
    if (wave == EVICT_NW - 1 && lane == 0) p.count[g] = hole + nhole;
  }
}

// The free places and moving rows of a segment, and the rows that stay.
__global__ __launch_bounds__(256) void evict_list_kernel(EvictParams p) {
  __shared__ int red[4], red2[4], red3[4];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, g = blockIdx.y, seg = blockIdx.x;
  const int32_t* h = p.head + 4 * g;
  const int64_t old = int64_t((uint64_t(uint32_t(h[1])) << 32) | uint32_t(h[0]));
  const uint32_t least = uint32_t(h[2]);
  const int need = h[3], budget = p.budget;
  const int32_t* bf = p.before + (int64_t(g) * p.nseg + seg) * 3;
  const int j = seg % p.nsub, run = p.steps * 64;
  const int first = (seg / p.nsub) * run + j * EVICT_SEG;
  const int end = min(first + min(EVICT_SEG, run - j * EVICT_SEG), p.n);  // one past the segment's rows
  const float* w = p.w + int64_t(g) * p.whs;
  const int32_t* pos = p.pos + int64_t(g) * p.phs;
  const int row0 = first + wave * 256 + lane;
  float wv[4];
  int32_t pv[4];
  uint32_t key[4];
  int neq = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = row0 + 64 * e;
    wv[e] = r < end ? w[r] : 0.0f;
    pv[e] = r < end ? pos[r] : 0;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool ok = row0 + 64 * e < end;
    key[e] = ok ? evict_key(wv[e], pv[e], old) : 0u;
    neq += __popcll(__builtin_amdgcn_ballot_w64(ok && key[e] == least));
  }
  if (lane == 0) red[wave] = neq;
  __syncthreads();
  int seen = bf[0];
  for (int x = 0; x < wave; ++x) seen += red[x];
  const uint64_t below = (1ull << lane) - 1ull;
  bool keep[4];
  int nhole = 0, nmove = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = row0 + 64 * e;
    const bool ok = r < end, low = r < budget;
    const uint64_t b = __builtin_amdgcn_ballot_w64(ok && key[e] == least);
    keep[e] = ok && (key[e] > least || (key[e] == least && seen + __popcll(b & below) < need));
    seen += __popcll(b);
    nhole += __popcll(__builtin_amdgcn_ballot_w64(ok && low && !keep[e]));
    nmove += __popcll(__builtin_amdgcn_ballot_w64(!low && keep[e]));
  }
  if (lane == 0) red2[wave] = nhole, red3[wave] = nmove;
  __syncthreads();
  int hole = bf[1], move = bf[2];
  for (int x = 0; x < wave; ++x) hole += red2[x], move += red3[x];
  int32_t* const holes = p.hole + int64_t(g) * p.most;
  int32_t* const movers = p.mover + int64_t(g) * p.most;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int r = row0 + 64 * e;
    const bool ok = r < end, low = r < budget;
    const uint64_t bh = __builtin_amdgcn_ballot_w64(ok && low && !keep[e]), bm = __builtin_amdgcn_ballot_w64(!low && keep[e]);
    if (ok && low && !keep[e]) holes[hole + __popcll(bh & below)] = r;
    if (!low && keep[e]) movers[move + __popcll(bm & below)] = r;
    hole += __popcll(bh);
    move += __popcll(bm);
    if (low && keep[e]) {
      p.kept[int64_t(g) * p.khs + r] = r;
      p.w_out[int64_t(g) * p.wos + r] = wv[e];
      p.pos_out[int64_t(g) * p.pos_os + r] = pv[e];
    }
  }
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

template <class C>
static void reorder_launch(const ReorderParams& p, int64_t blocks, hipStream_t stream) {
  const dim3 grid{unsigned(blocks), unsigned(p.nouter), 1};
  if (p.n <= 4)
    reorder_kernel<C, 4><<<grid, 256, 0, stream>>>(p);
  else if (p.n <= 8)
    reorder_kernel<C, 8><<<grid, 256, 0, stream>>>(p);
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
    for (int64_t x : {int64_t(reinterpret_cast<uintptr_t>(r.data)), size > 1 ? r.axis_stride : 0, outer > 1 ? r.outer_stride : 0,
                      r.runs > 1 ? r.run_stride : 0, r.run_bytes})
      while (x % align != 0) align = align == 16 ? 4 : 1;
  }
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
      if (b > INT32_MAX / 2) return fail(W8A8_ENOTSUP, "%s: tensor %lld too large", what, (long long)i0);
      if (blocks + b > INT32_MAX / 2) break;
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

// Steps of 64 rows that each wave of the selection owns, and segments of the lists.
static int evict_steps(int64_t n) { return int((n + 64 * EVICT_NW - 1) / (64 * EVICT_NW)); }
static int evict_segments(int64_t n) {
  return n <= EVICT_FUSED ? 0 : EVICT_NW * ((evict_steps(n) * 64 + EVICT_SEG - 1) / EVICT_SEG);
}

extern "C" int64_t w8a8_evict_workspace_bytes(int64_t KV, int64_t n, int64_t budget) {
  if (KV < 1 || KV > 65535 || n < 1 || n > INT32_MAX / 2 || budget < 1 || budget > n) return -1;
  return KV * (5 + 2 * std::min(budget, n - budget) + 3 * int64_t(evict_segments(n))) * 4;
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
  p.steps = evict_steps(n);
  p.nseg = evict_segments(n);
  p.nsub = p.nseg / EVICT_NW;
  p.count = static_cast<int32_t*>(workspace);
  p.head = p.count + KV;
  p.before = p.head + 4 * KV;
  p.hole = p.before + 3 * KV * p.nseg;
  p.mover = p.hole + KV * p.most;
  p.k = static_cast<char*>(k); p.kh = k_head_stride; p.kr = k_row_stride;
  p.v = static_cast<char*>(v); p.vh = v_head_stride; p.vr = v_row_stride;
  p.row_cols = int(row_bytes / 16);
  if (n <= 1024 * 4)
    evict_select_kernel<4><<<unsigned(KV), 1024, 0, stream>>>(p);
  else if (n <= 1024 * 8)
    evict_select_kernel<8><<<unsigned(KV), 1024, 0, stream>>>(p);
  else if (n <= EVICT_FUSED)
    evict_select_kernel<16><<<unsigned(KV), 1024, 0, stream>>>(p);
  else if (n <= 1024 * 64)
    evict_select_kernel<64><<<unsigned(KV), 1024, 0, stream>>>(p);
  else
    evict_select_kernel<0><<<unsigned(KV), 1024, 0, stream>>>(p);
  if (p.nseg > 0) evict_list_kernel<<<dim3{unsigned(p.nseg), unsigned(KV), 1}, 256, 0, stream>>>(p);
  if (p.most > 0) {
    const int64_t blocks = std::min<int64_t>((int64_t(p.most) * p.row_cols + 255) / 256, 2048);
    evict_move_kernel<<<dim3{unsigned(blocks), unsigned(KV), 1}, 256, 0, stream>>>(p);
  }
  return check_launch(what);
}
