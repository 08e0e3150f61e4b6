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
// evict_select_kernel: one workgroup per KV head finds the budget-th largest key by a radix select (four
// passes over 8-bit digits), then every wave walks its own run of rows with ballots, so that ranks among
// equal keys, free places and moving rows come out in row order.  evict_move_kernel copies the rows.

constexpr int EVICT_NW = 16;

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
  int most;                             // min(budget, n - budget)
  char* k; int64_t kh, kr;              // the cache's bytes: strides of heads and rows
  char* v; int64_t vh, vr;
  int row_cols;                         // 16-byte columns per row
};

// Order of the rows: larger is kept first.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t pos, int64_t newest_old) {
  if (int64_t(pos) > newest_old) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;
  if ((b & 0x7fffffffu) == 0u) return 0x80000000u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// E rows per thread in registers (n <= 1024 E), or with E = 0 read again at each pass.
template <int E>
__global__ __launch_bounds__(1024) void evict_select_kernel(EvictParams p) {
  __shared__ uint32_t hist[256];
  __shared__ int red[EVICT_NW], red2[EVICT_NW];
  __shared__ uint32_t digit_s;
  __shared__ int need_s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, g = blockIdx.x;
  const float* w = p.w + int64_t(g) * p.whs;
  const int32_t* pos = p.pos + int64_t(g) * p.phs;
  const int n = p.n, budget = p.budget;
  // wave w's rows: steps of 64 from w * steps * 64 on
  const int steps = (n + 64 * EVICT_NW - 1) / (64 * EVICT_NW);
  const int row0 = wave * steps * 64 + lane;

  int newest = INT32_MIN;
  for (int r = t; r < n; r += 1024) newest = max(newest, pos[r]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) newest = max(newest, __shfl_xor(newest, o, 64));
  if (lane == 0) red[wave] = newest;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < EVICT_NW; ++x) newest = max(newest, red[x]);
  const int64_t old = int64_t(newest) - p.recent;

  uint32_t key[E > 0 ? E : 1];
  if constexpr (E > 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int r = row0 + 64 * e;
      key[e] = e < steps && r < n ? evict_key(w[r], pos[r], old) : 0u;
    }
  }
  // f(key, row, valid) for each of this thread's rows, in order; the whole wave takes part in each step
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (E > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < steps) f(key[e], row0 + 64 * e, row0 + 64 * e < n);
    } else {
      for (int e = 0; e < steps; ++e) {
        const int r = row0 + 64 * e;
        f(r < n ? evict_key(w[r], pos[r], old) : 0u, r, r < n);
      }
    }
  };

  // the budget-th largest key: its digits from the top, and how many of the rows with that key are kept
  uint32_t prefix = 0;
  int need = budget;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) hist[t] = 0u;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    each([&](uint32_t k, int, bool ok) {
      if (ok && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
    });
    __syncthreads();
    if (wave == 0) {
      // lane l holds digits 4 l .. 4 l + 3; rows of larger digits come first
      int c[4], sum = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) c[x] = int(hist[4 * lane + x]), sum += c[x];
      int above = sum;  // rows of this lane's and later lanes' digits
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_down(above, o, 64);
        if (lane + o < 64) above += v;
      }
      above -= sum;
#pragma unroll
      for (int x = 3; x >= 0; --x) {
        if (above < need && above + c[x] >= need) digit_s = uint32_t(4 * lane + x), need_s = need - above;
        above += c[x];
      }
    }
    __syncthreads();
    prefix |= digit_s << shift;
    need = need_s;
    __syncthreads();
  }

  // exclusive sum over the waves of a per-wave count
  auto scan = [&](int v, int* buf) __attribute__((always_inline)) {
    if (lane == 0) buf[wave] = v;
    __syncthreads();
    int s = 0;
    for (int x = 0; x < wave; ++x) s += buf[x];
    return s;
  };
  int neq = 0;
  each([&](uint32_t k, int, bool ok) { neq += __popcll(__builtin_amdgcn_ballot_w64(ok && k == prefix)); });
  int eq = scan(neq, red2);
  const uint64_t below = (1ull << lane) - 1ull;
  // kept(key): for each of the wave's rows in order
  auto kept = [&](uint32_t k, bool ok, int& seen) __attribute__((always_inline)) {
    const uint64_t b = __builtin_amdgcn_ballot_w64(ok && k == prefix);
    const int rank = seen + __popcll(b & below);
    seen += __popcll(b);
    return ok && (k > prefix || (k == prefix && rank < need));
  };
  int nhole = 0, nmove = 0, seen = eq;
  each([&](uint32_t k, int r, bool ok) {
    const bool keep = kept(k, ok, seen);
    nhole += __popcll(__builtin_amdgcn_ballot_w64(ok && r < budget && !keep));
    nmove += __popcll(__builtin_amdgcn_ballot_w64(ok && r >= budget && keep));
  });
  __syncthreads();
  int hole = scan(nhole, red), move = scan(nmove, red2);
  int32_t* const holes = p.hole + int64_t(g) * p.most;
  int32_t* const movers = p.mover + int64_t(g) * p.most;
  int32_t* const ko = p.kept + int64_t(g) * p.khs;
  float* const wo = p.w_out + int64_t(g) * p.wos;
  int32_t* const po = p.pos_out + int64_t(g) * p.pos_os;
  seen = eq;
  each([&](uint32_t k, int r, bool ok) {
    const bool keep = kept(k, ok, seen);
    const bool is_hole = ok && r < budget && !keep, is_move = ok && r >= budget && keep;
    const uint64_t bh = __builtin_amdgcn_ballot_w64(is_hole), bm = __builtin_amdgcn_ballot_w64(is_move);
    if (is_hole) holes[hole + __popcll(bh & below)] = r;
    if (is_move) movers[move + __popcll(bm & below)] = r;
    hole += __popcll(bh);
    move += __popcll(bm);
    if (r < budget && keep) ko[r] = r, wo[r] = w[r], po[r] = pos[r];
  });
  if (wave == EVICT_NW - 1 && lane == 0) p.count[g] = hole, need_s = hole;
  __threadfence_block();
  __syncthreads();
  for (int i = t; i < need_s; i += 1024) {
    const int dst = holes[i], src = movers[i];
    ko[dst] = src;
    wo[dst] = w[src];
    po[dst] = pos[src];
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
    const int64_t c = (x % p.row_cols) * 16;
    const int64_t dst = holes[m], src = movers[m];
    const v4u a = *reinterpret_cast<const v4u*>(k + src * p.kr + c);
    const v4u b = *reinterpret_cast<const v4u*>(v + src * p.vr + c);
    *reinterpret_cast<v4u*>(k + dst * p.kr + c) = a;
    *reinterpret_cast<v4u*>(v + dst * p.vr + c) = b;
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

extern "C" int64_t w8a8_evict_workspace_bytes(int64_t KV, int64_t n, int64_t budget) {
  if (KV < 1 || KV > 65535 || n < 1 || n > INT32_MAX / 2 || budget < 1 || budget > n) return -1;
  return KV * (2 * std::min(budget, n - budget) + 1) * 4;
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
  p.count = static_cast<int32_t*>(workspace);
  p.hole = p.count + KV;
  p.mover = p.hole + KV * p.most;
  p.k = static_cast<char*>(k); p.kh = k_head_stride; p.kr = k_row_stride;
  p.v = static_cast<char*>(v); p.vh = v_head_stride; p.vr = v_row_stride;
  p.row_cols = int(row_bytes / 16);
  if (n <= 1024 * 4)
    evict_select_kernel<4><<<unsigned(KV), 1024, 0, stream>>>(p);
  else if (n <= 1024 * 16)
    evict_select_kernel<16><<<unsigned(KV), 1024, 0, stream>>>(p);
  else
    evict_select_kernel<0><<<unsigned(KV), 1024, 0, stream>>>(p);
  if (p.most > 0) {
    const int64_t blocks = std::min<int64_t>((int64_t(p.most) * p.row_cols + 255) / 256, 2048);
    evict_move_kernel<<<dim3{unsigned(blocks), unsigned(KV), 1}, 256, 0, stream>>>(p);
  }
  return check_launch(what);
}
