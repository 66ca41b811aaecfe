// paged.cu -- book-keeping and append of the paged KV cache.
//
// paged_plan: one step's block tables, offsets, positions and slots from the
//   request lengths.
// paged_append: QK-Norm + NeoX RoPE of the step's rows, keys and values into
//   their slots.
#include <algorithm>
#include <climits>
#include <cmath>

#include "common.cuh"
#include "launch_state.h"
#include "paged.cuh"

namespace ctts {

namespace {

// ------------------------------------------------------------------- plan
//
// The step is three prefix sums over the requests (pages wanted, pages given
// back, rows) and lists filled from them.  Integers only; a few bytes per row
// and page, so the cost is the launch and the latency of the scan.  Every CTA
// runs the whole scan (at most 4096 requests, 3 words each) and fills its
// share of the lists: no second launch and no wait between CTAs.  Nothing that
// one CTA writes is read by another: the entry of a page given back in this
// step and taken again in it is read from the finished request's table row,
// not from the stack.
constexpr int kPlanThreads = 512;
constexpr int kPlanRowsPerThread = 4;  // rows a thread fills in turn before another CTA is worth its scan

// first index i in [0, n) with a[i + 1] > v; a is non-decreasing, a[0] <= v < a[n]
CTTS_DEV int owner_of(const int* a, int n, int v) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid + 1] > v) hi = mid; else lo = mid + 1;
  }
  return lo;
}

struct PlanReq {
  int held, rows, after;  // pages held, rows wanted, pages after them
  bool done;
};
CTTS_DEV PlanReq plan_req(const ctts_paged_plan& p, int b, int shift) {
  const long long ctx = max(p.ctx_lens[b], 0);
  const int nw = p.new_lens[b];
  const int up = p.page_size - 1;
  PlanReq r;
  r.done = nw < 0;
  r.rows = max(nw, 0);
  r.held = (int)min((ctx + up) >> shift, (long long)p.max_pages);
  // capped one above what fits: the request is refused either way
  r.after = r.rows > 0 ? (int)min((ctx + r.rows + up) >> shift, (long long)p.max_pages + 1) : r.held;
  return r;
}

struct Sum3 {
  long long need, gone, rows;
};
CTTS_DEV Sum3 operator+(const Sum3& a, const Sum3& b) { return {a.need + b.need, a.gone + b.gone, a.rows + b.rows}; }

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const ctts_paged_plan p, int shift) {
  extern __shared__ int plan_smem[];
  const int n = p.batch, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* const need0 = plan_smem;        // [n + 1] exclusive sums; requests from the first refused one on: the total
  int* const gone0 = need0 + n + 1;
  int* const rows0 = gone0 + n + 1;
  __shared__ Sum3 wsum[kPlanThreads / 32];
  __shared__ int refused;
  grid_dep_enter();
  const int count = min(max(*p.free_count, 0), p.free_capacity);
  if (tid == 0) refused = n;

  // a thread sums `per` consecutive requests, the block scans the threads
  const int per = (n + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(n, tid * per), b1 = min(n, b0 + per);
  Sum3 mine = {0, 0, 0};
  for (int b = b0; b < b1; b++) {
    const PlanReq r = plan_req(p, b, shift);
    mine = mine + Sum3{r.done ? 0 : r.after - r.held, r.done ? r.held : 0, r.rows};
  }
  Sum3 inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sum3 y = {__shfl_up_sync(0xffffffffu, inc.need, o), __shfl_up_sync(0xffffffffu, inc.gone, o),
                    __shfl_up_sync(0xffffffffu, inc.rows, o)};
    if (lane >= o) inc = inc + y;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  Sum3 base = {0, 0, 0};
  long long gone_all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; w++) {
    if (w < warp) base = base + wsum[w];
    gone_all += wsum[w].gone;
  }
  const int avail = (int)min(count + gone_all, (long long)p.free_capacity);
  Sum3 at = {base.need + inc.need - mine.need, base.gone + inc.gone - mine.gone, base.rows + inc.rows - mine.rows};
  // the first request that does not fit ends the step
  int first_bad = n;
  for (int b = b0; b < b1; b++) {
    const PlanReq r = plan_req(p, b, shift);
    const Sum3 to = at + Sum3{r.done ? 0 : r.after - r.held, r.done ? r.held : 0, r.rows};
    const bool fits = to.need <= avail && to.rows <= p.max_rows && (r.rows == 0 || r.after <= p.max_pages);
    if (!fits && first_bad == n) first_bad = b;
    // sums behind the first refused request are overwritten below: they may be cut here
    need0[b] = (int)min(at.need, (long long)INT_MAX);
    gone0[b] = (int)min(at.gone, (long long)INT_MAX);
    rows0[b] = (int)min(at.rows, (long long)INT_MAX);
    at = to;
  }
  if (b1 == n && b0 < n) {
    need0[n] = (int)min(at.need, (long long)INT_MAX);
    gone0[n] = (int)min(at.gone, (long long)INT_MAX);
    rows0[n] = (int)min(at.rows, (long long)INT_MAX);
  }
  if (first_bad < n) atomicMin(&refused, first_bad);
  __syncthreads();
  const int granted = refused;
  const int taken = need0[granted], rows_all = rows0[granted], freed = min(gone0[n], p.free_capacity - count);
  __syncthreads();
  for (int b = granted + 1 + tid; b <= n; b += kPlanThreads) {
    need0[b] = taken;
    rows0[b] = rows_all;
  }
  __syncthreads();

  // entry i of the stack after the pages given back are on it
  auto stack = [&](int i) {
    if (i < count) return p.free_pages[i];
    const int b = owner_of(gone0, n, i - count);
    return p.block_tables[(long)b * p.table_ld + (i - count - gone0[b])];
  };
  const int gt = blockIdx.x * kPlanThreads + tid, gn = gridDim.x * kPlanThreads;
  for (int r = gt; r < p.max_rows; r += gn) {
    int pos = -1, slot = -1;
    if (r < rows_all) {
      const int b = owner_of(rows0, n, r);
      pos = max(p.ctx_lens[b], 0) + r - rows0[b];
      const int col = pos >> shift, held = (max(p.ctx_lens[b], 0) + p.page_size - 1) >> shift;
      const int page = col < held ? p.block_tables[(long)b * p.table_ld + col] : stack(avail - 1 - need0[b] - (col - held));
      // a page number that no pool has leaves the row without a slot
      slot = page < 0 || page > (INT_MAX >> shift) - 1 ? -1 : page * p.page_size + (pos & (p.page_size - 1));
    }
    p.positions[r] = pos;
    p.slots[r] = slot;
  }
  for (int t = gt; t < taken; t += gn) {
    const int b = owner_of(need0, n, t);
    const int held = (max(p.ctx_lens[b], 0) + p.page_size - 1) >> shift;
    p.block_tables[(long)b * p.table_ld + held + (t - need0[b])] = stack(avail - 1 - t);
  }
  for (int t = gt; t < freed; t += gn) p.free_pages[count + t] = stack(count + t);
  for (int b = gt; b < n; b += gn) {
    p.seq_lens[b] = p.new_lens[b] < 0 ? 0 : max(p.ctx_lens[b], 0) + (b < granted ? max(p.new_lens[b], 0) : 0);
    p.cu_rows[b] = rows0[b];
  }
  if (gt == 0) {
    p.cu_rows[n] = rows_all;
    p.state[0] = avail - taken;
    p.state[1] = rows_all;
    p.state[2] = granted;
    p.state[3] = taken;
  }
}

// ----------------------------------------------------------------- append
//
// Bound by bandwidth: each element is read once, and written once as a query
// or into the cache.  A lane holds V elements of both halves of a head (the
// RoPE pairs (d, d + hd/2)), L = hd/(2V) lanes hold a head, so the norm is a
// sum over L lanes and the rotation stays in the lane; loads and stores are
// 16 bytes.  The sine and cosine of a row's hd/2 angles are computed once per
// row, for all its heads, after the row's first loads are in flight.
constexpr int kAppThreads = 256;

// Turns per position of each frequency: theta^(-2i/hd) / (2 pi).  In double
// and reduced to a fraction of a turn before rounding: in float32 an angle of
// 10^5 radians is off by 4e-3.
struct AppFreq {
  double turns[64];
};

template <typename T, int V>
struct Vec;
template <>
struct Vec<float, 4> {
  float v[4];
  CTTS_DEV void load(const void* p, long i) {
    const float4 f = ld_stream_f4(static_cast<const float*>(p) + i);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  }
};
template <>
struct Vec<uint16_t, 8> {
  float v[8];
  CTTS_DEV void load(const void* p, long i) {
    const uint4 u = ld_stream_u4(static_cast<const uint16_t*>(p) + i);
    v[0] = bf_lo(u.x); v[1] = bf_hi(u.x); v[2] = bf_lo(u.y); v[3] = bf_hi(u.y);
    v[4] = bf_lo(u.z); v[5] = bf_hi(u.z); v[6] = bf_lo(u.w); v[7] = bf_hi(u.w);
  }
};
CTTS_DEV uint32_t pack2(float lo, float hi) { return (uint32_t)f2bf(lo) | ((uint32_t)f2bf(hi) << 16); }
template <int V>
CTTS_DEV void store(void* p, int bf16, long i, const float* v) {
  if (bf16) {
    uint16_t* q = static_cast<uint16_t*>(p) + i;
    if (V == 8)
      *reinterpret_cast<uint4*>(q) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4 % V], v[5 % V]), pack2(v[6 % V], v[7 % V]));
    else
      *reinterpret_cast<uint2*>(q) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
  } else {
    float* q = static_cast<float*>(p) + i;
#pragma unroll
    for (int j = 0; j < V; j += 4) *reinterpret_cast<float4*>(q + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  }
}

// grid (rows), kAppThreads threads; XT float or uint16_t (bf16 bits)
template <typename XT, int V, int HD>
__global__ void __launch_bounds__(kAppThreads) paged_append_kernel(const ctts_paged_append a, const AppFreq fr, int shift) {
  constexpr int HALF = HD / 2, L = HALF / V, UNITS = kAppThreads / L;
  __shared__ __align__(16) float cs[HALF], sn[HALF];
  grid_dep_enter();
  const int row = blockIdx.x, tid = threadIdx.x;
  const int sub = tid % L, d = sub * V;
  const int nq = a.n_heads, nkv = a.kv.n_kv_heads, heads = nq + 2 * nkv;
  const int slot = a.slots[row];
  if (slot < 0 || slot >= a.kv.n_pages * a.kv.page_size) return;
  const XT* x = static_cast<const XT*>(a.x) + (long)row * a.x_ld;
  Vec<XT, V> lo, hi;
  int h = tid / L;
  if (h < heads) {
    lo.load(x, h * HD + d);
    hi.load(x, h * HD + HALF + d);
  }
  if (tid < HALF) {
    const double t = (double)a.positions[row] * fr.turns[tid];
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    cs[tid] = c;
    sn[tid] = s;
  }
  __syncthreads();
  const long kv_at = (long)(slot >> shift) * a.kv.page_stride + (long)(slot & (a.kv.page_size - 1)) * a.kv.token_stride;
  const bool normed = a.q_norm != nullptr;
  // (every lane of a warp takes the same number of turns: the sums below are warp-wide)
  for (int h0 = 0; h0 < heads; h0 += UNITS, h += UNITS) {
    const bool on = h < heads;
    Vec<XT, V> nlo, nhi;  // the next head, in flight over this one
    if (h + UNITS < heads) {
      nlo.load(x, (h + UNITS) * HD + d);
      nhi.load(x, (h + UNITS) * HD + HALF + d);
    }
    const bool is_q = h < nq, is_v = h >= nq + nkv;
    float ss = 0.0f;
    if (on && !is_v && normed) {
#pragma unroll
      for (int j = 0; j < V; j++) ss = fmaf(lo.v[j], lo.v[j], fmaf(hi.v[j], hi.v[j], ss));
    }
    if (normed) {
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    if (on) {
      if (!is_v) {
        if (normed) {
          const float inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
          const float* g = is_q ? a.q_norm : a.k_norm;
#pragma unroll
          for (int j = 0; j < V; j++) {
            lo.v[j] = lo.v[j] * inv * g[d + j];
            hi.v[j] = hi.v[j] * inv * g[HALF + d + j];
          }
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float x1 = lo.v[j], x2 = hi.v[j], c = cs[d + j], s = sn[d + j];
          lo.v[j] = x1 * c - x2 * s;
          hi.v[j] = x1 * s + x2 * c;
        }
      }
      if (is_q) {
        const long at = (long)row * a.q_ld + h * HD + d;
        store<V>(a.q, a.q_dtype == CTTS_BF16, at, lo.v);
        store<V>(a.q, a.q_dtype == CTTS_BF16, at + HALF, hi.v);
      } else {
        const long at = kv_at + (long)(is_v ? h - nq - nkv : h - nq) * a.kv.head_stride + d;
        store<V>(is_v ? a.kv.v : a.kv.k, a.kv.dtype == CTTS_BF16, at, lo.v);
        store<V>(is_v ? a.kv.v : a.kv.k, a.kv.dtype == CTTS_BF16, at + HALF, hi.v);
      }
    }
    lo = nlo;
    hi = nhi;
  }
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) s++;
  return s;
}

}  // namespace

cudaError_t launch_paged_plan(const ctts_paged_plan& p, cudaStream_t s) {
  static SmemOptIn opt;
  const size_t smem = (size_t)3 * (p.batch + 1) * sizeof(int);
  CTTS_LK(opt.ensure(reinterpret_cast<const void*>(paged_plan_kernel), smem));
  const int per_cta = kPlanThreads * kPlanRowsPerThread;
  const int want = std::max(p.max_rows, p.batch);
  const int grid = std::max(1, std::min(device_sms(), want / per_cta + (want % per_cta != 0)));
  return launch_k(paged_plan_kernel, dim3(grid), dim3(kPlanThreads), smem, s, p, log2_of(p.page_size));
}

cudaError_t launch_paged_append(const ctts_paged_append& a, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  const int hd = a.kv.head_dim, shift = log2_of(a.kv.page_size);
  AppFreq fr;
  // theta^(-2i/hd) by repeated products: i <= 63 of them, each off by 2^-53
  const double step = pow(a.theta, -2.0 / hd);
  double f = 1.0 / (2.0 * 3.14159265358979323846);
  for (int i = 0; i < 64; i++, f *= step) fr.turns[i] = i < hd / 2 ? f : 0.0;
  const dim3 grid(a.rows), block(kAppThreads);
  const bool bf = a.x_dtype == CTTS_BF16;
  if (hd == 64)
    return bf ? launch_k(paged_append_kernel<uint16_t, 8, 64>, grid, block, 0, s, a, fr, shift)
              : launch_k(paged_append_kernel<float, 4, 64>, grid, block, 0, s, a, fr, shift);
  return bf ? launch_k(paged_append_kernel<uint16_t, 8, 128>, grid, block, 0, s, a, fr, shift)
            : launch_k(paged_append_kernel<float, 4, 128>, grid, block, 0, s, a, fr, shift);
}

}  // namespace ctts
