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
// share of the lists, a row a thread: no second launch and no wait between
// CTAs.  64 requests of one row each: 4.0 us; 1500 requests, 44 thousand
// rows: 7.7 us (four rows a thread: 11.3).  Nothing that
// one CTA writes is read by another: the entry of a page given back in this
// step and taken again in it is read from the finished request's table row,
// not from the stack.
constexpr int kPlanThreads = 512;

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
// 16 bytes.  A warp takes a row: it passes over 32/L heads at a time with the
// same dims in a lane, so a lane computes its V angles once for all of them
// (after the first heads' loads are in flight), and nothing is shared or
// waited for between warps.  Few rows (a decode step): several warps a row.
// 16381 rows, 16 + 2 x 8 heads of 128, bf16: 55 us, 4.9 TB/s (one row a block
// and its angles through shared memory: 89 us; four passes in flight at fewer
// warps: 58 us, eight: 64 us; slots a page after the other, as plan gives
// them, instead of scattered ones: 54.9 us).  4001 rows, 12 + 2 x 4 heads of 64, float32:
// 9.5 us, 4.3 TB/s.
constexpr int kAppWarps = 4;   // a block
constexpr int kAppAhead = 2;   // loads in flight: passes of a warp

// Turns per position of each frequency: theta^(-2i/hd) / (2 pi).  In double
// and reduced to a fraction of a turn before rounding: in float32 an angle of
// 10^5 radians is off by 4e-3.
struct AppFreq {
  double turns[64];
};

CTTS_DEV uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
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
// 16 bytes: four float32 or eight bf16
template <int V>
CTTS_DEV void widen(const uint4& u, float* v) {
  if (V == 4) {
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
  } else {
    v[0] = bf_lo(u.x); v[1] = bf_hi(u.x); v[2] = bf_lo(u.y); v[3] = bf_hi(u.y);
    v[4 % V] = bf_lo(u.z); v[5 % V] = bf_hi(u.z); v[6 % V] = bf_lo(u.w); v[7 % V] = bf_hi(u.w);
  }
}

// `parts` warps a row; V = 4 (float32 x) or 8 (bf16)
template <int V, int HD>
__global__ void __launch_bounds__(kAppWarps * 32, V == 8 ? 7 : 8) paged_append_kernel(const ctts_paged_append a, const __grid_constant__ AppFreq fr, int shift,
                                                                      int parts) {
  constexpr int HALF = HD / 2, L = HALF / V, AT_ONCE = 32 / L, ES = 16 / V;
  grid_dep_enter();
  const int lane = threadIdx.x & 31, w = blockIdx.x * kAppWarps + (threadIdx.x >> 5);
  const int row = w / parts, part = w - row * parts;
  if (row >= a.rows) return;
  const int nq = a.n_heads, nkv = a.kv.n_kv_heads, heads = nq + 2 * nkv;
  const int d = (lane % L) * V;
  const uint8_t* x = static_cast<const uint8_t*>(a.x) + ((long)row * a.x_ld + d) * ES;
  const int slot = a.slots[row], pos = a.positions[row];
  const bool normed = a.q_norm != nullptr;
  const int step = parts * AT_ONCE;
  float cs[V], sn[V];
  bool ready = false;
  // (every lane of a warp makes the same passes: the sums are warp-wide)
  for (int h0 = part * AT_ONCE; h0 < heads; h0 += kAppAhead * step) {
    uint4 lo[kAppAhead], hi[kAppAhead];
#pragma unroll
    for (int i = 0; i < kAppAhead; i++) {
      const int h = h0 + i * step + lane / L;
      if (h < heads) {
        lo[i] = ld_stream_u4(x + (long)h * HD * ES);
        hi[i] = ld_stream_u4(x + (long)h * HD * ES + HALF * ES);
      }
    }
    if (!ready) {
      ready = true;
      if (slot < 0 || slot >= a.kv.n_pages * a.kv.page_size) return;
#pragma unroll
      for (int j = 0; j < V; j++) {
        const double t = (double)pos * fr.turns[d + j];
        sincospif(2.0f * (float)(t - rint(t)), &sn[j], &cs[j]);
      }
    }
    const long kv_at = (long)(slot >> shift) * a.kv.page_stride + (long)(slot & (a.kv.page_size - 1)) * a.kv.token_stride + d;
#pragma unroll
    for (int i = 0; i < kAppAhead; i++) {
      const int h = h0 + i * step + lane / L;
      if (h0 + i * step >= heads) break;
      const bool on = h < heads, is_q = h < nq, is_v = h >= nq + nkv;
      float u[V], v[V];
      widen<V>(lo[i], u);
      widen<V>(hi[i], v);
      if (normed) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < V; j++) ss = fmaf(u[j], u[j], fmaf(v[j], v[j], ss));
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (!is_v) {
          const float inv = 1.0f / sqrtf(ss / (float)HD + a.eps);
          const float* g = (is_q ? a.q_norm : a.k_norm) + d;  // (512 bytes that stay in L1)
#pragma unroll
          for (int j = 0; j < V; j += 4) {
            const float4 p = *reinterpret_cast<const float4*>(g + j), q = *reinterpret_cast<const float4*>(g + HALF + j);
            u[j] *= inv * p.x; u[j + 1] *= inv * p.y; u[j + 2] *= inv * p.z; u[j + 3] *= inv * p.w;
            v[j] *= inv * q.x; v[j + 1] *= inv * q.y; v[j + 2] *= inv * q.z; v[j + 3] *= inv * q.w;
          }
        }
      }
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float x1 = u[j], x2 = v[j];
          u[j] = x1 * cs[j] - x2 * sn[j];
          v[j] = x1 * sn[j] + x2 * cs[j];
        }
      }
      if (on) {
        void* to = is_q ? a.q : (is_v ? a.kv.v : a.kv.k);
        const int bf16 = (is_q ? a.q_dtype : a.kv.dtype) == CTTS_BF16;
        const long at = is_q ? (long)row * a.q_ld + h * HD + d : kv_at + (long)(is_v ? h - nq - nkv : h - nq) * a.kv.head_stride;
        store<V>(to, bf16, at, u);
        store<V>(to, bf16, at + HALF, v);
      }
    }
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
  const int want = std::max(p.max_rows, p.batch);
  const int grid = std::max(1, std::min(device_sms(), want / kPlanThreads + (want % kPlanThreads != 0)));
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
  const bool bf = a.x_dtype == CTTS_BF16;
  // warps a row: enough for about 48 warps an SM, up to a pass each
  const int passes = (a.n_heads + 2 * a.kv.n_kv_heads) * hd / (bf ? 512 : 256);
  int parts = 1;
  while (parts * 2 <= passes && (long)a.rows * parts < 48L * device_sms()) parts *= 2;
  const dim3 grid((unsigned)(((long)a.rows * parts + kAppWarps - 1) / kAppWarps)), block(kAppWarps * 32);
  if (hd == 64)
    return bf ? launch_k(paged_append_kernel<8, 64>, grid, block, 0, s, a, fr, shift, parts)
              : launch_k(paged_append_kernel<4, 64>, grid, block, 0, s, a, fr, shift, parts);
  return bf ? launch_k(paged_append_kernel<8, 128>, grid, block, 0, s, a, fr, shift, parts)
            : launch_k(paged_append_kernel<4, 128>, grid, block, 0, s, a, fr, shift, parts);
}

}  // namespace ctts
