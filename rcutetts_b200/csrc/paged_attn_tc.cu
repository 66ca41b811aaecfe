// paged_attn_tc.cu -- attention of chunks of new rows over a bf16 paged cache
// on the 5th-generation tensor cores (tcgen05).
//
// An item is up to two sub-tiles of 128 packed rows (one row per TMEM lane)
// of one request and KV head.  Per key tile and sub-tile:
//   S = Q . K^T   both operands in shared memory (K-major, 128-byte swizzle),
//   softmax       one thread per row: S read from TMEM, the weights written
//                 back over it in bf16,
//   O += P . V    P read from TMEM, V from shared memory as it lies in the
//                 pages ([key][dim]: the MN-major form of the B operand).
// Warps 0-3 and 4-7 run the softmax of the two sub-tiles, so one computes
// exponentials while the tensor core multiplies for the other; warp 8 issues
// the MMAs, warp 9 the TMA copies: one box per page and 64 dims (a 4D map over
// the pool), K and V in rings of their own.  Missing pages are boxes
// outside the map, which arrive as zeros.
//
// The output is rescaled only when a row's maximum has grown by more than
// 2^8 since the last time: weights up to 256 lose nothing in floating point,
// and the pass over O in TMEM becomes rare.  S(j+1) of a sub-tile is issued
// behind P.V(j), so O is at rest while its softmax threads hold S.
//
// float32 queries: queries and weights enter as three bf16 terms (24 bits),
// key tiles are 64 wide so that three terms of the weights fit over S.  Each
// P.V starts at zero and its threads add it to an output row in registers:
// the tensor core cuts the sums it accumulates instead of rounding them, which
// over a thousand keys costs 2^-18 of the output (measured against 64 bits).
//
// Every wait is bounded; one that gives up raises a flag that ends all roles.
#include <algorithm>

#include "common.cuh"
#include "launch_state.h"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "tc_ptx.cuh"

namespace ctts {

namespace {

// Warps: 4 of softmax per sub-tile, then one that issues MMAs and one that
// issues copies (the block is rounded up to whole warpgroups).  Two softmax
// warpgroups take registers from the third: 2 x 216 + 72 = 3 x 168.
template <bool QF, int HD>
struct TcShape {
  static constexpr int THREADS = QF && HD == 128 ? 256 : 384;
  static constexpr bool REGS = THREADS == 384;
  static constexpr int LAUNCH_REGS = 168, SOFTMAX_REGS = 216, OTHER_REGS = 72;
  static constexpr int KT = QF ? 64 : 128;                // keys per tile
  static constexpr int NSUB = QF && HD == 128 ? 1 : 2;    // three terms of 256 wide queries would not fit
  static constexpr int R = 128 * NSUB;                    // packed rows per item
  static constexpr int NT = QF ? 3 : 1;                   // terms of queries and weights
  static constexpr int NC = HD / 64;                      // 128-byte column blocks
  static constexpr uint32_t QTERM = NC * 128 * 128;       // bytes of one term of one sub-tile
  static constexpr uint32_t TILE = NC * KT * 128;         // bytes of a K or V tile
  static constexpr int NS = QF ? (HD == 64 ? 6 : 3) : (HD == 64 ? 4 : 2);
  static constexpr size_t SMEM = (size_t)NSUB * NT * QTERM + (size_t)2 * NS * TILE + 1024;
};

// Shared-memory descriptor of a 128-byte swizzled operand.  K-major: lbo
// unused (1).  MN-major: rows of 64 dims per key, `lbo` bytes between blocks
// of 64 dims, 1024 bytes between groups of 8 keys.
CTTS_DEV uint64_t tc_desc(uint32_t saddr, uint32_t lbo) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)(lbo >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
// D f32, A and B bf16, M = 128, N = n; B K-major or MN-major
CTTS_DEV constexpr uint32_t tc_idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
CTTS_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {  // A from TMEM
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
CTTS_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
CTTS_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
CTTS_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// uses of r[0..31] stay behind this point
CTTS_DEV void pin32(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; i += 16)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]),
                 "+r"(r[i + 7]), "+r"(r[i + 8]), "+r"(r[i + 9]), "+r"(r[i + 10]), "+r"(r[i + 11]), "+r"(r[i + 12]), "+r"(r[i + 13]),
                 "+r"(r[i + 14]), "+r"(r[i + 15]));
}
CTTS_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
CTTS_DEV void tmem_st32(uint32_t taddr, const uint32_t* r) {
  tmem_st16(taddr, r);
  tmem_st16(taddr + 16, r + 16);
}

struct TcBars {
  uint64_t k_full[6], k_empty[6], v_full[6], v_empty[6];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2], drain;
};

template <bool QF, int HD>
__global__ void __launch_bounds__(TcShape<QF, HD>::THREADS, 1) paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                      const __grid_constant__ CUtensorMap tmV, const PagedAttnArgs a,
                                                                      int box, int order) {
  using S = TcShape<QF, HD>;
  constexpr int KT = S::KT, R = S::R, NS = S::NS, NT = S::NT, NC = S::NC;
  constexpr int W_MMA = 4 * S::NSUB, W_TMA = W_MMA + 1;
  extern __shared__ uint8_t tc_smem[];
  __shared__ AttnStart start;
  __shared__ __align__(8) TcBars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int gave_up;
  const uint32_t sbase = (smem_u32(tc_smem) + 1023u) & ~1023u;
  const uint32_t qs = sbase, ks = qs + S::NSUB * NT * S::QTERM, vs = ks + NS * S::TILE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(&bars.k_full[i], 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], 1);
      mbar_init(&bars.v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&bars.q_full[i], 128);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.o_full[i], 1);
    }
    mbar_init(&bars.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    gave_up = 0;
  }
  if (warp == W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  grid_dep_enter();
  attn_find_start<R, KT, S::THREADS>(a, &start);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;  // S and P of sub-tile s at column 128 s, O at 256 + 128 s
  const long units = start.units;
  if (tid == 0) a.parts[blockIdx.x].pieces = 0;  // no divided item yet
  __syncthreads();

  if (warp >= W_MMA) {
    if (S::REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::OTHER_REGS));
    if (units > 0 && warp == W_TMA) {
      // ---- producer: lane i copies page box i of each tile
      AttnCursor cu = AttnCursor::at<R, KT>(a, start);
      const int nbox = KT / box;
      long u = 0;
      for (; u < units; u++) {
        const int st = (int)(u % NS);
        const uint32_t par = (uint32_t)((u / NS) & 1);
        const int kk = cu.kt * KT + lane * box;
        int page = -1;
        if (lane < nbox && kk < cu.len) page = a.p.block_tables[(long)cu.b * a.p.table_ld + (kk >> a.shift)];
        if ((unsigned)page >= (unsigned)a.p.kv.n_pages) page = a.p.kv.n_pages;  // outside the map: zeros
        const int slot = kk & (a.p.kv.page_size - 1);
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
          uint64_t* full = kv ? &bars.v_full[st] : &bars.k_full[st];
          if (u >= NS && !mbar_wait(kv ? &bars.v_empty[st] : &bars.k_empty[st], par ^ 1)) gave_up = 1;
          if (__any_sync(0xffffffffu, gave_up)) goto produced;
          if (lane == 0) mbar_expect_tx(full, S::TILE);
          __syncwarp();
          if (lane < nbox) {
            const uint32_t dst = (kv ? vs : ks) + st * S::TILE + (uint32_t)(lane * box) * 128u;
#pragma unroll
            for (int c = 0; c < NC; c++) copy_box(dst + c * KT * 128, kv ? &tmV : &tmK, order, c * 64, slot, cu.h, page, full);
          }
        }
        if (u + 1 < units) cu.next<R, KT>(a);
      }
    produced:
      __syncwarp();
      if (gave_up)  // copies in flight land before the block may leave
        for (long w = u > NS ? u - NS : 0; w <= u && w < units; w++) {
          mbar_wait(&bars.k_full[w % NS], (uint32_t)((w / NS) & 1));
          mbar_wait(&bars.v_full[w % NS], (uint32_t)((w / NS) & 1));
        }
    } else if (units > 0 && warp == W_MMA) {
      // ---- MMA issue (one thread)
      if (lane == 0) {
        AttnCursor cu = AttnCursor::at<R, KT>(a, start);
        uint32_t q_par = 0, p_par = 0;  // one bit per sub-tile
        auto wait = [&](uint64_t* bar, uint32_t par) {
          if (gave_up || !mbar_wait(bar, par)) gave_up = 1;
          fence_after();
          return !gave_up;
        };
        auto scores = [&](int s, int st) {
          // (opaque: the descriptors are made as they are used, not kept in
          // registers over the loop)
          uint32_t kb = ks + st * S::TILE, qb = qs + s * NT * S::QTERM, acc = 0;
          asm volatile("" : "+r"(kb), "+r"(qb));
          // small terms first: the tensor core cuts what it adds to the
          // accumulator's precision
#pragma unroll
          for (int t = NT - 1; t >= 0; t--)
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
              for (int k = 0; k < 4; k++) {
                umma_bf16(tmem + 128 * s, tc_desc(qb + t * S::QTERM + c * 16384 + k * 32, 16),
                          tc_desc(kb + c * KT * 128 + k * 32, 16), tc_idesc(KT, false), acc);
                acc = 1;
              }
          umma_commit(&bars.s_full[s]);
        };
        auto values = [&](int s, int st, uint32_t acc) {
          uint32_t vb = vs + st * S::TILE;
          asm volatile("" : "+r"(vb));
#pragma unroll
          for (int t = NT - 1; t >= 0; t--)
#pragma unroll
            for (int k = 0; k < KT / 16; k++) {
              mma_ts(tmem + 256 + 128 * s, tmem + 128 * s + t * (KT / 2) + k * 8, tc_desc(vb + k * 2048, KT * 128), tc_idesc(HD, true), acc);
              acc = 1;
            }
        };
        bool fresh = true, ok = true;
        int nsub = 1;
        for (long u = 0; u < units && ok; u++) {
          const int st = (int)(u % NS);
          if (fresh) {  // a piece begins: its first scores
            nsub = min(R, cu.nn * a.group - cu.m * R) > 128 ? 2 : 1;
            ok = wait(&bars.k_full[st], (uint32_t)((u / NS) & 1));
            for (int s = 0; s < nsub && ok; s++) {
              ok = wait(&bars.q_full[s], (q_par >> s) & 1);
              q_par ^= 1u << s;
              if (ok) scores(s, st);
            }
            if (!ok) break;
            umma_commit(&bars.k_empty[st]);
          }
          const bool last = cu.kt + 1 == cu.nt || u + 1 == units;
          ok = wait(&bars.v_full[st], (uint32_t)((u / NS) & 1));
          const int sn = (int)((u + 1) % NS);
          if (ok && !last) ok = wait(&bars.k_full[sn], (uint32_t)(((u + 1) / NS) & 1));
          for (int s = 0; s < nsub && ok; s++) {
            ok = wait(&bars.p_full[s], (p_par >> s) & 1);
            p_par ^= 1u << s;
            if (!ok) break;
            values(s, st, fresh || QF ? 0u : 1u);
            if (last)
              umma_commit(&bars.o_full[s]);
            else
              scores(s, sn);
          }
          if (!ok) break;
          umma_commit(&bars.v_empty[st]);
          if (!last) umma_commit(&bars.k_empty[sn]);
          fresh = last;
          if (u + 1 < units) cu.next<R, KT>(a);
        }
        if (!ok) {  // MMAs in flight end before TMEM is given back
          umma_commit(&bars.drain);
          mbar_wait(&bars.drain, 0);
        }
      }
      __syncwarp();
    }
  } else {
    if (S::REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::SOFTMAX_REGS));
    if (units > 0) {
      // ---- softmax: one thread per packed row
      const int s = warp >> 2, row = (warp & 3) * 32 + lane;
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t tS = tmem + 128 * s + lane_base, tO = tmem + 256 + 128 * s + lane_base;
      const float c2 = a.c2_hi;
      AttnCursor cu = AttnCursor::at<R, KT>(a, start);
      uint32_t s_par = 0, o_par = 0;
      bool fresh = true, ok = true;
      int kt0 = 0, nrows = 0, pk = 0, pos = 0, pos_lo = 0;
      bool mine = false, warp_on = false, on = false;
      float m = -INFINITY, l = 0.0f;
      float o_row[QF ? HD : 1];  // float32 calls: the output row so far
      // adds the product of the last tile to it
      auto gather = [&]() {
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld32_nowait(tO + c, o);
          tmem_wait();
          pin32(o);
#pragma unroll
          for (int j = 0; j < 32; j++) o_row[QF ? c + j : 0] += __uint_as_float(o[j]);
        }
      };
      for (long u = 0; u < units && ok; u++) {
        if (fresh) {
          fresh = false;
          kt0 = cu.kt;
          nrows = min(R, cu.nn * a.group - cu.m * R);
          on = s * 128 < nrows;  // the sub-tile has rows
          mine = s * 128 + row < nrows;
          warp_on = s * 128 + (warp & 3) * 32 < nrows;
          pk = cu.m * R + s * 128 + row;
          pos = cu.len - cu.cnt + pk / a.group;
          pos_lo = cu.len - cu.cnt + (pk - lane) / a.group;
          m = -INFINITY;
          l = 0.0f;
#pragma unroll
          for (int c = 0; c < (QF ? HD : 1); c++) o_row[c] = 0.0f;
          if (on) {
            // the warp's 32 queries as bf16 terms: eight lanes read 128 bytes
            // of a row (as bf16), four rows at a time, all loads in flight
            // before the first is used; rows behind the item are zero
            const int r0 = (warp & 3) * 32, p0 = cu.m * R + s * 128 + r0;
#pragma unroll
            for (int c = 0; c < NC; c++) {
              constexpr int RP = 8;  // rows a lane reads: 4 i + lane / 8
              uint4 x[RP], y[QF ? RP : 1];
#pragma unroll
              for (int i = 0; i < RP; i++) {
                const int r = 4 * i + (lane >> 3), p = p0 + r;
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (QF) y[QF ? i : 0] = x[i];
                if (s * 128 + r0 + r < nrows) {
                  const int tok = p / a.group;
                  const long at = (long)(cu.r0 + tok) * a.p.q_ld + (cu.h * a.group + p - tok * a.group) * HD + c * 64 + (lane & 7) * 8;
                  if (QF) {
                    x[i] = *reinterpret_cast<const uint4*>(static_cast<const float*>(a.p.q) + at);
                    y[QF ? i : 0] = *reinterpret_cast<const uint4*>(static_cast<const float*>(a.p.q) + at + 4);
                  } else {
                    x[i] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.p.q) + at);
                  }
                }
              }
#pragma unroll
              for (int i = 0; i < RP; i++) {
                const int r = r0 + 4 * i + (lane >> 3);
                uint32_t t[4][NT];
                if (QF) {
                  const uint4 z = y[QF ? i : 0];
                  split_bf2<NT>(__uint_as_float(x[i].x), __uint_as_float(x[i].y), t[0]);
                  split_bf2<NT>(__uint_as_float(x[i].z), __uint_as_float(x[i].w), t[1]);
                  split_bf2<NT>(__uint_as_float(z.x), __uint_as_float(z.y), t[2]);
                  split_bf2<NT>(__uint_as_float(z.z), __uint_as_float(z.w), t[3]);
                } else {
                  t[0][0] = x[i].x; t[1][0] = x[i].y; t[2][0] = x[i].z; t[3][0] = x[i].w;
                }
                const uint32_t dst = qs + s * NT * S::QTERM + c * 16384 + r * 128 + (uint32_t)(((lane ^ r) & 7) << 4);
#pragma unroll
                for (int k = 0; k < NT; k++)
                  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + k * S::QTERM), "r"(t[0][k]), "r"(t[1][k]), "r"(t[2][k]),
                               "r"(t[3][k])
                               : "memory");
              }
            }
            fence_async();
            mbar_arrive(&bars.q_full[s]);
          }
        }
        const bool ends = cu.kt + 1 == cu.nt, last = ends || u + 1 == units;
        if (on) {
          const int key0 = cu.kt * KT;
          // 8-key groups whose page does not exist
          uint32_t dead = 0;
          {
            const int kk = key0 + lane * 8;
            bool d = false;
            if (lane < KT / 8 && kk < cu.len)
              d = (unsigned)a.p.block_tables[(long)cu.b * a.p.table_ld + (kk >> a.shift)] >= (unsigned)a.p.kv.n_pages;
            dead = __ballot_sync(0xffffffffu, d);
          }
          if (s == 0 && key0 + KT > cu.len) {
            // slots behind the length may hold anything, and 0 * NaN is NaN:
            // their values become zeros (both sub-tiles' products come after
            // this sub-tile's arrival at p_full)
            const int st = (int)(u % NS);
            if (!mbar_wait(&bars.v_full[st], (uint32_t)((u / NS) & 1))) gave_up = 1;
            if (row < KT && key0 + row >= cu.len) {
#pragma unroll
              for (int c = 0; c < NC * 8; c++)
                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vs + st * S::TILE + (c >> 3) * KT * 128 + row * 128 + (c & 7) * 16), "r"(0)
                             : "memory");
            }
            fence_async();
          }
          if (!mbar_wait(&bars.s_full[s], s_par)) gave_up = 1;
          s_par ^= 1;
          if (__any_sync(0xffffffffu, gave_up)) {
            ok = false;
            break;
          }
          if (warp_on) {
            fence_after();
            uint32_t x[KT];
#pragma unroll
            for (int c = 0; c < KT; c += 32) tmem_ld32_nowait(tS + c, x + c);
            tmem_wait();
#pragma unroll
            for (int c = 0; c < KT; c += 32) pin32(x + c);
            if (key0 + KT - 1 > pos_lo || dead) {
              const int lim = pos - key0;
#pragma unroll
              for (int c = 0; c < KT; c++)
                if (c > lim || ((dead >> (c >> 3)) & 1)) x[c] = 0xff800000u;  // -inf
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < KT; c += 4)
#pragma unroll
              for (int j = 0; j < 4; j++) mx[j] = fmaxf(mx[j], __uint_as_float(x[c + j]));
            const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c2;
            if (QF) {
              if (cu.kt > kt0) gather();
              const float mm = fmaxf(m, mn), f = mm == -INFINITY ? 0.0f : exp2_fast(m - mm);
              m = mm;
              l *= f;
#pragma unroll
              for (int c = 0; c < (QF ? HD : 1); c++) o_row[c] *= f;
            } else if (cu.kt == kt0) {
              m = mn;  // O is overwritten by the first product
            } else {
              const bool grow = mn > m + 8.0f;
              if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? exp2_fast(m - mn) : 1.0f;
                if (grow) m = mn;
                l *= f;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                  uint32_t o[32];
                  tmem_ld32_nowait(tO + c, o);
                  tmem_wait();
                  pin32(o);
#pragma unroll
                  for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                  tmem_st32(tO + c, o);
                }
                tmem_st_wait();
              }
            }
            const float mz = m == -INFINITY ? 0.0f : m;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KT; c += 32) {
              uint32_t p[NT][16];
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                const float e0 = exp2_fast(attn_arg<QF>(a, __uint_as_float(x[c + j]), mz));
                const float e1 = exp2_fast(attn_arg<QF>(a, __uint_as_float(x[c + j + 1]), mz));
                sum[j & 2] += e0;
                sum[(j & 2) + 1] += e1;
                uint32_t t[NT];
                split_bf2<NT>(e0, e1, t);
#pragma unroll
                for (int k = 0; k < NT; k++) p[k][j >> 1] = t[k];
              }
#pragma unroll
              for (int k = 0; k < NT; k++) tmem_st16(tS + k * (KT / 2) + (c >> 1), p[k]);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st_wait();
            fence_before();
          }
          mbar_arrive(&bars.p_full[s]);

          if (last) {
            const bool whole = ends && kt0 == 0;
            const int slot = 2 * blockIdx.x + (kt0 == 0 ? 1 : 0);
            if (!ends && kt0 == 0 && s == 0 && row == 0) {
              AttnPart d;
              d.pieces = attn_pieces(a, start, cu.nt - 1 - cu.kt);
              d.row0 = cu.r0; d.packed0 = cu.m * R; d.rows = nrows; d.h = cu.h;
              a.parts[blockIdx.x] = d;
            }
            if (!mbar_wait(&bars.o_full[s], o_par)) gave_up = 1;
            o_par ^= 1;
            if (__any_sync(0xffffffffu, gave_up)) {
              ok = false;
              break;
            }
            if (warp_on) {
              fence_after();
              const float inv = !whole ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
              const long at = (long)(cu.r0 + pk / a.group) * a.p.out_ld + (long)(cu.h * a.group + pk % a.group) * HD;
              const long pr = (long)slot * a.tile_rows + s * 128 + row;
              if (!whole && mine) a.ml[pr] = make_float2(m, l);
              if (QF) gather();
#pragma unroll
              for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (QF) {
#pragma unroll
                  for (int j = 0; j < 32; j++) o[j] = __float_as_uint(o_row[QF ? c + j : 0]);
                } else {
                  tmem_ld32_nowait(tO + c, o);
                  tmem_wait();
                  pin32(o);
                }
                if (mine) {
                  float v[32];
#pragma unroll
                  for (int j = 0; j < 32; j++) v[j] = l == 0.0f ? 0.0f : __uint_as_float(o[j]) * inv;
                  if (whole && !QF) {
                    uint16_t* w = static_cast<uint16_t*>(a.p.out) + at + c;
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                      *reinterpret_cast<uint4*>(w + j) = make_uint4(pack_bf2(v[j], v[j + 1]), pack_bf2(v[j + 2], v[j + 3]),
                                                                    pack_bf2(v[j + 4], v[j + 5]), pack_bf2(v[j + 6], v[j + 7]));
                  } else {
                    float* w = whole ? static_cast<float*>(a.p.out) + at + c : a.acc + pr * HD + c;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(w + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                  }
                }
              }
              fence_before();
            }
          }
        }
        if (last) fresh = true;
        if (u + 1 < units) cu.next<R, KT>(a);
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <bool QF, int HD>
cudaError_t launch_tc(const PagedAttnArgs& a, cudaStream_t s) {
  using S = TcShape<QF, HD>;
  static SmemOptIn opt;
  CTTS_LK(opt.ensure(reinterpret_cast<const void*>(paged_attn_tc_kernel<QF, HD>), S::SMEM));
  const int box = std::min(a.p.kv.page_size, S::KT);
  if (S::REGS) {
    // the register split below adds up only for a block launched with these
    static PerDeviceInt regs;
    const int n = regs.get([] {
      cudaFuncAttributes at;
      return cudaFuncGetAttributes(&at, paged_attn_tc_kernel<QF, HD>) == cudaSuccess ? at.numRegs : 0;
    });
    if (n != S::LAUNCH_REGS) return cudaErrorLaunchOutOfResources;
  }
  CUtensorMap mk, mv;
  int order = 0;
  if (!paged_pool_map(&mk, a.p.kv.k, a.p.kv, box, &order) || !paged_pool_map(&mv, a.p.kv.v, a.p.kv, box, &order)) return cudaErrorInvalidValue;
  return launch_k(paged_attn_tc_kernel<QF, HD>, dim3(a.ctas), dim3(S::THREADS), S::SMEM, s, mk, mv, a, box, order);
}

}  // namespace

PagedAttnTc paged_attn_tc_plan(const ctts_paged_attn& p) {
  PagedAttnTc t;
  t.ctas = device_sms();
  t.tile_rows = p.q_dtype == CTTS_F32 && p.kv.head_dim == 128 ? 128 : 256;
  return t;
}

cudaError_t launch_paged_attn_tc(const PagedAttnArgs& a, cudaStream_t s) {
  const bool qf = a.p.q_dtype == CTTS_F32;
  if (a.p.kv.head_dim == 64) return qf ? launch_tc<true, 64>(a, s) : launch_tc<false, 64>(a, s);
  return qf ? launch_tc<true, 128>(a, s) : launch_tc<false, 128>(a, s);
}

}  // namespace ctts
