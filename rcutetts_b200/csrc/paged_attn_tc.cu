// paged_attn_tc.cu -- attention of chunks of new rows over a paged cache on
// the 5th-generation tensor cores (tcgen05).
//
// An item is one or two sub-tiles of 128 packed rows (one row per TMEM lane)
// of one request and KV head.  Per key tile and sub-tile:
//   S = Q . K^T   both operands in shared memory (K-major, 128-byte swizzle),
//   softmax       one thread per row: S read from TMEM, the weights written
//                 back in bf16 (bf16 calls: over S),
//   O += P . V    P read from TMEM, V from shared memory as it lies in the
//                 pages ([key][dim]: the MN-major form of the B operand).
// Four warps run the softmax of a sub-tile, one warp issues the MMAs.  A bf16
// cache comes in by one warp's TMA copies: a box per page and 64 dims (a 4D
// map over the pool), K and V in rings of their own; missing pages are boxes
// outside the map, which arrive as zeros.  A float32 cache comes in by two or
// four warps' plain loads, which split it into its bf16 terms on the way.
//
// Two sub-tiles take turns: one computes exponentials while the tensor core
// multiplies for the other, and P arrives in two halves, so that P.V begins
// over the second half's exponentials.  One sub-tile (where shared memory or
// registers hold no second) has two S instead: the scores of tile i + 1 are
// computed over the softmax of tile i.  bf16 items with rows for one sub-tile
// only (single tokens among chunks) give every other key tile to the second.
//
// bf16: the output is rescaled only when a row's maximum has grown by more
// than 2^8 since the last time: weights up to 256 lose nothing in floating
// point, and the pass over O in TMEM becomes rare.  The scores stay in
// registers between the maximum and the exponentials.  The weights are rounded
// to bf16 (2^-8 of each at most), as the tensor core takes one type for both
// operands of P . V: the output's relative error is 0.0020 to 0.0023 where its
// own rounding to bf16 makes 0.0017.
//
// float32 queries: queries and weights enter as three bf16 terms (24 bits),
// and so do keys and values of a float32 cache; of the products those below
// 2^-24 of the whole are left out, which leaves three or six.  Key tiles are
// 64 wide so that three terms of the weights fit beside S.  Each P.V starts
// at zero and its threads add it to an output row in registers: the tensor
// core cuts the sums it accumulates instead of rounding them, which over a
// thousand keys costs 2^-18 of the output (measured against 64 bits).
//
// What bounds it.  bf16, 128 dims: a 256 x 128 tile costs 2048 clocks of
// tensor time and 2900 in the steady state, the rest is the chain scores ->
// softmax -> weights of two sub-tiles that cannot cover one another whole
// (tensor pipe 62 %, special functions 60 % busy); 4 chunks of 1500 to 2048
// rows over 4000 to 6100 tokens, 16 heads over 8 KV heads: 335 to 350 us, 910
// to 960 TFLOP/s.  float32: three or six products a tile and as many splits;
// 8 prompts of 190 to 900 rows, 12 heads of 64 over 4, bf16 cache: 36 us;
// 2 chunks of 700 to 1500 over float32: 59 us (both to a fifth more at the
// clocks that follow long calls).  Short calls: some 5 us from
// the launch to the first scores, 2 to 3 for each further item, and the join.
//
// Every wait is bounded; after one that gives up no role waits any more, and
// what the block still writes is NaN.
#include <algorithm>

#include "common.cuh"
#include "launch_state.h"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "tc_ptx.cuh"

namespace ctts {

namespace {

// Warps: 4 of softmax per sub-tile, one that issues MMAs, and one that issues
// the copies of a bf16 cache or some that bring in a float32 one.
template <bool QF, bool KF, int HD>
struct TcShape {
  static constexpr int KT = QF ? 64 : 128;                     // keys per tile
  static constexpr int NSUB = KF || (QF && HD == 128) ? 1 : 2; // sub-tiles: as many as shared memory and registers hold
  static constexpr int R = 128 * NSUB;                         // packed rows per item
  // warps that bring in a float32 cache: two leave the softmax of 128 dims the
  // registers of an output row
  static constexpr int CW = HD == 64 ? 4 : 2;
  static constexpr int THREADS = R + 32 + (KF ? 32 * CW : 32);
  static constexpr int NT = QF ? 3 : 1;                        // bf16 terms of queries and weights
  static constexpr int NK = KF ? 3 : 1;                        // of keys and values
  static constexpr int NC = HD / 64;                           // 128-byte column blocks
  static constexpr uint32_t QTERM = NC * 128 * 128;            // bytes of one term of one sub-tile
  static constexpr uint32_t KTERM = NC * KT * 128;             // of one term of a K or V tile
  static constexpr uint32_t TILE = NK * KTERM;
  static constexpr int NS = KF ? (HD == 64 ? 3 : 1) : (QF ? (HD == 64 ? 6 : 3) : (HD == 64 ? 4 : 2));
  // One sub-tile: the scores of tile i + 1 are computed while tile i is in its
  // softmax, into the other of two S.  Two: they take turns instead.
  static constexpr bool PIPE = NSUB == 1;
  // Two sub-tiles and an item with rows for one: they share its key tiles, the
  // second takes every other one, and their states merge at the end (bf16: the
  // output in TMEM is open to the other sub-tile's warps).  Such a tile then
  // takes 0.9 us instead of 1.4 (64 dims), one of two sub-tiles 1.8.
  static constexpr bool SHARE = NSUB == 2 && !QF;
  // Costs on the line, from the clocks of CTAs by least squares over their
  // tiles and pieces: what equal tiles left uneven.  43 single tokens with 5
  // chunks of 200 to 512, 64 dims: 35.4 us at equal costs and no sharing, 30;
  // 81 with 9: 59, 48; 40 chunks of 20 to 120, 128 dims: 189, 177; 43 with 5
  // there: 101, 79 (costs of 3, 4, 6: 88).
  // float32 queries: with single tokens as above 75 us at equal costs, 69.  (One
  // sub-tile: costs of 1, 3 and 4 tiles an item were no better than 2 in all.)
  using Item = std::conditional_t<
      NSUB == 1, AttnItem<R, KT, 1, 1, 2>,
      std::conditional_t<QF, AttnItem<R, KT, 3, 4, 4>, std::conditional_t<HD == 64, AttnItem<R, KT, 2, 4, 5>, AttnItem<R, KT, 3, 5, 8>>>>;
  // TMEM columns of sub-tile s: S at s * SREG (PIPE: two of KT columns), P over
  // it (bf16) or behind it (three terms of KT / 2), O at OREG + s * OSTEP
  static constexpr uint32_t SREG = QF ? 192 : 128, PCOL = PIPE ? 2 * KT : (QF ? KT : 0);
  static constexpr uint32_t OREG = QF && NSUB == 2 ? 384 : 256, OSTEP = QF ? 64 : 128;
  static_assert(OREG + (NSUB - 1) * OSTEP + HD <= 512 && (PIPE ? PCOL + NT * (KT / 2) <= OREG : PCOL + NT * (KT / 2) <= SREG && NSUB * SREG <= OREG),
                "TMEM columns");
  static constexpr size_t SMEM = (size_t)NSUB * NT * QTERM + (size_t)2 * NS * TILE + NSUB * 4 * 4096 + 1024;  // and 4 KB a softmax warp
};

// Shared-memory descriptors of 128-byte swizzled operands, as their two words.
// K-major: the field for the leading distance is unused (1).  MN-major: rows
// of 64 dims per key, `lbo` bytes between blocks of 64 dims.  Both: 1024 bytes
// between groups of 8 rows.  An operand d bytes on: the low word + d / 16.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
CTTS_DEV uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | ((lbo >> 4) << 16); }
// D f32, A and B bf16, M = 128, N = n; B K-major or MN-major
CTTS_DEV constexpr uint32_t tc_idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
CTTS_DEV void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi));
}
CTTS_DEV void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {  // A from TMEM
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi));
}
// True in one lane of the warp.
CTTS_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
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

CTTS_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Pairs of float32 in one instruction.
CTTS_DEV float2 fma2(float2 x, float a, float b) {  // x * a + b
  float2 r;
  asm("{\n\t.reg .b64 x, a, b;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 a, {%4, %4};\n\tmov.b64 b, {%5, %5};\n\t"
      "fma.rn.f32x2 x, x, a, b;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x.x), "f"(x.y), "f"(a), "f"(b));
  return r;
}
CTTS_DEV float2 add2(float2 x, float2 y) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return r;
}

// Warps w and w + 4 meet.
CTTS_DEV void pair_sync(int w) { asm volatile("bar.sync %0, 64;" ::"r"(w + 1) : "memory"); }

// Byte offsets of packed rows p, p + 4, p + 8, ... (row of q times its stride
// plus head times width), one division for all of them.
struct RowWalk {
  long off, step, wrap;
  int g, over, group;
  CTTS_DEV RowWalk(int p, int grp, long ld_bytes, int head_bytes) : group(grp) {
    const int row = p / grp, per = 4 / grp;
    g = p - row * grp;
    over = 4 - per * grp;
    off = row * ld_bytes + g * head_bytes;
    step = per * ld_bytes + over * head_bytes;
    wrap = ld_bytes - grp * head_bytes;
  }
  CTTS_DEV void next4() {
    off += step;
    g += over;
    if (g >= group) {
      g -= group;
      off += wrap;
    }
  }
};

struct TcBars {
  uint64_t k_full[6], k_empty[6], v_full[6], v_empty[6];
  uint64_t q_full[2], s_full[2], p_half[2], p_full[2], o_full[2], drain;
};

template <bool QF, bool KF, int HD>
__global__ void __launch_bounds__(TcShape<QF, KF, HD>::THREADS, 1) paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                                    const __grid_constant__ CUtensorMap tmV,
                                                                                    const __grid_constant__ PagedAttnArgs a, int box, int order) {
  using S = TcShape<QF, KF, HD>;
  using Cursor = AttnCursor<typename S::Item>;
  constexpr int KT = S::KT, R = S::R, NS = S::NS, NT = S::NT, NC = S::NC;
  constexpr int W_MMA = 4 * S::NSUB, W_TMA = W_MMA + 1;
  constexpr int KS = KT / 16, HALF = QF ? 0 : KS / 2;  // bf16 calls: P arrives in two halves
  extern __shared__ uint8_t tc_smem[];
  __shared__ AttnStart start;
  __shared__ __align__(8) TcBars bars;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t dead_keys[8];  // 8-key groups of a tile whose page does not exist
  __shared__ volatile uint32_t tries;  // of a wait; 0: one gave up
  __shared__ float2 shared_ml[S::SHARE ? 128 : 1];  // maximum and sum of the second sub-tile of a shared item
  const uint32_t sbase = (smem_u32(tc_smem) + 1023u) & ~1023u;
  const uint32_t qs = sbase, ks = qs + S::NSUB * NT * S::QTERM, vs = ks + NS * S::TILE;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);

  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(&bars.k_full[i], KF ? 32 * S::CW : 1);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], KF ? 32 * S::CW : 1);
      mbar_init(&bars.v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&bars.q_full[i], 128);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_half[i], 128);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.o_full[i], 1);
    }
    mbar_init(&bars.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tries = a.tries;
  }
  if (warp == W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  grid_dep_enter();
  attn_find_start<typename S::Item, S::THREADS>(a.line, &start);
  if (tid == 0) a.parts[blockIdx.x].pieces = 0;  // no divided item yet
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  int left;
  Cursor cu = Cursor::at(a.line, start, &left);

  if (!KF && left > 0 && warp == W_TMA) {
    // ---- producer: lane i looks up the page of keys 8i..8i+7 of a tile, the
    // lanes at the boxes' starts copy them
    int kt = cu.kt, end = cu.kt + cu.tiles(left);  // of the piece
    auto page_of = [&]() {
      const int kk = kt * KT + 8 * lane;
      return lane < KT / 8 && kk < cu.len ? a.p.block_tables[(long)cu.b * a.p.table_ld + (kk >> a.shift)] : -1;
    };
    int page = page_of(), st = 0, u = 0;
    uint32_t par = 0;
#pragma unroll 1
    for (bool more = true; more && tries; u++) {
      const int kk = kt * KT + 8 * lane, h = cu.h, slot = kk & (a.p.kv.page_size - 1);
      const bool none = (unsigned)page >= (unsigned)a.p.kv.n_pages;
      const uint32_t dead = __ballot_sync(0xffffffffu, lane < KT / 8 && kk < cu.len && none);
      const int from = none ? a.p.kv.n_pages : page;  // outside the map: zeros
      if (++kt == end) {
        left = cu.behind(left, end - cu.kt);
        more = left > 0;
        if (more) {
          cu = Cursor::next(a.line, cu);
          kt = 0;
          end = cu.tiles(left);
        }
      }
      if (more) page = page_of();  // of the next tile, over the waits
      const bool copies = lane < KT / 8 && (8 * lane & (box - 1)) == 0;
#pragma unroll 1
      for (int kv = 0; kv < 2; kv++) {
        uint64_t* full = kv ? &bars.v_full[st] : &bars.k_full[st];
        if (u >= NS) mbar_wait_or(kv ? &bars.v_empty[st] : &bars.k_empty[st], par ^ 1, &tries);
        if (lane == 0) {
          if (kv == 0) dead_keys[u & 7] = dead;  // read behind the scores' barrier; the copies are at most 6 tiles ahead
          mbar_expect_tx(full, S::TILE);
        }
        __syncwarp();
        if (copies) {
          const uint32_t dst = (kv ? vs : ks) + st * S::TILE + (uint32_t)lane * 1024u;
#pragma unroll 1
          for (int c = 0; c < NC; c++) copy_box(dst + c * KT * 128, kv ? &tmV : &tmK, order, c * 64, slot, h, from, full);
        }
      }
      if (++st == NS) {
        st = 0;
        par ^= 1;
      }
    }
    // copies in flight land before the block may leave, whoever gave up
#pragma unroll 1
    for (int w = max(0, u - NS); w < u; w++) {
      mbar_wait(&bars.k_full[w % NS], (uint32_t)(w / NS) & 1);
      mbar_wait(&bars.v_full[w % NS], (uint32_t)(w / NS) & 1);
    }
  } else if (KF && left > 0 && warp > W_MMA) {
    // ---- producers of a float32 cache: keys and values come in by plain
    // loads (16 threads a row of 64 dims), 64 dims of 64 keys ahead of the
    // ones that are being split into their bf16 terms
    const int ct = tid - 32 * (W_MMA + 1), f4 = ct & 15, kr = ct >> 4;
    constexpr int JOBS = 2 * NC;  // a tile: K's blocks of 64 dims, then V's
    constexpr int RT = 2 * S::CW, NI = KT / RT;  // rows a turn, turns
    int kt = cu.kt, end = cu.kt + cu.tiles(left), st = 0, u = 0;
    uint32_t par = 0, dead = 0, dead_next = 0;
    int page = -1;
    bool more = true;
    float4 buf[2][NI];
    auto look = [&]() {  // lane i: the page of keys 8i..8i+7 of tile kt
      const int kk = kt * KT + 8 * lane;
      page = lane < 8 && kk < cu.len ? a.p.block_tables[(long)cu.b * a.p.table_ld + (kk >> a.shift)] : -1;
      const bool none = (unsigned)page >= (unsigned)a.p.kv.n_pages;
      dead_next = __ballot_sync(0xffffffffu, lane < 8 && kk < cu.len && none);
      if (none) page = -1;
    };
    auto fetch = [&](int job, float4* r) {
      const float* pool = static_cast<const float*>(job < NC ? a.p.kv.k : a.p.kv.v) + (long)cu.h * a.p.kv.head_stride + (job % NC) * 64 + f4 * 4;
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int key = kt * KT + RT * i + kr, pg = __shfl_sync(0xffffffffu, page, RT * i >> 3);
        r[i] = make_float4(0.f, 0.f, 0.f, 0.f);  // slots behind the length and missing pages
        if (key < cu.len && pg >= 0)
          r[i] = *reinterpret_cast<const float4*>(pool + (long)pg * a.p.kv.page_stride + (long)(key & (a.p.kv.page_size - 1)) * a.p.kv.token_stride);
      }
    };
    look();
    fetch(0, buf[0]);
#pragma unroll 1
    while (more) {
      dead = dead_next;
#pragma unroll
      for (int job = 0; job < JOBS; job++) {
        if (job + 1 < JOBS) {
          fetch(job + 1, buf[(job + 1) & 1]);
        } else {
          if (++kt == end) {
            left = cu.behind(left, end - cu.kt);
            more = left > 0;
            if (more) {
              cu = Cursor::next(a.line, cu);
              kt = 0;
              end = cu.tiles(left);
            }
          }
          if (more) {
            look();
            fetch(0, buf[0]);
          }
        }
        const int kv = job / NC, c = job % NC;
        uint64_t* full = kv ? &bars.v_full[st] : &bars.k_full[st];
        if (c == 0 && u >= NS) mbar_wait_or(kv ? &bars.v_empty[st] : &bars.k_empty[st], par ^ 1, &tries);
        const uint32_t dst = (kv ? vs : ks) + st * S::TILE + c * KT * 128;
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const float4 x = buf[job & 1][i];
          const int key = RT * i + kr;
          uint32_t t[2][3];
          split_bf2<3>(x.x, x.y, t[0]);
          split_bf2<3>(x.z, x.w, t[1]);
#pragma unroll
          for (int k = 0; k < 3; k++)
            asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(dst + k * S::KTERM + key * 128 + (((f4 >> 1) ^ key) & 7) * 16 + (f4 & 1) * 8),
                         "r"(t[0][k]), "r"(t[1][k])
                         : "memory");
        }
        if (c == NC - 1) {
          if (job == NC - 1 && ct == 0) dead_keys[u & 7] = dead;
          fence_async();
          mbar_arrive(full);
        }
      }
      u++;
      if (++st == NS) {
        st = 0;
        par ^= 1;
      }
    }
  } else if (left > 0 && warp == W_MMA) {
    // ---- MMA issue.  The warp runs through as one (what it computes with is
    // uniform), one lane issues; between its products it does next to nothing:
    // what it spends there the tensor core stands still.
    const bool leader = elect_one();
    // Products of terms i of one operand and j of the other whose orders add
    // up to more than two are left out: they lie below 2^-24 of the whole.
    // Small ones first: the tensor core cuts what it adds to the accumulator's
    // precision.
    constexpr int ORDER = (NT - 1) > (S::NK - 1) ? NT - 1 : S::NK - 1;
    auto scores = [&](int s, int st, uint32_t col, uint64_t* bar) {
      const uint32_t kb = desc_lo(ks + st * S::TILE, 16), qb = desc_lo(qs + s * NT * S::QTERM, 16);
      fence_after();
      if (leader) {
        uint32_t acc = 0;
#pragma unroll
        for (int o = ORDER; o >= 0; o--)
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const int j = o - t;
            if (j < 0 || j >= S::NK) continue;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
              for (int k = 0; k < 4; k++) {
                mma_ss(tmem + col, qb + (t * S::QTERM + c * 16384 + k * 32) / 16, kb + (j * S::KTERM + c * KT * 128 + k * 32) / 16,
                       tc_idesc(KT, false), acc);
                acc = 1;
              }
          }
        umma_commit(bar);
      }
      __syncwarp();
    };
    auto values = [&](int s, int st, int k0, int k1, uint32_t acc) {
      const uint32_t vb = desc_lo(vs + st * S::TILE, KT * 128);
      fence_after();
      if (leader) {
#pragma unroll
        for (int o = ORDER; o >= 0; o--)
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const int j = o - t;
            if (j < 0 || j >= S::NK) continue;
#pragma unroll
            for (int k = k0; k < k1; k++) {
              mma_ts(tmem + S::OREG + S::OSTEP * s, tmem + S::SREG * s + S::PCOL + t * (KT / 2) + k * 8, vb + j * (S::KTERM / 16) + k * 128,
                     tc_idesc(HD, true), acc);
              acc = 1;
            }
          }
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
    };
    const bool keeps = a.keep_cta0 && blockIdx.x == 0;
    auto release = [&](uint64_t* bar) {  // a stage back to the producer
      if (!keeps) commit(bar);
    };
    uint32_t q_par = 0, p_par = 0;  // one bit per sub-tile
    uint32_t par = 0, par_p = 0;    // of the fills of stages st (tile i) and sp (tile i - 1)
    int st = 0, sp = 0;
#pragma unroll 1
    while (true) {
      const int n = __shfl_sync(0xffffffffu, cu.tiles(left), 0);
      const int nsub = __shfl_sync(0xffffffffu, cu.rows(a.line, R) > 128 ? 2 : 1, 0);
      if (S::PIPE) {
        // a turn: scores of tile i, then P.V of tile i - 1
        mbar_wait_or(&bars.q_full[0], q_par, &tries);
        q_par ^= 1;
#pragma unroll 1
        for (int i = 0; i <= n; i++) {
          if (i < n) {
            mbar_wait_or(&bars.k_full[st], par, &tries);
            scores(0, st, (i & 1) * KT, &bars.s_full[i & 1]);
            release(&bars.k_empty[st]);
          }
          if (i > 0) {
            mbar_wait_or(&bars.p_full[0], p_par, &tries);
            p_par ^= 1;
            mbar_wait_or(&bars.v_full[sp], par_p, &tries);
            values(0, sp, 0, KS, 0);
            commit(&bars.o_full[0]);
            release(&bars.v_empty[sp]);
          }
          if (i < n) {
            sp = st;
            par_p = par;
            if (++st == NS) {
              st = 0;
              par ^= 1;
            }
          }
        }
      } else if (S::SHARE && nsub == 1) {
        // a turn: scores of tile i, then P.V of tile i - 1 for the other sub-tile
#pragma unroll 1
        for (int i = 0; i <= n; i++) {
          if (i < n) {
            const int s = i & 1;
            if (i < 2) {
              mbar_wait_or(&bars.q_full[s], (q_par >> s) & 1, &tries);
              q_par ^= 1u << s;
            }
            mbar_wait_or(&bars.k_full[st], par, &tries);
            scores(s, st, S::SREG * s, &bars.s_full[s]);
            release(&bars.k_empty[st]);
          }
          if (i > 0) {
            const int s = (i - 1) & 1;
            mbar_wait_or(&bars.v_full[sp], par_p, &tries);
            mbar_wait_or(&bars.p_half[s], (p_par >> s) & 1, &tries);
            values(s, sp, 0, HALF, i > 2);
            mbar_wait_or(&bars.p_full[s], (p_par >> s) & 1, &tries);
            p_par ^= 1u << s;
            values(s, sp, HALF, KS, 1u);
            if (i + 1 >= n) commit(&bars.o_full[s]);  // its last tile
            release(&bars.v_empty[sp]);
          }
          if (i < n) {
            sp = st;
            par_p = par;
            if (++st == NS) {
              st = 0;
              par ^= 1;
            }
          }
        }
      } else {
        // a turn: P.V of tile i - 1, scores of tile i
#pragma unroll 1
        for (int i = 0; i <= n; i++) {
          if (i > 0) mbar_wait_or(&bars.v_full[sp], par_p, &tries);
#pragma unroll 1
          for (int s = 0; s < nsub; s++) {
            if (i > 0) {
              if (HALF) {
                mbar_wait_or(&bars.p_half[s], (p_par >> s) & 1, &tries);
                values(s, sp, 0, HALF, i > 1);
              }
              mbar_wait_or(&bars.p_full[s], (p_par >> s) & 1, &tries);
              p_par ^= 1u << s;
              values(s, sp, HALF, KS, HALF ? 1u : 0u);
              if (i == n) commit(&bars.o_full[s]);
            }
            if (i < n) {
              if (i == 0) {
                mbar_wait_or(&bars.q_full[s], (q_par >> s) & 1, &tries);
                q_par ^= 1u << s;
              }
              if (s == 0) mbar_wait_or(&bars.k_full[st], par, &tries);
              scores(s, st, S::SREG * s, &bars.s_full[s]);
            }
          }
          if (i > 0) release(&bars.v_empty[sp]);
          if (i < n) {
            release(&bars.k_empty[st]);
            sp = st;
            par_p = par;
            if (++st == NS) {
              st = 0;
              par ^= 1;
            }
          }
        }
      }
      left = __shfl_sync(0xffffffffu, cu.behind(left, n), 0);
      if (left == 0) break;
      cu = Cursor::next(a.line, cu);
    }
    if (tries == 0) {  // MMAs in flight end before TMEM is given back
      commit(&bars.drain);
      mbar_wait(&bars.drain, 0);
    }
  } else if (left > 0 && warp < W_MMA) {
    // ---- softmax: one thread per packed row
    const int s = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS0 = tmem + S::SREG * s + lane_base, tP = tS0 + S::PCOL, tO = tmem + S::OREG + S::OSTEP * s + lane_base;
    const float c2 = a.c2;
    uint32_t s_par = 0, o_par = 0;
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
    // A turn: the queries of the next piece go to shared memory (and its first
    // scores may begin), then the piece before is written out, then the next
    // one's tiles run.
    Cursor nx = cu;
    int u = 0, end = -1;  // tiles of the pieces before; of the current piece (-1: none yet)
    int over = 0;         // units by which its last tile reaches past the CTA's end
    auto shares = [&](const Cursor& c) { return S::SHARE && c.rows(a.line, R) <= 128; };
    // the sub-tile takes part in a piece of n tiles
    auto takes_part = [&](const Cursor& c, int n) { return s * 128 < c.rows(a.line, R) || (S::SHARE && n > 1); };
    float m = -INFINITY, l = 0.0f;
#pragma unroll 1
    while (true) {
      if (left > 0 && takes_part(nx, nx.tiles(left))) {
        const int r0 = (shares(nx) ? 0 : s * 128) + (warp & 3) * 32, nrows = nx.rows(a.line, R);  // the warp's first row in the item
        // the warp's 32 queries as bf16 terms: eight lanes read 128 bytes of a
        // row (as bf16), four rows at a time, all loads in flight before the
        // first is used; rows behind the item are zero
#pragma unroll 1
        for (int c = 0; c < NC; c++) {
          constexpr int RP = 8;  // rows a lane reads: 4 i + lane / 8
          uint4 x[RP], y[QF ? RP : 1];
          constexpr int ES = QF ? 4 : 2;
          RowWalk w(nx.m * R + r0 + (lane >> 3), a.group, a.p.q_ld * ES, HD * ES);
          const uint8_t* q = static_cast<const uint8_t*>(a.p.q) + ((long)nx.r0 * a.p.q_ld + nx.h * a.group * HD + c * 64 + (lane & 7) * 8) * ES;
          const int left = nrows - r0 - (lane >> 3);  // rows behind the item (4 i >= left) read its first row and count as zero
#pragma unroll
          for (int i = 0; i < RP; i++) {
            const uint4* at = reinterpret_cast<const uint4*>(q + (4 * i < left ? w.off : 0));
            x[i] = at[0];
            if (QF) y[QF ? i : 0] = at[1];
            w.next4();
          }
          if (r0 + 32 > nrows) {
#pragma unroll
            for (int i = 0; i < RP; i++)
              if (4 * i >= left) {
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (QF) y[QF ? i : 0] = x[i];
              }
          }
#pragma unroll
          for (int i = 0; i < RP; i++) {
            const int r = (warp & 3) * 32 + 4 * i + (lane >> 3);
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
      if (end >= 0 && takes_part(cu, end - cu.kt)) {
        const int nrows = cu.rows(a.line, R), first_row = shares(cu) ? 0 : s * 128;
        const bool mine = first_row + row < nrows, warp_on = first_row + (warp & 3) * 32 < nrows;
        const bool shared = shares(cu) && end - cu.kt > 1;
        // ---- the piece's output, or its partial state
        const bool ends = end == cu.nt, whole = ends && cu.kt == 0;
        const int place = 2 * blockIdx.x + (cu.kt == 0 ? 1 : 0);
        if (!ends && cu.kt == 0 && s == 0 && row == 0) {
          AttnPart d;
          d.pieces = attn_pieces<typename S::Item>(a.line, start, over + (cu.nt - end - 1) * cu.w);
          d.row0 = cu.r0; d.packed0 = cu.m * R; d.rows = nrows; d.h = cu.h;
          a.parts[blockIdx.x] = d;
        }
        mbar_wait_or(&bars.o_full[s], o_par, &tries);
        o_par ^= 1;
        if (shared && s == 1) {
          // the other sub-tile's warp of the same rows (and TMEM lanes) merges
          // the states and writes them; O stays until it has
          if (warp_on) {
            shared_ml[row] = make_float2(m, l);
            fence_before();
            pair_sync(warp & 3);
            pair_sync(warp & 3);
            fence_after();
          }
        } else if (warp_on) {
          float f0 = 1.0f, f1 = 0.0f;
          if (shared) {
            pair_sync(warp & 3);
            const float2 other = shared_ml[row];
            const float mm = fmaxf(m, other.x), mz = mm == -INFINITY ? 0.0f : mm;
            f0 = exp2_fast(attn_arg(m, mz, c2));
            f1 = exp2_fast(attn_arg(other.x, mz, c2));
            m = mm;
            l = fmaf(other.y, f1, l * f0);
          }
          fence_after();
          const bool none = l == 0.0f;  // the row saw no key (one that saw any has a weight of 1, or NaN)
          float inv = whole && !none ? 1.0f / l : 1.0f;
          if (tries == 0) inv = __int_as_float(0x7fffffff);  // a wait gave up: what was computed since may be anything
          if (!whole && mine) a.ml[(long)place * a.tile_rows + first_row + row] = make_float2(m, l);
          if (QF) gather();
          // 32 columns of the warp's 32 rows by way of shared memory: a lane
          // holds a row, eight lanes write 128 bytes of one (four lanes 64
          // bytes in bf16)
          const uint32_t stage = vs + NS * S::TILE + warp * 4096;
          const bool half = whole && !QF;
          const int r0 = first_row + (warp & 3) * 32, left = nrows - r0 - (lane >> 3), es = half ? 2 : 4;
          RowWalk w0(cu.m * R + r0 + (lane >> 3), a.group, a.p.out_ld * es, HD * es);
          uint8_t* dst = static_cast<uint8_t*>(a.p.out) + ((long)cu.r0 * a.p.out_ld + cu.h * a.group * HD) * es;
          if (!whole) {  // rows of the partial state follow one another
            w0.off = (long)(r0 + (lane >> 3)) * HD * 4;
            w0.step = 4 * HD * 4;
            w0.g = w0.over = 0;
            dst = reinterpret_cast<uint8_t*>(a.acc + (long)place * a.tile_rows * HD);
          }
          dst += (lane & 7) * 16;
          const bool writes = !half || (lane & 7) < 4;
          auto put = [&](int c, uint32_t* o) {
            if (none) {
#pragma unroll
              for (int j = 0; j < 32; j++) o[j] = 0u;
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
              float v[4];
#pragma unroll
              for (int e = 0; e < 4; e++) v[e] = __uint_as_float(o[4 * j + e]) * inv;
              if (half)
                asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(stage + lane * 128 + (((j >> 1) ^ lane) & 7) * 16 + (j & 1) * 8),
                             "r"(pack_bf2(v[0], v[1])), "r"(pack_bf2(v[2], v[3]))
                             : "memory");
              else
                asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * 128 + ((j ^ lane) & 7) * 16), "f"(v[0]), "f"(v[1]),
                             "f"(v[2]), "f"(v[3])
                             : "memory");
            }
            __syncwarp();
            RowWalk w = w0;
            uint8_t* d = dst + c * es;
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
              const int r = 4 * i + (lane >> 3);
              asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(v[i].x), "=r"(v[i].y), "=r"(v[i].z), "=r"(v[i].w)
                           : "r"(stage + r * 128 + ((lane ^ r) & 7) * 16)
                           : "memory");
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
              if (writes && 4 * i < left) *reinterpret_cast<uint4*>(d + w.off) = v[i];
              w.next4();
            }
            __syncwarp();
          };
          if (QF) {
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
#pragma unroll
              for (int j = 0; j < 32; j++) o[j] = __float_as_uint(o_row[QF ? c + j : 0]);
              put(c, o);
            }
          } else {
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              tmem_ld32_nowait(tO + c, o);
              if (shared) {
                uint32_t o1[32];
                tmem_ld32_nowait(tO + S::OSTEP + c, o1);
                tmem_wait();
                pin32(o);
                pin32(o1);
#pragma unroll
                for (int j = 0; j < 32; j++) o[j] = __float_as_uint(fmaf(__uint_as_float(o1[j]), f1, __uint_as_float(o[j]) * f0));
              } else {
                tmem_wait();
                pin32(o);
              }
              put(c, o);
            }
          }
          fence_before();
          if (shared) pair_sync(warp & 3);
        }
      }
      if (left == 0) break;
      // ---- a piece: tiles cu.kt .. end of an item
      if (end >= 0) u += end - cu.kt;
      cu = nx;
      end = cu.kt + cu.tiles(left);
      const int nrows = cu.rows(a.line, R);
      if (takes_part(cu, end - cu.kt)) {
        const int first_row = shares(cu) ? 0 : s * 128;
        const int first = cu.kt + (shares(cu) ? s : 0), step = shares(cu) ? 2 : 1;  // its tiles
        const bool warp_on = first_row + (warp & 3) * 32 < nrows;
        const int pk = cu.m * R + first_row + row;
        const int pos = cu.pos0() + pk / a.group, pos_lo = cu.pos0() + (pk - lane) / a.group;
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int c = 0; c < (QF ? HD : 1); c++) o_row[c] = 0.0f;
#pragma unroll 1
        for (int kt = first; kt < end; kt += step) {
          const int key0 = kt * KT;
          const int sb = S::PIPE ? (kt - cu.kt) & 1 : s;
          const uint32_t tS = tS0 + (S::PIPE ? sb * KT : 0);
          mbar_wait_or(&bars.s_full[sb], (s_par >> sb) & 1, &tries);
          s_par ^= 1u << sb;
          if (!KF && (s == 0 || step == 2) && key0 + KT > cu.len) {
            // slots behind the length may hold anything, and 0 * NaN is NaN:
            // their values become zeros (the products come after this
            // sub-tile's arrival at p_half or p_full, both sub-tiles' ones).
            // Behind the scores, as a barrier's parity tells the fill of this
            // tile from the one before last only once that one is over.
            const int w = u + kt - cu.kt, st = w % NS;
            mbar_wait_or(&bars.v_full[st], (uint32_t)(w / NS) & 1, &tries);
            if (row < KT && key0 + row >= cu.len) {
#pragma unroll 1
              for (int c = 0; c < NC * 8; c++)
                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(vs + st * S::TILE + (c >> 3) * KT * 128 + row * 128 + (c & 7) * 16), "r"(0)
                             : "memory");
            }
            fence_async();
          }
          if (warp_on) {
            fence_after();
            const uint32_t dead = dead_keys[(u + kt - cu.kt) & 7];
            if (key0 + KT - 1 > pos_lo || dead) {
              // hidden keys: -inf over their scores
#pragma unroll 1
              for (int c = 0; c < KT; c += 32) {
                uint32_t x[32];
                tmem_ld32_nowait(tS + c, x);
                tmem_wait();
                pin32(x);
#pragma unroll
                for (int g = 0; g < 4; g++) {
                  const int lim = (dead >> (c / 8 + g)) & 1 ? -1 : pos - key0 - c - 8 * g;  // the last key of the eight that is seen
#pragma unroll
                  for (int j = 0; j < 8; j++)
                    if (j > lim) x[8 * g + j] = 0xff800000u;
                }
                tmem_st32(tS + c, x);
              }
              tmem_st_wait();
            }
            float mn;
            uint32_t x[KT];
            {
#pragma unroll
              for (int c = 0; c < KT; c += 32) tmem_ld32_nowait(tS + c, x + c);
              tmem_wait();
#pragma unroll
              for (int c = 0; c < KT; c += 32) pin32(x + c);
              float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int c = 0; c < KT; c += 8)
#pragma unroll
                for (int j = 0; j < 4; j++) mx[j] = max3(mx[j], __uint_as_float(x[c + 2 * j]), __uint_as_float(x[c + 2 * j + 1]));
              mn = max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
            }
            if (QF) {
              if (kt > cu.kt) {
                if (S::PIPE) {  // (two sub-tiles: the scores were issued behind it)
                  mbar_wait_or(&bars.o_full[0], o_par, &tries);
                  o_par ^= 1;
                  fence_after();
                }
                gather();
              }
              const float mm = fmaxf(m, mn), f = mm == -INFINITY ? 0.0f : exp2_fast(attn_arg(m, mm, c2));
              m = mm;
              l *= f;
#pragma unroll
              for (int c = 0; c < (QF ? HD : 1); c++) o_row[c] *= f;
            } else if (kt == first) {
              m = mn;  // O is overwritten by the first product
            } else {
              const bool grow = (mn - m) * c2 > 8.0f;
              if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? exp2_fast(attn_arg(m, mn, c2)) : 1.0f;
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
            // the weights, 32 keys at a time (bf16 calls from the scores in
            // registers; float32 ones read theirs again)
            if (QF) {
              float sum[2] = {0.f, 0.f};
#pragma unroll 1
              for (int c = 0; c < KT; c += 32) {
                uint32_t x[32], p[NT][16];
                tmem_ld32_nowait(tS + c, x);
                tmem_wait();
                pin32(x);
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                  const float e0 = exp2_fast(attn_arg(__uint_as_float(x[j]), mz, c2));
                  const float e1 = exp2_fast(attn_arg(__uint_as_float(x[j + 1]), mz, c2));
                  sum[0] += e0;
                  sum[1] += e1;
                  uint32_t t[NT];
                  split_bf2<NT>(e0, e1, t);
#pragma unroll
                  for (int k = 0; k < NT; k++) p[k][j >> 1] = t[k];
                }
#pragma unroll
                for (int k = 0; k < NT; k++) tmem_st16(tP + k * (KT / 2) + (c >> 1), p[k]);
              }
              l += sum[0] + sum[1];
            } else {
              // One rounding of m * c2 costs 2^-24 of it, far below bf16 while it
              // is moderate; of huge scores the maximum is taken off first.
              // (Always: 64 more instructions a tile, chunks 1 %, mixed
              // batches 3 % slower.)
              float mc = mz * c2;
              if (__any_sync(0xffffffffu, fabsf(mc) > 16384.0f)) {
#pragma unroll
                for (int j = 0; j < KT; j++) x[j] = __float_as_uint(__uint_as_float(x[j]) - mz);
                mc = 0.0f;
              }
              float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
              auto weights = [&](const uint32_t* x, int c) {
                uint32_t p[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                  float2 e = fma2(make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), c2, -mc);
                  e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                  sum[j & 1] = add2(sum[j & 1], e);
                  p[j] = pack_bf2(e.x, e.y);
                }
                tmem_st16(tP + (c >> 1), p);
              };
#pragma unroll
              for (int c = 0; c < KT; c += 32) {
                weights(x + c, c);
                if (c + 32 == HALF * 16) {
                  tmem_st_wait();
                  fence_before();
                  mbar_arrive(&bars.p_half[s]);
                }
              }
              l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            tmem_st_wait();
            fence_before();
          } else if (!QF) {
            mbar_arrive(&bars.p_half[s]);
          } else if (S::PIPE && kt > cu.kt) {
            // a warp without rows keeps step: its arrival for this tile must
            // not count for the one before
            mbar_wait_or(&bars.o_full[0], o_par, &tries);
            o_par ^= 1;
          }
          mbar_arrive(&bars.p_full[s]);
        }
      }
      over = (end - cu.kt) * cu.w - left;
      left = cu.behind(left, end - cu.kt);
      if (left > 0) nx = Cursor::next(a.line, cu);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <bool QF, bool KF, int HD>
cudaError_t launch_tc(const PagedAttnArgs& a, cudaStream_t s) {
  using S = TcShape<QF, KF, HD>;
  static SmemOptIn opt;
  CTTS_LK(opt.ensure(reinterpret_cast<const void*>(paged_attn_tc_kernel<QF, KF, HD>), S::SMEM));
  const int box = std::min(a.p.kv.page_size, (int)S::KT);
  CUtensorMap mk{}, mv{};
  int order = 0;
  if (!KF && (!paged_pool_map(&mk, a.p.kv.k, a.p.kv, box, &order) || !paged_pool_map(&mv, a.p.kv.v, a.p.kv, box, &order)))
    return cudaErrorInvalidValue;
  return launch_k(paged_attn_tc_kernel<QF, KF, HD>, dim3(a.line.ctas), dim3(S::THREADS), S::SMEM, s, mk, mv, a, box, order);
}

// f(QF, KF, HD as integral constants) of the call
template <class F>
auto with_tc_shape(const ctts_paged_attn& p, F f) {
  using T = std::true_type;
  using N = std::false_type;
  auto g = [&](auto hd) {
    if (p.q_dtype == CTTS_BF16) return f(N{}, N{}, hd);
    return p.kv.dtype == CTTS_F32 ? f(T{}, T{}, hd) : f(T{}, N{}, hd);
  };
  return p.kv.head_dim == 128 ? g(std::integral_constant<int, 128>{}) : g(std::integral_constant<int, 64>{});
}

}  // namespace

int paged_attn_tc_rows(const ctts_paged_attn& p) {
  return with_tc_shape(p, [](auto q, auto k, auto hd) { return TcShape<decltype(q)::value, decltype(k)::value, decltype(hd)::value>::R; });
}

cudaError_t launch_paged_attn_tc(const PagedAttnArgs& a, cudaStream_t s) {
  return with_tc_shape(a.p, [&](auto q, auto k, auto hd) { return launch_tc<decltype(q)::value, decltype(k)::value, decltype(hd)::value>(a, s); });
}

}  // namespace ctts
