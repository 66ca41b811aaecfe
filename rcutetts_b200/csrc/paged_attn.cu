// paged_attn.cu -- attention of new rows over a paged KV cache.
//
//   out_r = sum_{j <= pos_r} w_rj v_j,  w_r = softmax(scale q_r . k_j)
//
// The query heads of a KV head and the new rows of a request are packed into
// one row axis (r = row * group + head in group), so keys and values are read
// once per KV head.  A work item is (request, tile of packed rows, KV head);
// its keys go by in tiles under an online softmax (running maximum and sum in
// float32).  The key tiles of all items form one line that is cut into equal
// pieces, one per persistent CTA: ragged lengths, one long request and many
// short ones all load the GPU evenly.  An item that a cut divides leaves
// partial states (maximum, sum, unnormalised output) in the workspace, which
// paged_attn_join_kernel merges in line order; the others are written at
// once.  Which CTA does what follows from the lengths on the device alone, so
// the host knows no lengths and a captured call follows them.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "launch_state.h"
#include "paged.cuh"
#include "paged_attn.cuh"

namespace ctts {

namespace {

constexpr int kNT = 128;   // threads that compute; a warp behind them issues the copies

CTTS_DEV void mma_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CTTS_DEV void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
CTTS_DEV void ldsm4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Short items: up to 16 packed rows (single tokens and short runs).  The four
// warps share the rows and split each key tile's keys, each with their own
// softmax states, which merge in warp order at the end of a piece.  RH = 1: no
// item has more than 8 rows (the upper half of the MMA's 16 rows stays zero
// and unread).  Bound by the cache's bytes: what there is to compute per key
// (mma.sync m16n8k16, two products of 16 rows) is far below what the tensor
// core's legacy path gives, so the tiles go by in a ring that one producer
// warp fills by TMA; where shared memory holds two blocks an SM they overlap
// their latencies.
// 30 requests of 2000 to 32000 tokens, 16 heads on 8 KV heads of 128, bf16:
// 181 us, 6.5 TB/s (plain cp.async loads by the computing warps: 272 us).
// With float32 queries an SM holds one block there: 273 us, 4.4 TB/s; over a
// float32 cache, twice the bytes, 565 us, 4.3 TB/s.
template <bool QF, bool KF, int HD, int RH>
struct Shape {
  static constexpr int R = 8 * RH;
  static constexpr int RQ = 16;  // query rows held
  // bf16 terms of a float32 operand (queries and softmax weights; keys and
  // values of a float32 cache): 24 bits, so a float32 call keeps float32
  static constexpr int NQ = QF ? 3 : 1;
  static constexpr int NP = QF ? 3 : 1;
  static constexpr int ES = KF ? 4 : 2;
  static constexpr int C = !KF && HD == 64 ? 128 : 64;  // keys per tile: 16 KB of K (float32 of 128 dims: 32), and as much of V
  static constexpr int NB = HD * ES / 128;              // 128-byte blocks of a row
  // (without the cost of items the CTAs that draw many short ones end last)
  using Item = AttnItem<R, C, 1, 1, 2>;
  static constexpr uint32_t TILE = NB * C * 128;        // a K or V tile: [block][key][128 B], 16-byte chunks swizzled by key
  static constexpr uint32_t STAGE = 2 * TILE;
  static constexpr int NS = STAGE <= 32768 ? 3 : 2;
  static constexpr int QBYTES = NQ * RQ * HD * 2;
  static constexpr int KT = C / 32;  // 8-key column tiles per warp and key tile
  // query fragments stay in registers where they are few
  static constexpr bool QREG = NQ * (HD / 16) * 2 * RH <= 16;
  static constexpr size_t smem(int rows_used) { return 1024 + (size_t)NS * STAGE + QBYTES + (size_t)4 * rows_used * (HD + 2) * 4; }
  // Blocks that an SM's shared memory holds: 228 KB, of which each takes 1 KB
  // and its static variables beside its own.  Two of 16 KB tiles while their
  // rows are few: 64 dims up to 8 rows and more, 128 dims up to 5 (float32
  // queries: a single one); else one.
  static constexpr int blocks(int rows_used) {
    const int n = (int)(228 * 1024 / (smem(rows_used) + 1024 + 512));
    return n < 1 ? 1 : (n > 4 ? 4 : n);
  }
  // What the registers have to leave room for: as many as with the fewest rows.
  // (Room for two where one fits made float32 queries over 128 dims spill: 64
  // single tokens of 150 to 1200, 16 heads on one 16.7 us, 15.9 without.)
  static constexpr int CTAS = blocks(RH == 1 ? 1 : 9);
};

template <bool QF, bool KF, int HD, int RH>
__global__ void __launch_bounds__(kNT + 32, Shape<QF, KF, HD, RH>::CTAS) paged_attn_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                                       const __grid_constant__ CUtensorMap tmV,
                                                                                       const __grid_constant__ PagedAttnArgs a, int box,
                                                                                       int order) {
  using S = Shape<QF, KF, HD, RH>;
  using Cursor = AttnCursor<typename S::Item>;
  constexpr int R = S::R, C = S::C, KT = S::KT, NO = HD / 8, KS = HD / 16, NS = S::NS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ AttnStart start;
  __shared__ __align__(8) uint64_t full[NS], empty[NS];
  __shared__ uint32_t dead_keys[NS];  // 8-key groups of a stage whose page does not exist
  __shared__ volatile uint32_t tries;  // of a wait; 0: one gave up
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (sbase - smem_u32(smem_raw));
  const uint32_t qbase = sbase + NS * S::STAGE;
  float* const wst = reinterpret_cast<float*>(smem + NS * S::STAGE + S::QBYTES);  // [warp][row][HD + 2]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3, mi = lane >> 3;
  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tries = a.tries;
  }
  grid_dep_enter();
  attn_find_start<typename S::Item, kNT + 32>(a.line, &start);
  if (tid == 0) a.parts[blockIdx.x].pieces = 0;  // no divided item yet
  int left;
  Cursor cu = Cursor::at(a.line, start, &left);
  if (left == 0) return;

  if (warp == 4) {
    // ---- producer: lane i looks up the page of keys 8i..8i+7 of a tile, the
    // lanes at the boxes' starts copy them.  Pages that do not exist are
    // outside the map and arrive as zeros.
    int kt = cu.kt, end = cu.kt + cu.tiles(left);  // of the piece
    auto page_of = [&]() {
      const int kk = kt * C + 8 * lane;
      return lane < C / 8 && kk < cu.len ? a.p.block_tables[(long)cu.b * a.p.table_ld + (kk >> a.shift)] : -1;
    };
    int page = page_of(), st = 0, u = 0;
    uint32_t par = 0;
#pragma unroll 1
    for (bool more = true; more && tries; u++) {
      const int kk = kt * C + 8 * lane, h = cu.h;
      const bool none = (unsigned)page >= (unsigned)a.p.kv.n_pages;
      const uint32_t dead = __ballot_sync(0xffffffffu, lane < C / 8 && kk < cu.len && none);
      const int mine = none ? a.p.kv.n_pages : page;
      if (++kt == end) {
        left = cu.behind(left, end - cu.kt);
        more = left > 0;
        if (more) {
          cu = Cursor::next(a.line, cu);
          kt = 0;
          end = cu.tiles(left);
        }
      }
      if (more) page = page_of();  // of the next tile, over the wait
      if (u >= NS) mbar_wait_or(&empty[st], par ^ 1, &tries);
      if (lane == 0) {
        dead_keys[st] = dead;
        mbar_expect_tx(&full[st], S::STAGE);
      }
      __syncwarp();
      if (lane < C / 8 && (8 * lane & (box - 1)) == 0) {
        const uint32_t dst = sbase + st * S::STAGE + (uint32_t)lane * 1024u;
        const int slot = kk & (a.p.kv.page_size - 1);
#pragma unroll 1
        for (int b = 0; b < S::NB; b++) {
          copy_box(dst + b * C * 128, &tmK, order, b * (128 / S::ES), slot, h, mine, &full[st]);
          copy_box(dst + S::TILE + b * C * 128, &tmV, order, b * (128 / S::ES), slot, h, mine, &full[st]);
        }
      }
      if (++st == NS) {
        st = 0;
        par ^= 1;
      }
    }
    // copies in flight land before the block may leave, whoever gave up
    for (int w = max(0, u - NS); w < u; w++) mbar_wait(&full[w % NS], (uint32_t)(w / NS) & 1);
    return;
  }
  auto sync_rows = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };  // the four computing warps

  auto q_addr = [&](int term, int row, int chunk) {  // 16-byte chunk of a query row, swizzled
    return qbase + (uint32_t)(term * S::RQ + row) * (HD * 2) + (uint32_t)((chunk & ~7) | ((chunk ^ row) & 7)) * 16u;
  };
  // 16-byte chunk of a key's row in a tile
  auto sw = [](int key, int chunk) { return (uint32_t)(chunk >> 3) * (C * 128) + (uint32_t)key * 128 + (uint32_t)((chunk ^ key) & 7) * 16u; };
  const float c2 = a.c2;
  uint32_t qr[S::QREG ? KS : 1][S::NQ][2 * RH];  // QREG: fragments of the item's queries
  float o[NO][4], m2[2], l2[2];
  int buf = 0;
  uint32_t par = 0;
#pragma unroll 1
  while (true) {
    // ---- a piece: tiles cu.kt .. end of an item
    const int end = cu.kt + cu.tiles(left);
    const int row_base = cu.m * R;  // first packed row of the item
    const int nrows = cu.rows(a.line, R);
    const int pos0 = cu.pos0();
    // its queries as bf16 terms; rows behind nrows are zero (what read the
    // item's before has synchronised since)
    constexpr int CH = HD / 8;
    for (int i = tid; i < S::RQ * CH; i += kNT) {
      const int r = i / CH, ch = i % CH;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = 0.0f;
      if (r < nrows) {
        const int pr = row_base + r;
        const long at = (long)(cu.r0 + pr / a.group) * a.p.q_ld + (long)(cu.h * a.group + pr % a.group) * HD + ch * 8;
        if (QF) {
          const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.p.q) + at);
          const float4 y = *reinterpret_cast<const float4*>(static_cast<const float*>(a.p.q) + at + 4);
          v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.p.q) + at);
          v[0] = bf_lo(x.x); v[1] = bf_hi(x.x); v[2] = bf_lo(x.y); v[3] = bf_hi(x.y);
          v[4] = bf_lo(x.z); v[5] = bf_hi(x.z); v[6] = bf_lo(x.w); v[7] = bf_hi(x.w);
        }
      }
      uint32_t t[4][3];
#pragma unroll
      for (int j = 0; j < 4; j++) split_bf2<S::NQ>(v[2 * j], v[2 * j + 1], t[j]);
#pragma unroll
      for (int k = 0; k < S::NQ; k++)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(q_addr(k, r, ch)), "r"(t[0][k]), "r"(t[1][k]),
                     "r"(t[2][k]), "r"(t[3][k])
                     : "memory");
    }
#pragma unroll
    for (int t = 0; t < NO; t++) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.0f;
    m2[0] = m2[1] = -INFINITY;
    l2[0] = l2[1] = 0.0f;
    sync_rows();
    if (S::QREG) {
#pragma unroll
      for (int ks = 0; ks < KS; ks++)
#pragma unroll
        for (int k = 0; k < S::NQ; k++) {
          uint32_t t[4];
          ldsm4(q_addr(k, lane & 15, 2 * ks + (lane >> 4)), t);
#pragma unroll
          for (int i = 0; i < 2 * RH; i++) qr[S::QREG ? ks : 0][k][i] = t[RH == 2 ? i : 2 * i];  // rows 8..15 (t[1], t[3]) are zero when RH = 1
        }
    }
    const int wkey = warp * (C / 4);  // the warp's keys
    // positions of the thread's two rows; rows behind the tile see nothing (their queries are zero, their states unused)
    int pr[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = gq + 8 * e;
      pr[e] = r < nrows ? pos0 + (row_base + r) / a.group : -1;
    }
    const int plast = pos0 + (row_base + nrows - 1) / a.group, pfirst = pos0 + row_base / a.group;
#pragma unroll 1
    for (int kt = cu.kt; kt < end; kt++) {
      const int key0 = kt * C + wkey;
      mbar_wait_or(&full[buf], par, &tries);
      if (key0 <= plast) {
        const uint32_t kt_s = sbase + buf * S::STAGE, vt_s = kt_s + S::TILE;
        const uint8_t* const kt_p = smem + buf * S::STAGE;
        const bool tail = key0 + 8 * KT > cu.len;  // slots behind the length: their values may be anything, and 0 * NaN is NaN
        if (!KF && tail) {
          for (int i = lane; i < 8 * KT * (HD / 8); i += 32) {
            const int key = wkey + i / (HD / 8);
            if (kt * C + key >= cu.len)
              *reinterpret_cast<uint4*>(smem + buf * S::STAGE + S::TILE + sw(key, i % (HD / 8))) = make_uint4(0u, 0u, 0u, 0u);
          }
          __syncwarp();
          fence_async();  // before the next copy into the stage
        }
        // The tensor core cuts what it adds to the accumulator's precision, so
        // the small products of a float32 call (all but the leading terms') are
        // summed apart and added once.
        float s[KT][4], lo[QF ? KT : 1][4];
#pragma unroll
        for (int j = 0; j < KT; j++) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < (QF ? KT : 1); j++) lo[j][0] = lo[j][1] = lo[j][2] = lo[j][3] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
          uint32_t qa[S::NQ][4];
#pragma unroll
          for (int k = 0; k < S::NQ; k++) {
            if (S::QREG) {
              const uint32_t* q = qr[S::QREG ? ks : 0][k];
              qa[k][0] = q[0];
              qa[k][1] = RH == 2 ? q[1] : 0u;
              qa[k][2] = q[RH];
              qa[k][3] = RH == 2 ? q[3 % (2 * RH)] : 0u;
            } else {
              ldsm4(q_addr(k, lane & 15, 2 * ks + (lane >> 4)), qa[k]);
            }
          }
          if (KF) {
#pragma unroll
            for (int j = 0; j < KT; j++) {
              const int key = wkey + 8 * j + gq, ch = 4 * ks + (tq >> 1);
              const float2 x = *reinterpret_cast<const float2*>(kt_p + sw(key, ch) + (tq & 1) * 8);
              const float2 y = *reinterpret_cast<const float2*>(kt_p + sw(key, ch + 2) + (tq & 1) * 8);
              uint32_t b0[3], b1[3];
              split_bf2<3>(x.x, x.y, b0);
              split_bf2<3>(y.x, y.y, b1);
              // products of terms whose orders add up to less than 2^-24 of the whole are left out
#pragma unroll
              for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                for (int k = 0; k <= sum; k++) mma_16816(sum ? lo[QF ? j : 0] : s[j], qa[QF ? k : 0], b0[sum - k], b1[sum - k]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < KT; j += 2) {
              // matrices: (keys 0-7, dims lo), (keys 0-7, dims hi), (keys 8-15, lo), (keys 8-15, hi)
              uint32_t kb[4];
              ldsm4(kt_s + sw(wkey + 8 * j + 8 * (mi >> 1) + (lane & 7), 2 * ks + (mi & 1)), kb);
#pragma unroll
              for (int k = S::NQ - 1; k >= 0; k--) {
                mma_16816(k ? lo[QF ? j : 0] : s[j], qa[k], kb[0], kb[1]);
                mma_16816(k ? lo[QF ? j + 1 : 0] : s[j + 1], qa[k], kb[2], kb[3]);
              }
            }
          }
        }
        if (QF) {
#pragma unroll
          for (int j = 0; j < KT; j++)
#pragma unroll
            for (int e = 0; e < 2 * RH; e++) s[j][e] += lo[QF ? j : 0][e];
        }
        // causal mask and missing pages; a tile that every row sees whole needs none
        const uint32_t gone = (dead_keys[buf] >> (wkey >> 3)) & ((1u << KT) - 1);
        if (key0 + 8 * KT - 1 > pfirst || gone) {
#pragma unroll
          for (int j = 0; j < KT; j++)
#pragma unroll
            for (int e = 0; e < 2 * RH; e++)
              if (key0 + 8 * j + 2 * tq + (e & 1) > pr[e >> 1] || ((gone >> j) & 1)) s[j][e] = -INFINITY;
        }
        float f[2] = {0.0f, 0.0f}, mm[2];
#pragma unroll
        for (int e = 0; e < RH; e++) {
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < KT; j++) mx = fmaxf(mx, fmaxf(s[j][2 * e], s[j][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m2[e], mx);
          mm[e] = mn == -INFINITY ? 0.0f : mn;
          f[e] = exp2_fast(attn_arg(m2[e], mm[e], c2));
          m2[e] = mn;
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < KT; j++) {
            s[j][2 * e] = exp2_fast(attn_arg(s[j][2 * e], mm[e], c2));
            s[j][2 * e + 1] = exp2_fast(attn_arg(s[j][2 * e + 1], mm[e], c2));
            sum += s[j][2 * e] + s[j][2 * e + 1];
          }
          l2[e] = l2[e] * f[e] + sum;  // this thread's share of the row sum
        }
#pragma unroll
        for (int t = 0; t < NO; t++) {
          o[t][0] *= f[0];
          o[t][1] *= f[0];
          if (RH == 2) {
            o[t][2] *= f[1];
            o[t][3] *= f[1];
          }
        }
#pragma unroll
        for (int j = 0; j < KT; j += 2) {
          uint32_t pa[S::NP][4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            uint32_t t[S::NP] = {};
            if (RH == 2 || (i & 1) == 0) split_bf2<S::NP>(s[j + (i >> 1)][2 * (i & 1)], s[j + (i >> 1)][2 * (i & 1) + 1], t);
#pragma unroll
            for (int k = 0; k < S::NP; k++) pa[k][i] = t[k];
          }
          // float32 calls: 16 keys at a time in an accumulator of their own,
          // small products first, added to the output in float32
          if (KF) {
#pragma unroll
            for (int t = 0; t < NO; t++) {
              const int key = wkey + 8 * j + 2 * tq;
              float v[4];
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const int kk = key + (i & 1) + 8 * (i >> 1);
                v[i] = *reinterpret_cast<const float*>(kt_p + S::TILE + sw(kk, 2 * t + (gq >> 2)) + (gq & 3) * 4);
                if (tail && kt * C + kk >= cu.len) v[i] = 0.0f;
              }
              uint32_t b0[3], b1[3];
              split_bf2<3>(v[0], v[1], b0);
              split_bf2<3>(v[2], v[3], b1);
              float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                for (int k = 0; k <= sum; k++) mma_16816(x, pa[QF ? k : 0], b0[sum - k], b1[sum - k]);
#pragma unroll
              for (int e = 0; e < 2 * RH; e++) o[t][e] += x[e];
            }
          } else {
#pragma unroll
            for (int t = 0; t < NO; t += 2) {
              // matrices: (keys 0-7, dims 8t..), (keys 8-15, 8t..), (keys 0-7, 8t+8..), (keys 8-15, 8t+8..)
              uint32_t vb[4];
              ldsm4_t(vt_s + sw(wkey + 8 * j + 8 * (mi & 1) + (lane & 7), t + (mi >> 1)), vb);
              if (QF) {
                float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = S::NP - 1; k >= 0; k--) {
                  mma_16816(x, pa[k], vb[0], vb[1]);
                  mma_16816(y, pa[k], vb[2], vb[3]);
                }
#pragma unroll
                for (int e = 0; e < 2 * RH; e++) {
                  o[t][e] += x[e];
                  o[t + 1][e] += y[e];
                }
              } else {
                mma_16816(o[t], pa[0], vb[0], vb[1]);
                mma_16816(o[t + 1], pa[0], vb[2], vb[3]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0 && !(a.keep_cta0 && blockIdx.x == 0)) mbar_arrive(&empty[buf]);  // the stage is consumed
      if (++buf == NS) {
        buf = 0;
        par ^= 1;
      }
    }

    // the piece is done: to the output when it is the whole item, else to the workspace
    const bool ends = end == cu.nt, whole = ends && cu.kt == 0;
    // a piece from the item's start goes to the CTA's second place, one that enters the CTA to its first
    const int slot = 2 * blockIdx.x + (cu.kt == 0 ? 1 : 0);
    float2* const pml = a.ml + (long)slot * a.tile_rows;
    float* const part = a.acc + (long)slot * a.tile_rows * HD;
    if (!ends && cu.kt == 0 && tid == 0) {
      AttnPart d;
      d.pieces = attn_pieces<typename S::Item>(a.line, start, cu.nt - end - 1);
      d.row0 = cu.r0; d.packed0 = row_base; d.rows = nrows; d.h = cu.h;
      a.parts[blockIdx.x] = d;
    }
#pragma unroll
    for (int e = 0; e < RH; e++) {
      l2[e] += __shfl_xor_sync(0xffffffffu, l2[e], 1);
      l2[e] += __shfl_xor_sync(0xffffffffu, l2[e], 2);
    }
    // the four warps' states, merged in warp order
#pragma unroll
    for (int e = 0; e < RH; e++) {
      const int r = gq + 8 * e;
      if (r >= nrows) continue;
      float* w = wst + (warp * a.rows_used + r) * (HD + 2);
      if (tq == 0) *reinterpret_cast<float2*>(w) = make_float2(m2[e], l2[e]);
#pragma unroll
      for (int t = 0; t < NO; t++)
        *reinterpret_cast<float2*>(w + 2 + 8 * t + 2 * tq) = make_float2(o[t][2 * e], o[t][2 * e + 1]);
    }
    sync_rows();
    const bool lost = tries == 0;  // a wait gave up: what was computed since may be anything
    for (int i = tid; i < nrows * (HD / 2); i += kNT) {
      const int r = i / (HD / 2), d = 2 * (i % (HD / 2));
      const float* w = wst + r * (HD + 2);
      const int ws = a.rows_used * (HD + 2);
      float M = -INFINITY, L = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; k++) M = fmaxf(M, w[k * ws]);
      const float mz = M == -INFINITY ? 0.0f : M;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float g = exp2_fast(attn_arg(w[k * ws], mz, c2));
        L = fmaf(w[k * ws + 1], g, L);
        x = fmaf(w[k * ws + 2 + d], g, x);
        y = fmaf(w[k * ws + 3 + d], g, y);
      }
      if (lost) x = y = __int_as_float(0x7fffffff);
      if (whole) {
        const int pk = row_base + r;
        const long at = (long)(cu.r0 + pk / a.group) * a.p.out_ld + (long)(cu.h * a.group + pk % a.group) * HD + d;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        if (QF)
          *reinterpret_cast<float2*>(static_cast<float*>(a.p.out) + at) = make_float2(x * inv, y * inv);
        else
          *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.p.out) + at) = pack_bf2(x * inv, y * inv);
      } else {
        if (d == 0) pml[r] = make_float2(M, L);
        *reinterpret_cast<float2*>(part + (long)r * HD + d) = make_float2(x, y);
      }
    }
    left = cu.behind(left, end - cu.kt);
    if (left == 0) break;
    cu = Cursor::next(a.line, cu);
  }
}

// Merges the pieces of the items that cuts divide: the blocks (c, *) take the
// item that leaves CTA c, if there is one.  HD/8 lanes hold a row (eight
// columns each: four need twice the blocks, which then run in two waves).  Few
// pieces (chunks; the usual case): each group of lanes takes a row of its own
// and walks its pieces.  Many (one long request): the block takes a row at a
// time, its groups share the pieces, and their states merge in shared memory
// in group order.
constexpr int kJoinThreads = 256;
template <bool BF, int HD>
__global__ void __launch_bounds__(kJoinThreads) paged_attn_join_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int COLS = HD / 8, G = kJoinThreads / COLS, FEW = 8;
  __shared__ float4 gv[G][2 * COLS];
  __shared__ float2 gml[G];
  const int tid = threadIdx.x, c = blockIdx.x, col = tid % COLS, grp = tid / COLS;
  grid_dep_enter();
  const AttnPart d = a.parts[c];
  if (d.pieces == 0) return;
  const bool shared_row = d.pieces > FEW;
  const int i0 = shared_row ? grp : 0, di = shared_row ? G : 1;
  const int rows_at_once = shared_row ? 1 : G;
  for (int base = blockIdx.y * rows_at_once; base < d.rows; base += gridDim.y * rows_at_once) {
    const int r = base + (shared_row ? 0 : grp);
    const bool on = r < d.rows;
    float m = -INFINITY, l = 0.0f, v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.0f;
    // the state (m2, l2, x, y) joins (m, l, v)
    auto add = [&](float m2, float l2, const float4& x, const float4& y) {
      const float mn = fmaxf(m, m2), mz = mn == -INFINITY ? 0.0f : mn;
      const float f = exp2_fast(attn_arg(m, mz, a.c2)), g = exp2_fast(attn_arg(m2, mz, a.c2));
      m = mn;
      l = fmaf(l2, g, l * f);
      const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = fmaf(w[e], g, v[e] * f);
    };
    if (on) {
#pragma unroll 4
      for (int i = i0; i < d.pieces; i += di) {
        const long at = (long)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * a.tile_rows + r;
        const float2 ml = a.ml[at];
        const float4* w = reinterpret_cast<const float4*>(a.acc + at * HD + 8 * col);
        add(ml.x, ml.y, w[0], w[1]);
      }
    }
    if (shared_row) {
      gv[grp][2 * col] = make_float4(v[0], v[1], v[2], v[3]);
      gv[grp][2 * col + 1] = make_float4(v[4], v[5], v[6], v[7]);
      if (col == 0) gml[grp] = make_float2(m, l);
      __syncthreads();
      if (tid < HD) {  // a column a thread
        float M = -INFINITY, x = 0.0f;
#pragma unroll
        for (int k = 0; k < G; k++) M = fmaxf(M, gml[k].x);
        if (M == -INFINITY) M = 0.0f;
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < G; k++) {
          const float g = exp2_fast(attn_arg(gml[k].x, M, a.c2));
          l = fmaf(gml[k].y, g, l);
          x = fmaf(reinterpret_cast<const float*>(gv[k])[tid], g, x);
        }
        const int pk = d.packed0 + r;
        const long at = (long)(d.row0 + pk / a.group) * a.p.out_ld + (long)(d.h * a.group + pk % a.group) * HD + tid;
        x *= l == 0.0f ? 0.0f : 1.0f / l;
        if (BF)
          static_cast<uint16_t*>(a.p.out)[at] = (uint16_t)pack_bf2(x, 0.0f);
        else
          static_cast<float*>(a.p.out)[at] = x;
      }
      __syncthreads();
    } else if (on) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int pk = d.packed0 + r;
      const long at = (long)(d.row0 + pk / a.group) * a.p.out_ld + (long)(d.h * a.group + pk % a.group) * HD + 8 * col;
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] *= inv;
      if (BF) {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.p.out) + at) =
            make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
      } else {
        float4* out = reinterpret_cast<float4*>(static_cast<float*>(a.p.out) + at);
        out[0] = make_float4(v[0], v[1], v[2], v[3]);
        out[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
  }
}

template <bool QF, bool KF, int HD, int RH>
cudaError_t launch_attn(const PagedAttnArgs& a, cudaStream_t s) {
  using S = Shape<QF, KF, HD, RH>;
  static SmemOptIn opt;
  const size_t smem = S::smem(a.rows_used);
  CTTS_LK(opt.ensure(reinterpret_cast<const void*>(paged_attn_kernel<QF, KF, HD, RH>), smem));
  CUtensorMap mk, mv;
  const int box = std::min(a.p.kv.page_size, (int)S::C);
  int order = 0;
  if (!paged_pool_map(&mk, a.p.kv.k, a.p.kv, box, &order) || !paged_pool_map(&mv, a.p.kv.v, a.p.kv, box, &order)) return cudaErrorInvalidValue;
  return launch_k(paged_attn_kernel<QF, KF, HD, RH>, dim3(a.line.ctas), dim3(kNT + 32), smem, s, mk, mv, a, box, order);
}

// f(QF, KF, HD, RH as integral constants) for short items of up to `rows`
// packed rows.
template <class F>
auto with_shape(const ctts_paged_attn& p, int rows, F f) {
  using T = std::true_type;
  using N = std::false_type;
  auto g = [&](auto q, auto k, auto hd) {
    return rows > 8 ? f(q, k, hd, std::integral_constant<int, 2>{}) : f(q, k, hd, std::integral_constant<int, 1>{});
  };
  auto h = [&](auto hd) {
    if (p.kv.dtype == CTTS_F32) return g(T{}, T{}, hd);
    return p.q_dtype == CTTS_F32 ? g(T{}, N{}, hd) : g(N{}, N{}, hd);
  };
  return p.kv.head_dim == 128 ? h(std::integral_constant<int, 128>{}) : h(std::integral_constant<int, 64>{});
}

// Items of up to 16 packed rows run on this file's kernel, calls with longer
// ones on the tcgen05 kernel (paged_attn_tc.cu) -- their short requests too: a
// tile of 128 rows costs a short item as much as a long one, yet in bf16 two
// launches after one another took longer (43 decodes and 5 chunks of 200 to
// 512: 40 us against 35, and 30 since such items share a CTA's two sub-tiles).
// With float32 queries they do not share, and two launches were not tried: 30
// single tokens of 2000 to 32000 take 62 us there on this file's kernel, 234
// beside a chunk of 20 rows (over a float32 cache 130 and 319; bf16 62 and 73).
bool is_short(const ctts_paged_attn& p) { return (long)p.max_new * (p.n_heads / p.kv.n_kv_heads) <= 16; }
int rows_used_of(const ctts_paged_attn& p) { return std::max(1, p.max_new * (p.n_heads / p.kv.n_kv_heads)); }

}  // namespace

bool paged_pool_map(CUtensorMap* m, const void* base, const ctts_paged_kv& kv, int box, int* order) {
  auto fn = encode_fn();
  if (!fn) return false;
  const int es = kv.dtype == CTTS_F32 ? 4 : 2;
  struct Dim {
    int64_t stride;
    int size, box, what;
  } d[3] = {{kv.token_stride, kv.page_size, box, 0}, {kv.head_stride, kv.n_kv_heads, 1, 1}, {kv.page_stride, kv.n_pages, 1, 2}};
  std::stable_sort(d, d + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim}, strides[3];
  cuuint32_t boxes[4] = {(cuuint32_t)(128 / es)}, estr[4] = {1, 1, 1, 1};
  *order = 0;
  for (int i = 0; i < 3; i++) {
    dims[i + 1] = (cuuint64_t)d[i].size;
    strides[i] = (cuuint64_t)d[i].stride * es;
    boxes[i + 1] = (cuuint32_t)d[i].box;
    *order |= d[i].what << (2 * i);
  }
  return fn(m, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, boxes,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static PagedAttnPlan plan_for(const ctts_paged_attn& p, int sms) {
  PagedAttnPlan pl;
  if (is_short(p)) {
    const int rows = rows_used_of(p);
    with_shape(p, rows, [&](auto q, auto k, auto hd, auto rh) {
      constexpr bool QF = decltype(q)::value, KF = decltype(k)::value;
      constexpr int HD = decltype(hd)::value, RH = decltype(rh)::value;
      using S = Shape<QF, KF, HD, RH>;
      pl.ctas = sms * S::blocks(rows);
      pl.tile_rows = S::R;
      return 0;
    });
  } else {
    pl.ctas = sms;
    pl.tile_rows = paged_attn_tc_rows(p);
  }
  pl.ws_bytes = pl.ctas * (sizeof(AttnPart) + (size_t)2 * pl.tile_rows * (p.kv.head_dim + 2) * sizeof(float));
  return pl;
}

PagedAttnPlan paged_attn_plan(const ctts_paged_attn& p) { return plan_for(p, device_sms()); }

// Fewer rows can want more: short items of few rows leave an SM room for more
// blocks, each with partial states of its own.
size_t paged_attn_ws_bytes(const ctts_paged_attn& p) {
  const int sms = device_sms();
  ctts_paged_attn q = p;
  size_t most = plan_for(p, sms).ws_bytes;
  for (q.max_new = 0; q.max_new < p.max_new && is_short(q); q.max_new++) most = std::max(most, plan_for(q, sms).ws_bytes);
  return most;
}

cudaError_t launch_paged_attn(const ctts_paged_attn& p, cudaStream_t s) {
  if (p.rows == 0 || p.max_new == 0) return cudaSuccess;
  const PagedAttnPlan pl = paged_attn_plan(p);
  PagedAttnArgs a;
  a.p = p;
  a.group = p.n_heads / p.kv.n_kv_heads;
  while ((1 << a.shift) < p.kv.page_size) a.shift++;
  AttnLine& ln = a.line;
  ln.cu_rows = p.cu_rows;
  ln.seq_lens = p.seq_lens;
  ln.batch = p.batch;
  ln.rows = p.rows;
  ln.max_new = p.max_new;
  ln.max_len = p.max_pages * p.kv.page_size;
  ln.group = a.group;
  ln.n_kv = p.kv.n_kv_heads;
  ln.ctas = pl.ctas;
  a.tile_rows = pl.tile_rows;
  a.c2 = (float)((double)p.scale * 1.4426950408889634);
  a.keep_cta0 = g_fault_skip.load(std::memory_order_relaxed);
  if (const uint32_t n = g_fault_spin_limit.load(std::memory_order_relaxed)) a.tries = n;
  a.parts = static_cast<AttnPart*>(p.workspace);
  a.acc = reinterpret_cast<float*>(a.parts + pl.ctas);
  a.ml = reinterpret_cast<float2*>(a.acc + (size_t)2 * pl.ctas * pl.tile_rows * p.kv.head_dim);
  if (is_short(p)) {
    a.rows_used = rows_used_of(p);
    CTTS_LK(with_shape(p, a.rows_used, [&](auto q, auto k, auto hd, auto rh) {
      return launch_attn<decltype(q)::value, decltype(k)::value, decltype(hd)::value, decltype(rh)::value>(a, s);
    }));
  } else {
    CTTS_LK(launch_paged_attn_tc(a, s));
  }
  const dim3 grid(pl.ctas, is_short(p) ? std::min(a.rows_used, 4) : p.kv.head_dim / 8), block(kJoinThreads);
  const bool bf = p.q_dtype == CTTS_BF16;
  if (p.kv.head_dim == 64)
    return bf ? launch_k(paged_attn_join_kernel<true, 64>, grid, block, 0, s, a) : launch_k(paged_attn_join_kernel<false, 64>, grid, block, 0, s, a);
  return bf ? launch_k(paged_attn_join_kernel<true, 128>, grid, block, 0, s, a) : launch_k(paged_attn_join_kernel<false, 128>, grid, block, 0, s, a);
}

}  // namespace ctts
