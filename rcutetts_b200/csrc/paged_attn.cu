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

constexpr int kKeys = 64;  // keys per tile
constexpr int kNT = 128;   // threads

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
// 16 bytes to shared memory, zeros when `bytes` is 0
CTTS_DEV void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
CTTS_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
CTTS_DEV void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One kernel shape.  CHUNK = false: 16 packed rows per item (single tokens and
// short runs), the four warps share the rows and split each key tile, 16 keys
// each, with their own softmax states.  CHUNK = true: 64 packed rows, 16 per
// warp, every warp takes all keys.
template <bool QF, bool KF, int HD, bool CHUNK>
struct Shape {
  static constexpr int R = CHUNK ? 64 : 16;
  // bf16 terms of a float32 operand (queries and softmax weights; keys and
  // values of a float32 cache): 24 bits, so a float32 call keeps float32
  static constexpr int NQ = QF ? 3 : 1;
  static constexpr int NP = QF ? 3 : 1;
  static constexpr int ES = KF ? 4 : 2;
  static constexpr int ROWB = HD * ES;
  // float32 rows are padded so that the fragment reads (8 keys x 8 bytes of K,
  // 8 keys x 8 words of V) fall in distinct banks; bf16 rows are swizzled
  static constexpr int KROW = ROWB + (KF ? 32 : 0), VROW = ROWB + (KF ? 16 : 0);
  static constexpr int STAGE = kKeys * (KROW + VROW);
  // stages: 48 KB in flight per CTA or more
  static constexpr int NS = STAGE <= 16384 ? 4 : (STAGE <= 36864 ? 3 : 2);
  static constexpr int QBYTES = NQ * R * HD * 2;
  static constexpr int KT = CHUNK ? 8 : 2;  // 8-key column tiles per warp and key tile
  static size_t smem(int rows_used) {
    return (size_t)NS * STAGE + QBYTES + (CHUNK ? 0 : (size_t)4 * rows_used * (HD + 2) * 4);
  }
};

template <bool QF, bool KF, int HD, bool CHUNK>
__global__ void __launch_bounds__(kNT) paged_attn_kernel(const PagedAttnArgs a) {
  using S = Shape<QF, KF, HD, CHUNK>;
  constexpr int R = S::R, KT = S::KT, NO = HD / 8, KS = HD / 16, NS = S::NS;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ AttnStart start;
  __shared__ uint8_t dead[NS][8];  // 8-key groups of a stage whose page does not exist
  const uint32_t sbase = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  const uint32_t qbase = sbase + NS * S::STAGE;
  float* const wst = reinterpret_cast<float*>(smem + NS * S::STAGE + S::QBYTES);  // [warp][row][HD + 2]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, tq = lane & 3, mi = lane >> 3;
  grid_dep_enter();

  attn_find_start<R, kKeys, kNT>(a, &start);
  const long units = start.units;
  if (tid == 0) a.parts[blockIdx.x].pieces = 0;  // no divided item yet
  if (units == 0) return;
  AttnCursor ld = AttnCursor::at<R, kKeys>(a, start), cu = ld;
  long to_load = units;

  auto q_addr = [&](int term, int row, int chunk) {  // 16-byte chunk of a query row, swizzled
    return qbase + (uint32_t)(term * R + row) * (HD * 2) + (uint32_t)((chunk & ~7) | ((chunk ^ row) & 7)) * 16u;
  };
  auto sw = [&](int key, int chunk) { return (uint32_t)key * (HD * 2) + (uint32_t)((chunk & ~7) | ((chunk ^ key) & 7)) * 16u; };

  int ld_buf = 0;
  auto issue = [&]() {  // the next unit's K and V rows into stage ld_buf (an empty group when there is none)
    if (to_load > 0) {
      constexpr int CH = S::ROWB / 16;  // chunks per row
      const int* tab = a.p.block_tables + (long)ld.b * a.p.table_ld;
      const int key0 = ld.kt * kKeys;
      const uint32_t kd = sbase + ld_buf * S::STAGE, vd = kd + kKeys * S::KROW;
#pragma unroll
      for (int i = 0; i < kKeys * CH / kNT; i++) {
        const int c = tid + i * kNT, key = c / CH, ch = c % CH;
        const int kk = key0 + key;
        long off = 0;
        bool ok = kk < ld.len;
        if (ok) {
          const int page = tab[kk >> a.shift];
          ok = (unsigned)page < (unsigned)a.p.kv.n_pages;
          if (ok)
            off = ((long)page * a.p.kv.page_stride + (long)(kk & (a.p.kv.page_size - 1)) * a.p.kv.token_stride +
                   (long)ld.h * a.p.kv.head_stride) * S::ES + ch * 16;
        }
        const uint32_t dk = KF ? (uint32_t)key * S::KROW + ch * 16u : sw(key, ch);
        const uint32_t dv = KF ? (uint32_t)key * S::VROW + ch * 16u : dk;
        cp_async16(kd + dk, static_cast<const uint8_t*>(a.p.kv.k) + off, ok ? 16 : 0);
        cp_async16(vd + dv, static_cast<const uint8_t*>(a.p.kv.v) + off, ok ? 16 : 0);
      }
      if (tid < 8) {
        const int kk = key0 + tid * 8;
        dead[ld_buf][tid] = kk < ld.len && (unsigned)tab[kk >> a.shift] >= (unsigned)a.p.kv.n_pages;
      }
      if (--to_load > 0) ld.next<R, kKeys>(a);
    }
    cp_commit();
    ld_buf = ld_buf + 1 == NS ? 0 : ld_buf + 1;
  };
#pragma unroll
  for (int i = 0; i < NS - 1; i++) issue();

  const float c2 = a.c2_hi;
  float o[NO][4], m2[2], l2[2];
  bool fresh = true;  // the unit begins a piece
  int unit0_kt = 0;   // the piece's first key tile
  int buf = 0;
  for (long u = 0; u < units; u++) {
    cp_wait<NS - 2>();
    __syncthreads();  // the stage has landed for everyone; the one before is consumed
    issue();
    const int row_base = cu.m * R;               // first packed row of the tile
    const int nrows = min(R, cu.nn * a.group - row_base);
    const int pos0 = cu.len - cu.cnt;            // position of the request's first new row
    if (fresh) {
      unit0_kt = cu.kt;
      // queries of the tile as bf16 terms; rows behind nrows are zero
      constexpr int CH = HD / 8;
      for (int i = tid; i < R * CH; i += kNT) {
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
      __syncthreads();
      fresh = false;
    }
    const int wrow = CHUNK ? warp * 16 : 0;      // the warp's rows and keys
    const int wkey = CHUNK ? 0 : warp * 16;
    const int key0 = cu.kt * kKeys + wkey;
    // positions of the thread's two rows; rows behind the tile see nothing (their queries are zero, their states unused)
    int pr[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = wrow + gq + 8 * e;
      pr[e] = r < nrows ? pos0 + (row_base + r) / a.group : -1;
    }
    const int plast = wrow < nrows ? pos0 + (row_base + min(nrows, wrow + 16) - 1) / a.group : -1;
    if (key0 <= plast) {
      const uint32_t kt_s = sbase + buf * S::STAGE, vt_s = kt_s + kKeys * S::KROW;
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
        for (int k = 0; k < S::NQ; k++) ldsm4(q_addr(k, wrow + (lane & 15), 2 * ks + (lane >> 4)), qa[k]);
        if (KF) {
#pragma unroll
          for (int j = 0; j < KT; j++) {
            const uint8_t* kp = smem + buf * S::STAGE + (wkey + 8 * j + gq) * S::KROW + (ks * 16 + 2 * tq) * 4;
            const float2 x = *reinterpret_cast<const float2*>(kp), y = *reinterpret_cast<const float2*>(kp + 32);
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
          for (int e = 0; e < 4; e++) s[j][e] += lo[QF ? j : 0][e];
      }
      // causal mask and missing pages; a tile that every row sees whole needs none
      const int pfirst = pos0 + (row_base + wrow) / a.group;
      uint32_t gone = 0;
#pragma unroll
      for (int j = 0; j < KT; j++) gone |= (uint32_t)(dead[buf][(wkey >> 3) + j] != 0) << j;
      if (key0 + 8 * KT - 1 > pfirst || gone) {
#pragma unroll
        for (int j = 0; j < KT; j++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (key0 + 8 * j + 2 * tq + (e & 1) > pr[e >> 1] || ((gone >> j) & 1)) s[j][e] = -INFINITY;
      }
      float f[2], mm[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < KT; j++) mx = fmaxf(mx, fmaxf(s[j][2 * e], s[j][2 * e + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m2[e], mx * c2);
        mm[e] = mn == -INFINITY ? 0.0f : mn;
        f[e] = exp2_fast(m2[e] - mm[e]);
        m2[e] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < KT; j++) {
          s[j][2 * e] = exp2_fast(attn_arg<QF>(a, s[j][2 * e], mm[e]));
          s[j][2 * e + 1] = exp2_fast(attn_arg<QF>(a, s[j][2 * e + 1], mm[e]));
          sum += s[j][2 * e] + s[j][2 * e + 1];
        }
        l2[e] = l2[e] * f[e] + sum;  // this thread's share of the row sum
      }
#pragma unroll
      for (int t = 0; t < NO; t++) {
        o[t][0] *= f[0];
        o[t][1] *= f[0];
        o[t][2] *= f[1];
        o[t][3] *= f[1];
      }
#pragma unroll
      for (int j = 0; j < KT; j += 2) {
        uint32_t pa[S::NP][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          uint32_t t[S::NP];
          split_bf2<S::NP>(s[j + (i >> 1)][2 * (i & 1)], s[j + (i >> 1)][2 * (i & 1) + 1], t);
#pragma unroll
          for (int k = 0; k < S::NP; k++) pa[k][i] = t[k];
        }
        // float32 calls: 16 keys at a time in an accumulator of their own,
        // small products first, added to the output in float32
        if (KF) {
#pragma unroll
          for (int t = 0; t < NO; t++) {
            const float* vp = reinterpret_cast<const float*>(smem + buf * S::STAGE + kKeys * S::KROW +
                                                             (wkey + 8 * j + 2 * tq) * S::VROW) + 8 * t + gq;
            constexpr int LD = S::VROW / 4;
            uint32_t b0[3], b1[3];
            split_bf2<3>(vp[0], vp[LD], b0);
            split_bf2<3>(vp[8 * LD], vp[9 * LD], b1);
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int sum = 2; sum >= 0; sum--)
#pragma unroll
              for (int k = 0; k <= sum; k++) mma_16816(x, pa[QF ? k : 0], b0[sum - k], b1[sum - k]);
#pragma unroll
            for (int e = 0; e < 4; e++) o[t][e] += x[e];
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
              for (int e = 0; e < 4; e++) {
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
    buf = buf + 1 == NS ? 0 : buf + 1;

    const bool ends = cu.kt + 1 == cu.nt;
    if (ends || u + 1 == units) {  // the piece is done: to the output when it is the whole item, else to the workspace
      const bool whole = ends && unit0_kt == 0;
      // a piece from the item's start goes to the CTA's second place, one that enters the CTA to its first
      const int slot = 2 * blockIdx.x + (unit0_kt == 0 ? 1 : 0);
      float2* const pml = a.ml + (long)slot * a.tile_rows;
      float* const part = a.acc + (long)slot * a.tile_rows * HD;
      if (!ends && unit0_kt == 0 && tid == 0) {
        AttnPart d;
        d.pieces = attn_pieces(a, start, cu.nt - 1 - cu.kt);
        d.row0 = cu.r0; d.packed0 = row_base; d.rows = nrows; d.h = cu.h;
        a.parts[blockIdx.x] = d;
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        l2[e] += __shfl_xor_sync(0xffffffffu, l2[e], 1);
        l2[e] += __shfl_xor_sync(0xffffffffu, l2[e], 2);
      }
      if (CHUNK) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int r = wrow + gq + 8 * e;
          if (r >= nrows) continue;
          if (whole) {
            const int pk = row_base + r;
            const long at = (long)(cu.r0 + pk / a.group) * a.p.out_ld + (long)(cu.h * a.group + pk % a.group) * HD + 2 * tq;
            const float inv = l2[e] == 0.0f ? 0.0f : 1.0f / l2[e];
#pragma unroll
            for (int t = 0; t < NO; t++) {
              const float x = o[t][2 * e] * inv, y = o[t][2 * e + 1] * inv;
              if (QF)
                *reinterpret_cast<float2*>(static_cast<float*>(a.p.out) + at + 8 * t) = make_float2(x, y);
              else
                *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.p.out) + at + 8 * t) = pack_bf2(x, y);
            }
          } else {
            if (tq == 0) pml[r] = make_float2(m2[e], l2[e]);
#pragma unroll
            for (int t = 0; t < NO; t++)
              *reinterpret_cast<float2*>(part + (long)r * HD + 8 * t + 2 * tq) = make_float2(o[t][2 * e], o[t][2 * e + 1]);
          }
        }
      } else {
        // the four warps' states, merged in warp order
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int r = gq + 8 * e;
          if (r >= nrows) continue;
          float* w = wst + (warp * a.rows_used + r) * (HD + 2);
          if (tq == 0) *reinterpret_cast<float2*>(w) = make_float2(m2[e], l2[e]);
#pragma unroll
          for (int t = 0; t < NO; t++)
            *reinterpret_cast<float2*>(w + 2 + 8 * t + 2 * tq) = make_float2(o[t][2 * e], o[t][2 * e + 1]);
        }
        __syncthreads();
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
            const float g = exp2_fast(w[k * ws] - mz);
            L = fmaf(w[k * ws + 1], g, L);
            x = fmaf(w[k * ws + 2 + d], g, x);
            y = fmaf(w[k * ws + 3 + d], g, y);
          }
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
      }
      fresh = true;
    }
    if (u + 1 < units) cu.next<R, kKeys>(a);
  }
}

// Merges the pieces of the items that cuts divide: the blocks (c, *) take the
// item that leaves CTA c, if there is one.  HD/4 lanes hold a row (four
// columns each).  Few pieces (chunks; the usual case): each group of lanes
// takes a row of its own and walks its pieces.  Many (one long request): the
// block takes a row at a time, its groups share the pieces, and their states
// merge in shared memory in group order.
constexpr int kJoinThreads = 256;
template <bool BF, int HD>
__global__ void __launch_bounds__(kJoinThreads) paged_attn_join_kernel(const PagedAttnArgs a) {
  constexpr int COLS = HD / 4, G = kJoinThreads / COLS, FEW = 8;
  __shared__ float4 gv[G][COLS];
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
    float m = -INFINITY, l = 0.0f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) {
#pragma unroll 4
      for (int i = i0; i < d.pieces; i += di) {
        const long at = (long)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * a.tile_rows + r;
        const float2 ml = a.ml[at];
        const float4 w = *reinterpret_cast<const float4*>(a.acc + at * HD + 4 * col);
        const float mn = fmaxf(m, ml.x), mz = mn == -INFINITY ? 0.0f : mn;
        const float f = exp2_fast(m - mz), g = exp2_fast(ml.x - mz);
        m = mn;
        l = fmaf(ml.y, g, l * f);
        v.x = fmaf(w.x, g, v.x * f);
        v.y = fmaf(w.y, g, v.y * f);
        v.z = fmaf(w.z, g, v.z * f);
        v.w = fmaf(w.w, g, v.w * f);
      }
    }
    if (shared_row) {
      gv[grp][col] = v;
      if (col == 0) gml[grp] = make_float2(m, l);
      __syncthreads();
      if (grp == 0) {
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < G; k++) M = fmaxf(M, gml[k].x);
        if (M == -INFINITY) M = 0.0f;
        l = 0.0f;
        v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < G; k++) {
          const float g = exp2_fast(gml[k].x - M);
          const float4 w = gv[k][col];
          l = fmaf(gml[k].y, g, l);
          v.x = fmaf(w.x, g, v.x);
          v.y = fmaf(w.y, g, v.y);
          v.z = fmaf(w.z, g, v.z);
          v.w = fmaf(w.w, g, v.w);
        }
      }
      __syncthreads();
    }
    if (on && (!shared_row || grp == 0)) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int pk = d.packed0 + r;
      const long at = (long)(d.row0 + pk / a.group) * a.p.out_ld + (long)(d.h * a.group + pk % a.group) * HD + 4 * col;
      if (BF)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.p.out) + at) = make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
      else
        *reinterpret_cast<float4*>(static_cast<float*>(a.p.out) + at) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
  }
}

template <bool QF, bool KF, int HD, bool CHUNK>
int attn_ctas(int rows_used) {
  using S = Shape<QF, KF, HD, CHUNK>;
  // shared memory per SM: 227 KB for blocks, 1 KB kept per block
  const int occ = std::max(1, std::min(4, (int)((227 * 1024) / (S::smem(rows_used) + 2048))));
  return device_sms() * occ;
}

template <bool QF, bool KF, int HD, bool CHUNK>
cudaError_t launch_attn(const PagedAttnArgs& a, cudaStream_t s) {
  using S = Shape<QF, KF, HD, CHUNK>;
  static SmemOptIn opt;
  const size_t smem = S::smem(a.rows_used);
  CTTS_LK(opt.ensure(reinterpret_cast<const void*>(paged_attn_kernel<QF, KF, HD, CHUNK>), smem));
  return launch_k(paged_attn_kernel<QF, KF, HD, CHUNK>, dim3(a.ctas), dim3(kNT), smem, s, a);
}

// The call's mma.sync shape: f(QF, KF, HD, CHUNK as integral constants)
template <class F>
auto with_shape(const ctts_paged_attn& p, F f) {
  const bool qf = p.q_dtype == CTTS_F32, kf = p.kv.dtype == CTTS_F32, wide = p.kv.head_dim == 128;
  // short runs share the key tile between the warps; beyond 16 packed rows
  // every warp has rows of its own
  const bool chunk = (long)p.max_new * (p.n_heads / p.kv.n_kv_heads) > 16;
  using T = std::true_type;
  using N = std::false_type;
  using H64 = std::integral_constant<int, 64>;
  using H128 = std::integral_constant<int, 128>;
  if (kf) {
    if (wide) return chunk ? f(T{}, T{}, H128{}, T{}) : f(T{}, T{}, H128{}, N{});
    return chunk ? f(T{}, T{}, H64{}, T{}) : f(T{}, T{}, H64{}, N{});
  }
  if (wide) return qf ? f(T{}, N{}, H128{}, N{}) : f(N{}, N{}, H128{}, N{});
  return qf ? f(T{}, N{}, H64{}, N{}) : f(N{}, N{}, H64{}, N{});
}

// Chunks over a bf16 cache run on tcgen05 (paged_attn_tc.cu).
bool use_tc(const ctts_paged_attn& p) {
  return p.kv.dtype == CTTS_BF16 && (long)p.max_new * (p.n_heads / p.kv.n_kv_heads) > 16;
}

int rows_used_of(const ctts_paged_attn& p) {
  return (int)std::min(16L, std::max(1L, (long)p.max_new * (p.n_heads / p.kv.n_kv_heads)));
}

}  // namespace

PagedAttnPlan paged_attn_plan(const ctts_paged_attn& p) {
  PagedAttnPlan pl;
  if (use_tc(p)) {
    const PagedAttnTc t = paged_attn_tc_plan(p);
    pl.ctas = t.ctas;
    pl.tile_rows = t.tile_rows;
  } else with_shape(p, [&](auto q, auto k, auto hd, auto ch) {
    constexpr bool QF = decltype(q)::value, KF = decltype(k)::value, CH = decltype(ch)::value;
    constexpr int HD = decltype(hd)::value;
    pl.ctas = attn_ctas<QF, KF, HD, CH>(rows_used_of(p));
    pl.tile_rows = Shape<QF, KF, HD, CH>::R;
    return 0;
  });
  pl.ws_bytes = pl.ctas * (sizeof(AttnPart) + (size_t)2 * pl.tile_rows * (p.kv.head_dim + 2) * sizeof(float));
  return pl;
}

cudaError_t launch_paged_attn(const ctts_paged_attn& p, cudaStream_t s) {
  if (p.rows == 0 || p.max_new == 0) return cudaSuccess;
  const PagedAttnPlan pl = paged_attn_plan(p);
  PagedAttnArgs a;
  a.p = p;
  a.group = p.n_heads / p.kv.n_kv_heads;
  while ((1 << a.shift) < p.kv.page_size) a.shift++;
  a.ctas = pl.ctas;
  a.tile_rows = pl.tile_rows;
  a.rows_used = rows_used_of(p);
  const double c2 = (double)p.scale * 1.4426950408889634;
  a.c2_hi = (float)c2;
  // the first part below the factor, so that the second is positive: -inf times either is -inf
  if ((double)a.c2_hi >= c2) a.c2_hi = std::nextafter(a.c2_hi, 0.0f);
  a.c2_lo = (float)(c2 - (double)a.c2_hi);
  a.parts = static_cast<AttnPart*>(p.workspace);
  a.acc = reinterpret_cast<float*>(a.parts + pl.ctas);
  a.ml = reinterpret_cast<float2*>(a.acc + (size_t)2 * pl.ctas * pl.tile_rows * p.kv.head_dim);
  if (use_tc(p))
    CTTS_LK(launch_paged_attn_tc(a, s));
  else
    CTTS_LK(with_shape(p, [&](auto q, auto k, auto hd, auto ch) {
      return launch_attn<decltype(q)::value, decltype(k)::value, decltype(hd)::value, decltype(ch)::value>(a, s);
    }));
  const int rows = (int)std::min((long)a.tile_rows, (long)p.max_new * a.group);
  const dim3 grid(a.ctas, rows > 16 ? 16 : std::min(rows, 4)), block(kJoinThreads);
  const bool bf = p.q_dtype == CTTS_BF16;
  if (p.kv.head_dim == 64)
    return bf ? launch_k(paged_attn_join_kernel<true, 64>, grid, block, 0, s, a) : launch_k(paged_attn_join_kernel<false, 64>, grid, block, 0, s, a);
  return bf ? launch_k(paged_attn_join_kernel<true, 128>, grid, block, 0, s, a) : launch_k(paged_attn_join_kernel<false, 128>, grid, block, 0, s, a);
}

}  // namespace ctts
