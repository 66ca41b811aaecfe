// paged_attn.cuh -- how the work of a paged attention call is cut: the line
// of key tiles, a CTA's piece of it, and the partial states of divided items.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "tc_ptx.cuh"

namespace ctts {

// Partial states in the workspace: CTA c has two places, 2c for a piece that
// enters it (the middle or the end of an item) and 2c + 1 for one that begins
// in it and leaves it.  An item that leaves CTA c is described by parts[c]:
// its pieces lie in places 2c + 1, 2(c + 1), 2(c + 2), ...
struct AttnPart {
  int pieces = 0;  // 0: no item leaves this CTA
  int row0 = 0;    // the request's first row of q
  int packed0 = 0, rows = 0, h = 0;  // first packed row, packed rows, KV head
  int pad[3] = {0, 0, 0};
};

// What the line follows from.  Functions that are called, not inlined, take
// it by value: a reference to a kernel's parameters would be read as memory.
struct AttnLine {
  const int *cu_rows = nullptr, *seq_lens = nullptr;
  int batch = 0, rows = 0, max_new = 0, max_len = 0;
  int group = 1, n_kv = 1;  // query heads per KV head, KV heads
  int ctas = 0;
};

struct PagedAttnArgs {
  ctts_paged_attn p;
  AttnLine line;
  int group = 1, shift = 0;      // query heads per KV head, log2 of the page size
  int tile_rows = 0;             // packed rows per item
  int rows_used = 0;             // packed rows a short item can have
  float c2 = 0;                  // scale * log2(e): scores to powers of two
  AttnPart* parts = nullptr;     // [ctas]
  uint32_t tries = kWaitLimit;   // of a wait
  int keep_cta0 = 0;             // error-path testing (ctts_debug_inject_wait_fault): CTA 0 never hands a stage back
  float2* ml = nullptr;          // [2 * ctas][tile_rows]: maximum of q . k, sum
  float* acc = nullptr;          // [2 * ctas][tile_rows][hd]: unnormalised output
};

CTTS_DEV uint32_t pack_bf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// x in N bf16 terms (packed pairs), each the rounding of what the ones before
// leave: N = 1, 2, 3 keep 8, 16, 24 bits.  What an infinite x leaves is NaN;
// the maximum turns that into a large negative number, so the sum of the
// terms is the infinity again (of a finite x less than 2^120 is left).
template <int N>
CTTS_DEV void split_bf2(float x0, float x1, uint32_t* t) {
#pragma unroll
  for (int i = 0; i < N; i++) {
    t[i] = pack_bf2(x0, x1);
    if (i + 1 < N) {
      x0 = fmaxf(x0 - bf_lo(t[i]), -1.3e36f);
      x1 = fmaxf(x1 - bf_hi(t[i]), -1.3e36f);
    }
  }
}

CTTS_DEV float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Score s = q . k under a maximum m to the exponential's argument.  The
// difference first: the roundings then cost a few 2^-24 of the argument, not
// of the score, and the maximum's own weight is 1 however large the scores are.
CTTS_DEV float attn_arg(float s, float m, float c2) { return (s - m) * c2; }

// A request's lengths, cut to what the buffers hold.
struct AttnReq {
  int r0, cnt, nn, len;  // first row, rows, rows computed (cnt cut to max_new), tokens
};
CTTS_DEV AttnReq attn_req(const AttnLine& ln, int b) {
  AttnReq r;
  r.r0 = min(max(ln.cu_rows[b], 0), ln.rows);
  r.cnt = min(max(ln.cu_rows[b + 1], r.r0), ln.rows) - r.r0;
  r.nn = min(r.cnt, ln.max_new);
  r.len = min(max(ln.seq_lens[b], 0), ln.max_len);
  return r;
}
// Row tiles of a request (packed rows fit 31 bits: the host checks).
template <int R>
CTTS_DEV int attn_row_tiles(const AttnReq& r, int group) {
  return (r.nn * group + R - 1) / R;
}
// Key tiles of row tile m: up to the position of its last row; at least one,
// which also writes the zeros of rows that see nothing.
template <int R, int C>
CTTS_DEV int attn_tiles(const AttnReq& r, int m, int group) {
  const int packed = (m + 1) * R;  // packed rows up to the tile's end
  const int ahead = packed >= r.nn * group ? r.nn : (packed - 1) / group + 1;
  return max(1, (min(r.len, r.len - r.cnt + ahead) + C - 1) / C);
}
// What an item is made of and what it costs on the line, in units: R packed
// rows, tiles of C keys, W1 units a tile of an item of up to 128 packed rows,
// W2 of one with more, and COST ahead of its tiles to begin and end it (queries
// in, output out).  A CTA has the tiles that begin in its piece.
template <int R_, int C_, int W1_, int W2_, int COST_>
struct AttnItem {
  static constexpr int R = R_, C = C_, W1 = W1_, W2 = W2_, COST = COST_;
  static CTTS_DEV int weight(int packed) { return packed > 128 ? W2 : W1; }  // of a tile, from the packed rows left in the request
  static CTTS_DEV int tiles_in(int units, int w) { return w == W1 ? (units + W1 - 1) / W1 : (units + W2 - 1) / W2; }  // that begin there
};

// The row tiles of a request in order: the rows ahead of each one's end by
// running quotient and remainder, without a division a tile.
template <int R, int C>
struct AttnRowWalk {
  const AttnReq& r;
  int group, per, over, ahead, rem;  // ahead = ((m + 1) R - 1) / group, rem its remainder
  CTTS_DEV AttnRowWalk(const AttnReq& req, int g) : r(req), group(g) {
    per = R / g;
    over = R - per * g;
    ahead = per;
    rem = over - 1;
    if (rem < 0) {
      rem += g;
      ahead--;
    }
  }
  CTTS_DEV int tiles() const { return max(1, (min(r.len, r.len - r.cnt + min(r.nn, ahead + 1)) + C - 1) / C); }
  CTTS_DEV void next() {
    ahead += per;
    rem += over;
    if (rem >= group) {
      rem -= group;
      ahead++;
    }
  }
};
template <class T>
CTTS_DEV long attn_units(const AttnLine& ln, const AttnReq& r) {
  const int mt = attn_row_tiles<T::R>(r, ln.group);
  AttnRowWalk<T::R, T::C> w(r, ln.group);
  long n = 0;
#pragma unroll 1
  for (int m = 0; m < mt; m++, w.next()) n += (long)w.tiles() * T::weight(r.nn * ln.group - m * T::R) + T::COST;
  return n * ln.n_kv;
}
// The line is cut into `ctas` pieces of `base` units, the first `rest` of them
// one longer; none shorter than a tile, so that the pieces of a divided item
// lie in neighbouring CTAs.
struct AttnCut {
  int ctas;
  long base, rest;
  CTTS_DEV AttnCut(int n, long total, int tile) {
    ctas = total < (long)n * tile ? (int)total / tile : n;
    if (ctas == 0) ctas = 1;
    base = total >> 32 ? total / ctas : (long)((unsigned)total / (unsigned)ctas);  // (a 64-bit division is ten times the latency)
    rest = total - base * ctas;
  }
  CTTS_DEV long begin(int c) const { return c < ctas ? c * base + min((long)c, rest) : base * ctas + rest; }
  CTTS_DEV int owner(long unit) const {  // the CTA that has a unit
    const long longer = rest * (base + 1);
    return (int)(unit < longer ? unit / (base + 1) : rest + (unit - longer) / base);
  }
};

struct AttnStart {
  long units;  // this CTA's
  long end, total;  // where they end on the line, and its length
  long skip;   // units of request b ahead of them
  int b;
  AttnReq req;
};

// This CTA's piece of the line.  The block sums the requests' units, a request
// a thread and turn; a second pass finds the request the piece begins in (from
// registers when one turn holds the batch).  (Code that runs once a launch is
// kept small throughout these kernels: what does not fit the instruction cache
// beside the main loop costs more than a rolled loop.)
template <class T, int NT>
CTTS_DEV void attn_find_start(const AttnLine& ln, AttnStart* out) {
  constexpr int W = NT / 32;
  __shared__ long wsum[2][W];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = ln.batch;
  long total = 0, first = 0, u0 = 0, u1 = 0;
  AttnReq rq = {0, 0, 0, 0};
  int ph = 0, pass = 0, base = 0;
  while (true) {
    // units of request base + tid, and those ahead of it in this turn
    const int b = base + tid;
    long u = 0;
    if (b < n) {
      rq = attn_req(ln, b);
      u = attn_units<T>(ln, rq);
    }
    long inc = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) wsum[ph][warp] = inc;
    __syncthreads();
    long all = 0, ahead = 0;
#pragma unroll
    for (int w = 0; w < W; w++) {
      const long y = wsum[ph][w];
      if (w < warp) ahead += y;
      all += y;
    }
    ph ^= 1;
    base += NT;
    if (pass == 0) {
      total += all;
      if (base < n) continue;
      const AttnCut cut(ln.ctas, total, max(T::W1, T::W2));
      u0 = cut.begin(blockIdx.x);
      u1 = cut.begin(blockIdx.x + 1);
      if (tid == 0) {
        out->units = u1 - u0;
        out->end = u1;
        out->total = total;
      }
      if (u1 == u0) break;
      if (n > NT) {
        pass = 1;
        base = 0;
        continue;
      }
    }
    const long at = first + ahead + inc - u;
    if (at <= u0 && u0 < at + u) {
      out->b = b;
      out->skip = u0 - at;
      out->req = rq;
    }
    first += all;
    if (first > u0) break;
  }
  __syncthreads();
}

// CTAs from this one to the one that has the unit `more` behind this CTA's end.
template <class T>
CTTS_DEV int attn_pieces(const AttnLine& ln, const AttnStart& s, int more) {
  return AttnCut(ln.ctas, s.total, max(T::W1, T::W2)).owner(s.end + more) - (int)blockIdx.x + 1;
}

// A place on the line: request, row tile, KV head, key tile.  A role walks its
// CTA's pieces: tiles kt .. of one item, then the next item's from 0.
template <class T>
struct AttnCursor {
  int b, m, h, kt, nt, mt;
  int w;  // units a tile
  int r0, cnt, nn, len;

  CTTS_DEV void set(const AttnLine& ln, const AttnReq& r) {
    r0 = r.r0; cnt = r.cnt; nn = r.nn; len = r.len;
    mt = attn_row_tiles<T::R>(r, ln.group);
  }
  // `skip` units into request b; kt: units behind the first tile's begin
  static __device__ __noinline__ AttnCursor seek(AttnLine ln, AttnReq req, int b, long skip) {
    AttnCursor c;
    c.b = b;
    c.set(ln, req);
    AttnRowWalk<T::R, T::C> walk(req, ln.group);
#pragma unroll 1
    for (c.m = 0;; c.m++, walk.next()) {
      c.nt = walk.tiles();
      c.w = T::weight(req.nn * ln.group - c.m * T::R);
      const long in = (long)(c.nt * c.w + T::COST) * ln.n_kv;
      if (skip < in || c.m + 1 >= c.mt) break;
      skip -= in;
    }
    const unsigned item = c.nt * c.w + T::COST;  // (skip is inside one row tile's heads: 31 bits)
    c.h = (unsigned)skip / item;
    c.kt = (int)((unsigned)skip % item) - T::COST;
    return c;
  }
  // The CTA's first piece; left: units from its first tile to the CTA's end
  // (0: nothing to do).
  static CTTS_DEV AttnCursor at(const AttnLine& ln, const AttnStart& s, int* left) {
    *left = (int)s.units;  // (of one CTA: 31 bits, the host checks)
    AttnCursor c{};
    if (*left > 0) {
      c = seek(ln, s.req, s.b, s.skip);
      if (T::W1 == 1 && T::W2 == 1) {
        *left += min(c.kt, 0);
        c.kt = max(c.kt, 0);
      } else {
        const int kt = c.kt > 0 ? T::tiles_in(c.kt, c.w) : 0;
        *left -= kt * c.w - c.kt;
        c.kt = kt;
        if (kt == c.nt) {  // the last tile began ahead of the piece
          *left -= T::COST;
          if (*left > 0) c = next(ln, c);
        }
      }
      *left = max(*left, 0);
    }
    return c;
  }
  // Tiles of the piece.
  CTTS_DEV int tiles(int left) const { return min(nt - kt, T::tiles_in(left, w)); }
  // What is left of the CTA's units at the first tile of the next item, behind
  // a piece of n tiles (0: there is none).
  CTTS_DEV int behind(int left, int n) const { return max(0, left - n * w - T::COST); }
  // The next item, from its first tile (never called at the end of the line).
  static CTTS_DEV AttnCursor next(const AttnLine& ln, AttnCursor c) {
    c.kt = 0;
    if (++c.h < ln.n_kv) return c;
    return next_rows(ln, c);
  }
  static __device__ __noinline__ AttnCursor next_rows(AttnLine ln, AttnCursor c) {
    c.h = 0;
    if (++c.m == c.mt) {
      c.m = 0;
#pragma unroll 1
      do {
        c.b++;
        c.set(ln, attn_req(ln, c.b));
      } while (c.mt == 0 && c.b + 1 < ln.batch);
    }
    c.nt = attn_tiles<T::R, T::C>(AttnReq{c.r0, c.cnt, c.nn, c.len}, c.m, ln.group);
    c.w = T::weight(c.nn * ln.group - c.m * T::R);
    return c;
  }
  // Packed rows of the item, and the position of the request's first new row.
  CTTS_DEV int rows(const AttnLine& ln, int R) const { return min(R, nn * ln.group - m * R); }
  CTTS_DEV int pos0() const { return len - cnt; }
};

// The pool as a 4D tensor map: 128 bytes of a head by `box` slots a copy, the
// slot, head and page dimensions by ascending stride.  order: what dimensions
// 1, 2 and 3 are (0 slot, 1 head, 2 page), two bits each.
bool paged_pool_map(CUtensorMap* m, const void* base, const ctts_paged_kv& kv, int box, int* order);

// One box: `block` 128-byte blocks into the head's row.
CTTS_DEV void copy_box(uint32_t dst, const CUtensorMap* m, int order, int x, int slot, int head, int page, uint64_t* bar) {
  const int c[3] = {slot, head, page};
  const int y = c[0] * ((order & 3) == 0) + c[1] * ((order & 3) == 1) + c[2] * ((order & 3) == 2);
  const int z = c[0] * ((order >> 2 & 3) == 0) + c[1] * ((order >> 2 & 3) == 1) + c[2] * ((order >> 2 & 3) == 2);
  const int w = c[0] * ((order >> 4) == 0) + c[1] * ((order >> 4) == 1) + c[2] * ((order >> 4) == 2);
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// Whether the phase with this parity is over.
CTTS_DEV bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return done != 0;
}
// Wait of *tries tries, which all roles of a block share.  The one that gives
// up sets them to zero: nobody waits after that, the block runs to its end.
CTTS_DEV void mbar_wait_or(uint64_t* bar, uint32_t parity, volatile uint32_t* tries) {
  if (mbar_try(bar, parity)) return;
#pragma unroll 1
  for (uint32_t it = 0; it < *tries; ++it)
    if (mbar_try(bar, parity)) return;
  *tries = 0;
}
CTTS_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
CTTS_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Long items on tcgen05 (paged_attn_tc.cu).
int paged_attn_tc_rows(const ctts_paged_attn& p);  // packed rows per item
cudaError_t launch_paged_attn_tc(const PagedAttnArgs& a, cudaStream_t s);

}  // namespace ctts
