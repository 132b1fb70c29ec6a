// What the two paged attention kernels (attention_paged.cu: mma.sync for few query rows,
// attention_paged_tc.cu: tcgen05 for many) share: how the work is cut, where partial results
// lie, masks, and the page loads.
//
// A unit is (sequence b, KV head h, tile i of `tpt` new tokens): its rows are the tile's tokens x
// the query heads of h, its keys the blocks of kKeys positions up to the last one that any of
// its rows sees.  All units' blocks in order (b, h, i) form one line; CTA c of G takes blocks
// [c * P, (c + 1) * P) of it, P = ceil(total / G).  So every SM reads the same number of keys
// whatever the batch, the lengths are read on the device only (a captured call follows them),
// and a unit cut by CTA borders is joined by combine_kernel.  A CTA leaves at most two pieces:
// slot 0 of a unit that began before it, slot 1 of one that goes on after it.
#pragma once

#include "paged.h"
#include "ptx.cuh"

namespace krb {
namespace paged {

struct Params {
  const uint16_t *q;
  uint16_t *out;
  long ldq, ldo;
  const int32_t *page_table, *kv_lens, *q_starts;
  const uint32_t *mask;
  long ldp, ldm;
  int N, HQ, HKV, group, D;
  int B, max_q, max_pages, pages, page_shift, mask_words;
  int tpt;       // tokens of a unit
  int tile_tok;  // tokens of one tensor-core tile of the unit (tc kernel; tpt = 1 or 2 tiles)
  int rows;      // rows of a partial result's slot
  float scale_log2;
  uint32_t *status;
  // workspace: G descriptors, then per CTA and slot: m and l [rows] (log2 units), O [rows][D]
  int4 *desc;
  float *ml;
  float *o;
};

struct Seq {
  int q0, T, ctx;  // first row, new tokens (0: none, or refused), positions before them
};

// `report`: say so where the sequence is refused
__device__ __forceinline__ Seq load_seq(const Params &p, int b, bool report) {
  const int q0 = p.q_starts[b], q1 = p.q_starts[b + 1], len = p.kv_lens[b];
  Seq s{q0, 0, 0};
  if (q0 == q1 && q0 >= 0) return s;
  const long room = static_cast<long>(p.max_pages) << p.page_shift;
  if (q0 < 0 || q1 < q0 || q1 > p.N || q1 - q0 > p.max_q || len < q1 - q0 || len > room) {
    if (report) report_status(p.status, kStatusBadArgs);
    return s;
  }
  s.T = q1 - q0;
  s.ctx = len - s.T;
  return s;
}

__device__ __forceinline__ int tiles_of(const Params &p, int T) { return (T + p.tpt - 1) / p.tpt; }

// positions that tile i of a sequence looks at: all of them under a mask, else up to its last token
__device__ __forceinline__ int kv_end(const Params &p, int T, int ctx, int i) {
  return ctx + (p.mask ? T : min(T, (i + 1) * p.tpt));
}

template <int kKeys>
__device__ __forceinline__ long blocks_per_head(const Params &p, int T, int ctx) {
  const int nt = tiles_of(p, T);
  long n = 0;
  for (int i = 0; i < nt; ++i) n += (kv_end(p, T, ctx, i) + kKeys - 1) / kKeys;
  return n;
}

// A CTA's place on the line, kept by every role of the CTA alike.
struct Walk {
  int b, h, i;       // current unit
  int q0, T, ctx;    // its sequence
  int blk, nblk;     // next block of the unit to take, its blocks
  long pos, end, per;  // line position of `blk`, this CTA's end, blocks per CTA
};

struct WalkStart {
  int b, h, i, blk;
  long pos, end, per;
};

// One warp finds the CTA's start (all lanes return it).
template <int kKeys>
__device__ __forceinline__ WalkStart find_start(const Params &p, int cta, int ctas) {
  const int lane = threadIdx.x & 31;
  long total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    long n = 0;
    if (b0 + lane < p.B) {
      const Seq s = load_seq(p, b0 + lane, cta == 0);
      if (s.T) n = blocks_per_head<kKeys>(p, s.T, s.ctx) * p.HKV;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total += n;
  }
  WalkStart w{0, 0, 0, 0, 0, 0, 1};
  if (total == 0) return w;
  w.per = (total + ctas - 1) / ctas;
  w.pos = min(total, w.per * cta);
  w.end = min(total, w.pos + w.per);
  if (w.pos >= w.end) return w;
  long before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    long n = 0, per_head = 0;
    Seq s{0, 0, 0};
    if (b0 + lane < p.B) {
      s = load_seq(p, b0 + lane, false);
      if (s.T) per_head = blocks_per_head<kKeys>(p, s.T, s.ctx);
      n = per_head * p.HKV;
    }
    long incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > w.pos);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const long excl = __shfl_sync(0xffffffffu, incl - n, l);
      per_head = __shfl_sync(0xffffffffu, per_head, l);
      const int T = __shfl_sync(0xffffffffu, s.T, l), ctx = __shfl_sync(0xffffffffu, s.ctx, l);
      long rem = w.pos - before - excl;
      w.b = b0 + l;
      w.h = static_cast<int>(rem / per_head);
      rem -= w.h * per_head;
      for (;;) {
        const int nb = (kv_end(p, T, ctx, w.i) + kKeys - 1) / kKeys;
        if (rem < nb) break;
        rem -= nb;
        ++w.i;
      }
      w.blk = static_cast<int>(rem);
      return w;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  w.pos = w.end = 0;
  return w;
}

template <int kKeys>
__device__ __forceinline__ Walk begin_walk(const Params &p, const WalkStart &s) {
  Walk w;
  w.b = s.b;
  w.h = s.h;
  w.i = s.i;
  w.blk = s.blk;
  w.pos = s.pos;
  w.end = s.end;
  w.per = s.per;
  w.q0 = w.T = w.ctx = w.nblk = 0;
  if (w.pos < w.end) {
    const Seq q = load_seq(p, w.b, false);
    w.q0 = q.q0;
    w.T = q.T;
    w.ctx = q.ctx;
    w.nblk = (kv_end(p, w.T, w.ctx, w.i) + kKeys - 1) / kKeys;
  }
  return w;
}

// this CTA's blocks of the current unit: [w.blk, piece_end(w))
__device__ __forceinline__ int piece_end(const Walk &w) {
  const long left = w.end - w.pos;
  return w.nblk - w.blk <= left ? w.nblk : w.blk + static_cast<int>(left);
}

// the unit after the piece that ends at block `e` (only when the CTA has blocks left)
template <int kKeys>
__device__ __forceinline__ void next_unit(const Params &p, Walk &w, int e) {
  w.pos += e - w.blk;
  w.blk = 0;
  if (w.pos >= w.end) return;
  if (++w.i >= tiles_of(p, w.T)) {
    w.i = 0;
    if (++w.h >= p.HKV) {
      w.h = 0;
      w.T = 0;
      while (!w.T && ++w.b < p.B) {
        const Seq q = load_seq(p, w.b, false);
        w.q0 = q.q0;
        w.T = q.T;
        w.ctx = q.ctx;
      }
      if (!w.T) {  // not reached: the line ends with the last sequence
        w.pos = w.end;
        return;
      }
    }
  }
  w.nblk = (kv_end(p, w.T, w.ctx, w.i) + kKeys - 1) / kKeys;
}

// Drafted tokens j0 .. j0+31 (j0 may be negative: cached positions) that row token t sees.
__device__ __forceinline__ uint32_t visible32(const Params &p, const uint32_t *row_mask, int T,
                                              int t, int j0) {
  const int n = (p.mask ? T : t + 1) - j0;  // positions of the window that are there at all
  if (n <= 0) return 0u;
  const uint32_t there = n >= 32 ? 0xffffffffu : (1u << n) - 1u;
  if (!p.mask || j0 <= -32) return there;
  const int w = j0 >> 5;  // floor
  const uint32_t lo = w < 0 ? 0xffffffffu : (w < p.mask_words ? row_mask[w] : 0u);
  const uint32_t hi = w + 1 < 0 ? 0xffffffffu : (w + 1 < p.mask_words ? row_mask[w + 1] : 0u);
  return __funnelshift_r(lo, hi, j0 & 31) & there;
}

// Page of key block position `key` (a page outside the cache is reported and read as page 0).
__device__ __forceinline__ int page_of(const Params &p, int b, int key) {
  const int id = p.page_table[static_cast<long>(b) * p.ldp + (key >> p.page_shift)];
  if (id < 0 || id >= p.pages) {
    report_status(p.status, kStatusBadIndex);
    return 0;
  }
  return id;
}

// What the combine kernel needs of a unit that CTA c starts and later CTAs go on with.
__device__ __forceinline__ int4 split_desc(const Params &p, const Walk &w) {
  // unit's end on the line; its last CTA holds position end - 1
  const long end = w.pos - w.blk + w.nblk;
  const int last = static_cast<int>((end - 1) / w.per);
  const int first = static_cast<int>(w.pos / w.per);
  const int tok0 = w.i * p.tpt;
  return make_int4(w.q0 + tok0, min(p.tpt, w.T - tok0), w.h, last - first + 1);
}

__device__ __forceinline__ float *slot_ml(const Params &p, int cta, int slot) {
  return p.ml + (static_cast<long>(cta) * 2 + slot) * 2 * p.rows;
}
__device__ __forceinline__ float *slot_o(const Params &p, int cta, int slot) {
  return p.o + (static_cast<long>(cta) * 2 + slot) * p.rows * p.D;
}

// Row of a slot that holds packed row r (token-major: token r / group, head r % group) of a
// unit: the tc kernel keeps each tile's tokens in 128 rows of its own.
__device__ __forceinline__ int slot_row(const Params &p, int tok, int g) {
  const int tile = tok / p.tile_tok;
  return tile * 128 + (tok - tile * p.tile_tok) * p.group + g;
}

__device__ __forceinline__ void pdl_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float exp2_mufu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Host side.  Joins the split units of a launch of `ctas` CTAs (programmatic dependent launch:
// its CTAs are set up while the attention kernel drains).
void launch_combine(const Params &p, int ctas, bool f16, cudaStream_t stream);
// the tensor maps of one layer's K and V, boxes of min(page_size, keys) slots
struct KvMaps {
  CUtensorMap k, v;
  int box;
};
KvMaps make_kv_maps(const krb_kv_cache &c, int layer, int keys);
// q [tokens, HQ, D] with token pitch ldq: boxes of tok x heads x 64
CUtensorMap make_tmap_rows(const void *q, int N, int HQ, int D, long ldq, int tok, int heads);
// attention_paged_tc.cu
void launch_tc(const krb_kv_cache &c, int layer, const Params &p, int ctas, int device,
               cudaStream_t stream);
size_t workspace_bytes(int ctas, int rows, int D);
void carve_workspace(Params &p, int ctas, void *ws);

}  // namespace paged
}  // namespace krb
