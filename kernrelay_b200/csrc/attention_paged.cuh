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
  int tile_tok;  // tokens of one 128-row tile of the unit (tcgen05; tpt is one or two tiles)
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
  int b, h, i;        // current unit
  int q0, T, ctx;     // its sequence
  int blk, nblk;      // next block of the unit to take, its blocks
  int pos, end, per;  // line position of `blk`, this CTA's end, blocks per CTA
};

// One warp finds the CTA's start (all lanes return it).  Everything waits for this, so the sums
// are 32 bits wide: a sequence of more than kMostBlocks blocks, or a batch of 2^31, is refused.
constexpr long kMostBlocks = 1L << 26;

template <int kKeys>
__device__ __forceinline__ Walk find_start(const Params &p, int cta, int ctas) {
  const int lane = threadIdx.x & 31;
  Seq s{0, 0, 0};
  uint32_t n = 0, per_head = 0;  // of sequence b0 + lane
  bool bad = false;
  auto load = [&](int b0, bool report) {
    s = Seq{0, 0, 0};
    n = per_head = 0;
    if (b0 + lane < p.B) {
      s = load_seq(p, b0 + lane, report);
      if (s.T) {
        const long k = blocks_per_head<kKeys>(p, s.T, s.ctx);
        bad |= k * p.HKV > kMostBlocks;
        per_head = static_cast<uint32_t>(k);
        n = bad ? 0 : per_head * p.HKV;
      }
    }
  };
  long total = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    load(b0, cta == 0);
    total += __reduce_add_sync(0xffffffffu, n);
  }
  Walk w{};
  w.per = 1;
  if (__any_sync(0xffffffffu, bad) || total > 0x7fffffffL) {
    if (cta == 0 && lane == 0) report_status(p.status, kStatusBadArgs);
    return w;
  }
  if (total == 0) return w;
  const uint32_t tot = static_cast<uint32_t>(total), per = (tot + ctas - 1) / ctas;
  const uint32_t pos = min(static_cast<unsigned long long>(per) * cta, static_cast<unsigned long long>(tot));
  w.per = per;
  w.pos = pos;
  w.end = min(tot, pos + per);
  if (w.pos >= w.end) return w;
  uint32_t before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    if (p.B > 32) load(b0, false);
    uint32_t incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > pos);
    if (hit) {
      const int l = __ffs(hit) - 1;
      uint32_t rem = pos - before - __shfl_sync(0xffffffffu, incl - n, l);
      const uint32_t ph = __shfl_sync(0xffffffffu, per_head, l);
      w.q0 = __shfl_sync(0xffffffffu, s.q0, l);
      w.T = __shfl_sync(0xffffffffu, s.T, l);
      w.ctx = __shfl_sync(0xffffffffu, s.ctx, l);
      w.b = b0 + l;
      w.h = rem / ph;
      rem -= w.h * ph;
      for (;; ++w.i) {
        w.nblk = (kv_end(p, w.T, w.ctx, w.i) + kKeys - 1) / kKeys;
        if (rem < static_cast<uint32_t>(w.nblk)) break;
        rem -= w.nblk;
      }
      w.blk = rem;
      return w;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  w.pos = w.end = 0;  // not reached: the line ends behind its last sequence
  return w;
}

// this CTA's blocks of the current unit: [w.blk, piece_end(w))
__device__ __forceinline__ int piece_end(const Walk &w) {
  return min(w.nblk, w.blk + (w.end - w.pos));
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
      if (!w.T) {  // not reached: the line ends behind its last sequence
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

// Entry `i` of sequence b's row of the page table (a page outside the cache is reported and read
// as page 0).
__device__ __forceinline__ int page_entry(const Params &p, int b, int i) {
  const int id = p.page_table[static_cast<long>(b) * p.ldp + i];
  if (id < 0 || id >= p.pages) {
    report_status(p.status, kStatusBadIndex);
    return 0;
  }
  return id;
}

// The page numbers of a piece, in order, to a producer warp: a lane holds one of 32, and the next
// 32 are on their way (under load a table entry takes as long as a block of keys).
struct PageFeed {
  int b, first, count;  // table row; first entry of the piece, entries
  int at;               // entry (from `first`) of cur's lane 0
  int cur, nxt;

  __device__ __forceinline__ int load(const Params &p, int i) const {
    return i < count ? page_entry(p, b, first + i) : 0;
  }
  // keys [key0, key1) of sequence b
  __device__ __forceinline__ void begin(const Params &p, int b_, int key0, int key1) {
    const int lane = threadIdx.x & 31;
    b = b_;
    first = key0 >> p.page_shift;
    count = ((key1 - 1) >> p.page_shift) - first + 1;
    at = 0;
    cur = load(p, lane);
    nxt = load(p, 32 + lane);
  }
  // To be called before pages of keys from `low` on are asked for; `low` never falls.
  __device__ __forceinline__ void advance(const Params &p, int low) {
    if ((low >> p.page_shift) - first >= at + 32) {
      at += 32;
      cur = nxt;
      nxt = load(p, at + 32 + (threadIdx.x & 31));
    }
  }
  // the page of `key` (the same for all lanes, within 32 pages of the last `low`)
  __device__ __forceinline__ int page(const Params &p, int key) const {
    const int i = (key >> p.page_shift) - first - at;
    return __shfl_sync(0xffffffffu, i < 32 ? cur : nxt, i & 31);
  }
};

// A wait of a whole warp whose lanes go on together or not at all: a wait that ran out for some of
// them may have come for the others at its last poll, and a lane that left alone would be missing
// from the warp's next vote or tensor-memory access.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t *bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, kMbarLimitNs));
}

// one lane of a warp that is converged (the same one every time)
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(r));
  return r != 0;
}

// Asks L2 for the page table while the schedule is searched: a line per thread of all CTAs.
__device__ __forceinline__ void prefetch_page_table(const Params &p, int thread, int threads) {
  const int lines = (p.max_pages + 31) / 32;  // of a row
  const long i = static_cast<long>(blockIdx.x) * threads + thread;
  if (i < static_cast<long>(lines) * p.B) {
    const long row = i / lines;
    const int32_t *at = p.page_table + row * p.ldp + (i - row * lines) * 32;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
  }
}

// What the combine kernel needs of a unit that CTA c starts and later CTAs go on with.
__device__ __forceinline__ int4 split_desc(const Params &p, const Walk &w) {
  // unit's end on the line; its last CTA holds position end - 1
  const uint32_t end = w.pos - w.blk + w.nblk, per = w.per;
  const int tok0 = w.i * p.tpt;
  return make_int4(w.q0 + tok0, min(p.tpt, w.T - tok0), w.h,
                   static_cast<int>((end - 1) / per - w.pos / per) + 1);
}

__device__ __forceinline__ float *slot_ml(const Params &p, int cta, int slot) {
  return p.ml + (static_cast<long>(cta) * 2 + slot) * 2 * p.rows;
}
__device__ __forceinline__ float *slot_o(const Params &p, int cta, int slot) {
  return p.o + (static_cast<long>(cta) * 2 + slot) * p.rows * p.D;
}

// P goes into PV in the cache's type, as 2^(s - m + shift) of a row whose offset m lags its maximum by
// at most LAG: fp16 starts losing bits at 2^-14, and many keys that small may outweigh the largest
// one, so P uses the type up to 2^15 (m and the sums of all pieces carry the same factor, which the
// division by the row sum takes out).  What is left below: a key's absolute error is 2^-25 of values
// whose largest is 2^(15 - LAG) or more.  bf16 has the exponents of fp32 and needs no shift.
//
// What the exponents subtract, m - shift for an offset m (0 for that of a row that has seen nothing), is
// rounded up, as m is where it is taken from a score (row_max): so an exponent is at most its bound
// however large the scores are (above 2^23 a rounding is 1 or more, and P would pass 2^16).
template <bool F16, int LAG>
__device__ __forceinline__ float p_offset(float m) {
  if (m == -INFINITY) m = 0.f;
  return F16 ? __fsub_ru(m, 15.f - LAG) : m;
}

// the running maximum's unit: a raw score's product with scale * log2(e) > 0
__device__ __forceinline__ float row_max(float top, float scale_log2) { return __fmul_ru(top, scale_log2); }

__device__ __forceinline__ float exp2_mufu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Host side: the tensor maps of one layer's K and V, boxes of min(page_size, keys) slots
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
