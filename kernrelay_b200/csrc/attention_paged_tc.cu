// Attention of new tokens over the paged K/V cache, the form for many query rows (wide drafts,
// chunks of a prompt): tcgen05 with S, P and O in TMEM.
//
// A unit is one or two 128-row tiles (whole tokens x the query heads of one KV head) that share
// every K and V block; a block is 128 keys.  Per block and tile: S = Q K^T (SS form, both K-major),
// the tile's 128 softmax threads (thread = row) turn S into P in place and O += P V (P from TMEM,
// V from shared memory as it lies in the cache, [key][d], so MN-major: no transposed copy).
// Issue order per block j: PV(A,j), QK(A,j+1), PV(B,j), QK(B,j+1), so one tile's products run
// under the other tile's softmax.
//
// Bound: with R rows the products take 4 R 128 D flop per block for 512 D bytes of K and V; from
// about 250 rows on the softmax (128 x 128 exponentials per tile and block, 16 per clock and SM)
// and the products bind, below it HBM does.
#include <algorithm>
#include <string>

#include "attention_paged.cuh"

namespace krb {
namespace paged {

namespace {

constexpr int kKeys = 128;
constexpr uint32_t kChunk = 128 * 128;  // 128 rows x 64 elements, bytes
constexpr uint32_t kTmemCols = 512;
// The running offset of a row moves (and O is rescaled) only when its maximum grew by more than
// 2^8: until then P <= 256, which both 2-byte types hold with their full precision.
constexpr float kRescaleLog2 = 8.0f;

template <int D, int NT>
struct Cfg {
  static constexpr int kTile = 256 * D;  // one Q tile, K block or V block, bytes
  static constexpr int kSlots = D == 64 ? 8 : (NT == 2 ? 5 : 6);
  static constexpr int kThreads = 64 + 128 * NT;
  static constexpr int kBars = 2 * kSlots + 2 + 3 * NT;
  static constexpr int kSmem =
      (NT + kSlots) * kTile + kBars * 8 + int(sizeof(Walk)) + 32 + 1024;
};

// D[tmem] (+)= A[tmem] * B[smem], A 16-bit pairs K-major
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32"
      " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
      " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Descriptor of a V block as the MN-major operand: 64-element (128-byte) rows of one key each,
// swizzled by 8 keys (1024 bytes: the K-direction step), the next 64 columns of D a chunk further
// (the MN-direction step).
__device__ __forceinline__ uint64_t sdesc_mnmajor_sw128(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kChunk >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// Where the blocks of a piece of n lie in the ring, counted from its first load: the order is
// K0, K1, V0, K2, V1, ... (K of the next block before V of this one).
__device__ __forceinline__ int k_at(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int v_at(int j, int n) { return j + 1 < n ? 2 * j + 2 : 2 * j + 1; }

// One block of one row: S (128 columns at s_col) -> P over its first 64 columns, in one pass of
// 32 scores at a time.  `see`(c): which of chunk c's 32 keys the row sees.  See attention_tc.cu's
// softmax for the stale offset; here rows may have seen nothing yet (m = -inf), whose offset is 0.
template <int D, bool F16, bool kMask, typename See>
__device__ __forceinline__ void softmax_block(uint32_t s_col, uint32_t o_col, float scale_log2,
                                              bool has_o, float &m_run, float &l_run, See see) {
  float m_cur = m_run;
  float r8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  uint32_t ra[32], rb[32];
  tmem_ld_32x32(s_col, ra);
  tmem_wait_ld();
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t(&r)[32] = (c & 1) ? rb : ra;
    if (c + 1 < 4) tmem_ld_32x32(s_col + (c + 1) * 32, (c & 1) ? ra : rb);
    if constexpr (kMask) {
      const uint32_t bits = see(c);
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!((bits >> e) & 1)) r[e] = 0xff800000u;  // -inf
    }
    float m8[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) m8[e] = __uint_as_float(r[e]);
#pragma unroll
    for (int e = 8; e < 32; ++e) m8[e & 7] = fmaxf(m8[e & 7], __uint_as_float(r[e]));
    const float cmax = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])),
                             fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7]))) * scale_log2;
    const bool grow = cmax - m_cur > kRescaleLog2;
    if (c > 0 && __any_sync(0xffffffffu, grow)) {
      // the P chunks of this block that are already written follow the new offset
      const float f = grow ? exp2_mufu(m_cur - cmax) : 1.f;
      tmem_wait_st();
#pragma unroll 1
      for (int pc = 0; pc < c; ++pc) {
        uint32_t q[16];
        tmem_ld16(s_col + pc * 16, q);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 pr = unpack2<F16>(q[e]);
          q[e] = pack2<F16>(pr.x * f, pr.y * f);
        }
        tmem_st16(s_col + pc * 16, q);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) r8[e] *= f;
    }
    if (grow) m_cur = cmax;
    const float off = m_cur == -INFINITY ? 0.f : m_cur;
    uint32_t pk[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p0 = exp2_mufu(fmaf(__uint_as_float(r[2 * e]), scale_log2, -off));
      const float p1 = exp2_mufu(fmaf(__uint_as_float(r[2 * e + 1]), scale_log2, -off));
      // P in the cache's type; the row sum takes the fp32 values
      pk[e] = pack2<F16>(p0, p1);
      r8[e & 7] += p0 + p1;
    }
    tmem_st16(s_col + c * 16, pk);
    if (c + 1 < 4) tmem_wait_ld();
  }
  tmem_wait_st();
  const float rs = ((r8[0] + r8[1]) + (r8[2] + r8[3])) + ((r8[4] + r8[5]) + (r8[6] + r8[7]));
  const bool moved = m_cur != m_run;
  const float alpha = moved ? exp2_mufu(m_run - m_cur) : 1.f;
  if (has_o && __any_sync(0xffffffffu, moved)) {
#pragma unroll 1
    for (int c = 0; c < D / 16; ++c) {
      uint32_t r[16];
      tmem_ld16(o_col + c * 16, r);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
      tmem_st16(o_col + c * 16, r);
    }
    tmem_wait_st();
  }
  l_run = l_run * alpha + rs;
  m_run = m_cur;
}

}  // namespace

template <int D, int NT, bool F16>
__global__ void __launch_bounds__(64 + 128 * NT, 1)
    attn_paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q,
                         const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const Params p, int box_shift) {
  using C = Cfg<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem =
      reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = smem + NT * C::kTile;
  uint64_t *full = reinterpret_cast<uint64_t *>(ring + C::kSlots * C::kTile);
  uint64_t *empty = full + C::kSlots;
  uint64_t *q_full = empty + C::kSlots;
  uint64_t *q_empty = q_full + 1;
  uint64_t *s_full = q_empty + 1;
  uint64_t *p_ready = s_full + NT;
  uint64_t *o_done = p_ready + NT;
  Walk *start = reinterpret_cast<Walk *>(o_done + NT);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(start + 1);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 32) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < NT; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_done[i], 1);
    }
    fence_mbar_init();
  }
  if (warp >= 2) prefetch_page_table(p, threadIdx.x - 64, C::kThreads - 64);
  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    const Walk s = find_start<kKeys>(p, blockIdx.x, gridDim.x);
    if (lane == 0) *start = s;
  } else if (warp == 1) {
    __syncwarp();
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Walk w = *start;

  if (warp == 0) {
    // ---------------- TMA producer: a box (page x 64 columns) per lane
    constexpr int kHalves = D / 64;
    const int box = 1 << box_shift;
    const int bx = lane / kHalves, half = lane % kHalves;  // page 8 at D 128: 16 boxes x 2 halves
    PageFeed feed;
    int n = 0, pieces = 0;
    bool ok = true;
    while (w.pos < w.end) {
      const int e = piece_end(w);
      const int nblk = e - w.blk;
      const int end = kv_end(p, w.T, w.ctx, w.i);
      const int tok0 = w.i * p.tpt;
      const bool has_b = NT > 1 && tok0 + p.tile_tok < w.T;
      feed.begin(p, w.b, w.blk * kKeys, min(end, e * kKeys));
      for (int a = 0; a < 2 * nblk && ok; ++a, ++n) {
        const bool is_v = a >= 2 && ((a & 1) == 0 || a == 2 * nblk - 1);
        const bool only = nblk == 1 && a == 1;  // one block: K0, V0
        const bool v = is_v || only;
        const int j = v ? (a == 2 * nblk - 1 ? nblk - 1 : a / 2 - 1) : (a + 1) / 2;
        const int key0 = (w.blk + j) * kKeys;
        const int nbox = (min(kKeys, end - key0) + box - 1) >> box_shift;
        const int key = key0 + (bx << box_shift);
        // K of the next block comes before V of this one: the lower of the two sets the feed
        const int page = feed.page(p, (w.blk + (v ? j : max(j - 1, 0))) * kKeys, key);
        const int s = n % C::kSlots;
        ok = mbar_wait(&empty[s], ((n / C::kSlots) & 1) ^ 1, kMbarLimitNs);
        if (a == 0 && ok) ok = mbar_wait(q_empty, (pieces & 1) ^ 1, kMbarLimitNs);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t *dst = ring + s * C::kTile;
        if (lane == 0) {
          if (a == 0) {
            const uint32_t bytes = p.tile_tok * p.group * D * 2;
            mbar_arrive_expect_tx(q_full, has_b ? 2 * bytes : bytes);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              if (x && !has_b) break;
#pragma unroll
              for (int c = 0; c < kHalves; ++c)
                tma_load_4d(smem + x * C::kTile + c * kChunk, &tm_q, q_full, 64 * c, w.h * p.group,
                            w.q0 + tok0 + x * p.tile_tok, 0);
            }
          }
          mbar_arrive_expect_tx(&full[s], nbox * box * 128 * kHalves);
        }
        __syncwarp();
        if (bx < nbox)
          tma_load_4d(dst + half * kChunk + (bx << box_shift) * 128, v ? &tm_v : &tm_k, &full[s],
                      half * 64, key & ((1 << p.page_shift) - 1), w.h, page);
      }
      if (!ok) break;
      ++pieces;
      next_unit<kKeys>(p, w, e);
    }
    if (!ok && lane == 0) report_status(p.status, kStatusTmaWait);
    // no TMA write may still be in flight when the CTA exits
    for (int i = max(0, n - C::kSlots); i < n; ++i)
      mbar_wait(&full[i % C::kSlots], (i / C::kSlots) & 1, kMbarLimitNs / 4);
    if (pieces) mbar_wait(q_full, (pieces - 1) & 1, kMbarLimitNs / 4);
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer
      constexpr uint32_t idesc_s = F16 ? idesc_f16_f32(128, 128) : idesc_bf16_f32(128, 128);
      // B (V) MN-major: bit 16
      constexpr uint32_t idesc_o = (F16 ? idesc_f16_f32(128, D) : idesc_bf16_f32(128, D)) | (1u << 16);
      const uint64_t dq = sdesc_kmajor_sw128(smem_u32(smem));
      const uint64_t dk = sdesc_kmajor_sw128(smem_u32(ring));
      const uint64_t dv = sdesc_mnmajor_sw128(smem_u32(ring));
      constexpr uint64_t kTile16 = C::kTile >> 4;
      int base = 0, pieces = 0;  // ring index of the piece's first load
      uint32_t done[2] = {0, 0};  // blocks of each tile so far (a piece may lack the second)
      bool ok = true;
      auto wait_full = [&](int at) {
        return mbar_wait(&full[at % C::kSlots], (at / C::kSlots) & 1, kMbarLimitNs);
      };
      auto issue_qk = [&](int x, int at) {
        tc_fence_after();
        const uint64_t q = dq + x * kTile16, k = dk + (at % C::kSlots) * kTile16;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          // 16 columns of D per step, 64 per chunk
          const uint64_t step = ((kk >> 2) * kChunk + (kk & 3) * 32) >> 4;
          umma_bf16(tmem + 256 * x, q + step, k + step, idesc_s, kk > 0);
        }
        umma_commit(&s_full[x]);
      };
      while (w.pos < w.end && ok) {
        const int e = piece_end(w);
        const int nblk = e - w.blk;
        const int nx = NT > 1 && w.i * p.tpt + p.tile_tok < w.T ? 2 : 1;
        ok = mbar_wait(q_full, pieces & 1, kMbarLimitNs) && wait_full(base);
        if (!ok) break;
        for (int x = 0; x < nx; ++x) issue_qk(x, base);
        umma_commit(&empty[base % C::kSlots]);
        if (nblk == 1) umma_commit(q_empty);
        for (int j = 0; j < nblk && ok; ++j) {
          const int vat = base + v_at(j, nblk), kat = base + k_at(j + 1);
          const bool more = j + 1 < nblk;
          for (int x = 0; x < nx; ++x) {
            const uint32_t par = done[x]++ & 1;
            ok = mbar_wait(&p_ready[x], par, kMbarLimitNs);
            if (ok && x == 0) ok = wait_full(vat);
            if (!ok) break;
            tc_fence_after();
            const uint64_t v = dv + (vat % C::kSlots) * kTile16;
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)  // 16 keys per step
              umma_ts(tmem + 256 * x + 128, tmem + 256 * x + kk * 8, v + ((kk * 2048) >> 4), idesc_o,
                      j > 0 || kk > 0);
            umma_commit(&o_done[x]);
            if (x == nx - 1) umma_commit(&empty[vat % C::kSlots]);
            // QK(x, j+1) overwrites P(x, j); the next piece's first one does, too
            ok = mbar_wait(&o_done[x], par, kMbarLimitNs);
            if (ok && more && x == 0) ok = wait_full(kat);
            if (!ok) break;
            if (more) {
              issue_qk(x, kat);
              if (x == nx - 1) {
                umma_commit(&empty[kat % C::kSlots]);
                if (j + 2 == nblk) umma_commit(q_empty);
              }
            }
          }
        }
        base += 2 * nblk;
        ++pieces;
        next_unit<kKeys>(p, w, e);
      }
      if (!ok) report_status(p.status, kStatusMmaWait);
    }
  } else {
    // ---------------- softmax, epilogue: 128 threads per tile, thread = row
    const int x = (warp - 2) >> 2;
    const int quad = warp & 3;  // TMEM lane quadrant of this warp
    const int row = quad * 32 + lane;
    const uint32_t s_col = tmem + (static_cast<uint32_t>(quad * 32) << 16) + 256 * x;
    const uint32_t o_col = s_col + 128;
    const int rt = row / p.group, rg = row - rt * p.group;
    int base = 0, mine = 0;  // ring index of the piece's first load; blocks of this tile so far
    bool ok = true;
    while (w.pos < w.end) {
      const int e = piece_end(w);
      const int nblk = e - w.blk;
      const int end = kv_end(p, w.T, w.ctx, w.i);
      const int tok0 = w.i * p.tpt + x * p.tile_tok;
      const int ntok = min(p.tile_tok, w.T - tok0);
      if (ntok > 0) {
        const int t = tok0 + rt;
        const bool row_ok = rt < ntok;
        const bool any_row = quad * 32 < ntok * p.group;  // of this warp
        const uint32_t *row_mask = p.mask ? p.mask + (w.q0 + (row_ok ? t : tok0)) * p.ldm : nullptr;
        const int hidden_from = w.ctx + (p.mask ? 0 : tok0 + 1);
        float m_run = -INFINITY, l_run = 0.f;
        for (int j = 0; j < nblk && ok; ++j) {
          const int key0 = (w.blk + j) * kKeys;
          ok = mbar_wait(&s_full[x], (mine + j) & 1, kMbarLimitNs);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (any_row) {
            if (key0 + kKeys > hidden_from)
              softmax_block<D, F16, true>(s_col, o_col, p.scale_log2, j > 0, m_run, l_run, [&](int c) {
                return visible32(p, row_mask, w.T, t, key0 + c * 32 - w.ctx);
              });
            else
              softmax_block<D, F16, false>(s_col, o_col, p.scale_log2, j > 0, m_run, l_run,
                                           [](int) { return 0u; });
          }
          if (x == 0 && key0 + kKeys > end) {
            // V rows behind the last key may be anything (stale or never written memory, whose
            // infinities a zero probability would not cancel): zero them before PV reads them
            const int at = base + v_at(j, nblk);
            ok = mbar_wait(&full[at % C::kSlots], (at / C::kSlots) & 1, kMbarLimitNs);
            const int z0 = end - key0;
            const uint32_t vt = smem_u32(ring + (at % C::kSlots) * C::kTile);
            if (ok)
              for (int u = row; u < (kKeys - z0) * (D / 8); u += 128) {
                const int key = z0 + u / (D / 8), c16 = u % (D / 8);
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                                 vt + (c16 >> 3) * kChunk + key * 128 + (c16 & 7) * 16),
                             "r"(0)
                             : "memory");
              }
            fence_proxy_async_shared();
          }
          tc_fence_before();
          mbar_arrive(&p_ready[x]);
        }
        mine += nblk;
        if (ok) ok = mbar_wait(&o_done[x], (mine - 1) & 1, kMbarLimitNs);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (any_row) {
          const bool whole = w.blk == 0 && e == w.nblk;
          const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
          uint16_t *out = p.out + (w.q0 + t) * p.ldo + static_cast<long>(w.h * p.group + rg) * D;
          const int slot = w.blk == 0, sr = x * 128 + row;
          float *po = slot_o(p, blockIdx.x, slot) + static_cast<long>(sr) * D;
          if (!whole && row_ok) {
            float *ml = slot_ml(p, blockIdx.x, slot);
            ml[sr] = m_run;
            ml[p.rows + sr] = l_run;
          }
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            tmem_ld_32x32(o_col + c * 32, r);
            tmem_wait_ld();
            if (row_ok && whole) {
              uint4 *o4 = reinterpret_cast<uint4 *>(out + c * 32);
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint4 v;
                v.x = pack2<F16>(__uint_as_float(r[q * 8 + 0]) * inv, __uint_as_float(r[q * 8 + 1]) * inv);
                v.y = pack2<F16>(__uint_as_float(r[q * 8 + 2]) * inv, __uint_as_float(r[q * 8 + 3]) * inv);
                v.z = pack2<F16>(__uint_as_float(r[q * 8 + 4]) * inv, __uint_as_float(r[q * 8 + 5]) * inv);
                v.w = pack2<F16>(__uint_as_float(r[q * 8 + 6]) * inv, __uint_as_float(r[q * 8 + 7]) * inv);
                o4[q] = v;
              }
            } else if (row_ok) {
              uint4 *o4 = reinterpret_cast<uint4 *>(po + c * 32);
#pragma unroll
              for (int q = 0; q < 8; ++q)
                o4[q] = make_uint4(r[q * 4], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]);
            }
          }
        }
      }
      base += 2 * nblk;
      const bool goes_on = w.blk == 0 && e < w.nblk;
      if (threadIdx.x == 64 && goes_on) p.desc[blockIdx.x] = split_desc(p, w);
      next_unit<kKeys>(p, w, e);
      // the piece that goes on is this CTA's last
      if (threadIdx.x == 64 && w.pos >= w.end && !goes_on)
        p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    if (threadIdx.x == 64 && (start->pos >= start->end || !ok))
      p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    if (!ok && lane == 0) report_status(p.status, kStatusEpiWait);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// ------------------------------------------------------------------ host side
template <int D, int NT, bool F16>
static void launch(const Params &p, const CUtensorMap &tm_q, const KvMaps &maps, int ctas, int device,
                   cudaStream_t stream) {
  auto *kern = attn_paged_tc_kernel<D, NT, F16>;
  using C = Cfg<D, NT>;
  static bool configured[64] = {false};
  if (!configured[device & 63]) {
    KRB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured[device & 63] = true;
  }
  int box_shift = 0;
  while ((1 << box_shift) < maps.box) ++box_shift;
  kern<<<ctas, C::kThreads, C::kSmem, stream>>>(tm_q, maps.k, maps.v, p, box_shift);
  KRB_CUDA(cudaGetLastError());
}

template <int D, bool F16>
static void launch_nt(const Params &p, const CUtensorMap &tm_q, const KvMaps &maps, int ctas,
                      int device, cudaStream_t stream) {
  if (p.tpt == p.tile_tok) launch<D, 1, F16>(p, tm_q, maps, ctas, device, stream);
  else launch<D, 2, F16>(p, tm_q, maps, ctas, device, stream);
}

void launch_tc(const krb_kv_cache &c, int layer, const Params &p, int ctas, int device,
               cudaStream_t stream) {
  const KvMaps maps = make_kv_maps(c, layer, kKeys);
  const CUtensorMap tm_q = make_tmap_rows(p.q, p.N, p.HQ, p.D, p.ldq, p.tile_tok, p.group);
  const bool f16 = c.dtype == 1;
  if (p.D == 128 && f16) launch_nt<128, true>(p, tm_q, maps, ctas, device, stream);
  else if (p.D == 128) launch_nt<128, false>(p, tm_q, maps, ctas, device, stream);
  else if (f16) launch_nt<64, true>(p, tm_q, maps, ctas, device, stream);
  else launch_nt<64, false>(p, tm_q, maps, ctas, device, stream);
}

}  // namespace paged
}  // namespace krb
