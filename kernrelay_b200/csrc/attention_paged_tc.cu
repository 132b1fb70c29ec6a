// Attention of new tokens over the paged K/V cache, the form for many query rows (wide drafts,
// chunks of a prompt): tcgen05 with S, P and O in TMEM.
//
// A unit is one or two 128-row tiles (whole tokens x the query heads of one KV head) that share
// every K and V block; a block is 64 keys.  Per block and tile: S = Q K^T (both operands K-major in
// shared memory), the tile's 128 softmax threads (thread = row) turn S into P in place, and
// O += P V (P from TMEM, V from shared memory as it lies in the cache, [key][d], so MN-major: no
// transposed copy).  One warp issues all QK, another all PV, and a tile has two S / P stages in
// TMEM: scores are a block ahead of the softmax.
//
// Bound: with R rows the products take 4 R 128 D flop per 128 keys for 512 D bytes of K and V, so to
// about 128 rows HBM binds, beyond it the chip.  Per 128 keys of two tiles the tensor pipe has 2600
// clocks of work (QK at N = 64 reads 6 KB of shared memory per 32 clocks of products, 128 bytes a
// clock are there), MUFU 2100; measured are 4000, since a wait on an mbarrier keeps an issuer from
// feeding the pipe for some 115 clocks even when it has come (its queue holds one or two products).
// A piece's start and end (first scores, last product, O out) cost some 5000 more.
// Measured (calls in a graph, three sets of inputs in turn): 64-token trees (8 sequences of 2 to 8
// thousand positions, 28 query heads over 4 KV heads of 128) 62 to 64 us, 0.32 of their flop at the
// library's rate; two chunks of 1024 tokens over 1 and 8 thousand positions 189 to 200 us, 0.41 to 0.44;
// 8-token trees (32 rows, 169 MB) 38 us, 0.69 of the copy's rate, 64 sequences of them 122 us, 0.84.
// The ring's depth hardly matters: 8-token trees at head_dim 128 take 37.9 us with 8 blocks, 38.0 with
// 10, and without the L2 hint 38.1 with 8, 39.1 with 12 (a deeper queue serves the SMs less evenly);
// wide trees 62.5 with 10, 61.7 with 8, chunks 197 and 196; head_dim 64 (14 heads over 2), 8 / 16 / 24
// blocks: 23.9 / 24.0 / 24.2, wide trees 54.4 / 54.5 / 54.9, chunks 156.7 / 156.9 / 156.1.
// Tried, the trees' and the chunks' time: 128-key blocks with one S stage (70, 205: the chain softmax
// -> PV -> QK), these with half blocks of P (69, 201) and an issuer per tile (79, 215); one issuer for
// all products on two stages (83, 239); QK issuers per tile on two stages (69, 203).
//
#include <algorithm>
#include <string>

#include "attention_paged.cuh"

namespace krb {
namespace paged {

namespace {

constexpr int kKeys = 64;
constexpr uint32_t kQChunk = 128 * 128;   // 128 query rows x 64 elements, bytes
constexpr uint32_t kChunk = kKeys * 128;  // a block's keys x 64 elements, bytes
constexpr int kSoftmaxWarp = 4;           // warps 0: Q and K, 3: V, 1: QK, 2: PV, 4 ..: softmax
constexpr uint32_t kTmemCols = 512;
// The running offset of a row moves (and O is rescaled) only when its maximum grew by more than
// 2^8: P is at most 2^8 in bf16, 2^15 in fp16.
constexpr int kRescaleLog2 = 8;

template <int D, int NT>
struct Cfg {
  static constexpr int kQTile = 256 * D;       // bytes
  static constexpr int kTile = kKeys * D * 2;  // K or V block
  static constexpr int kSlots = D == 64 ? 16 : (NT == 2 ? 10 : 8);
  static constexpr int kThreads = 32 * kSoftmaxWarp + 128 * NT;
  static constexpr int kBars = 2 * kSlots + 2 + 6 * NT;
  static constexpr int kSmem =
      NT * kQTile + kSlots * kTile + kBars * 8 + int(sizeof(Walk)) + 32 + 1024;
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

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0],"
      " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16,"
      " %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
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

// P = 2^(s * scale - off) of 64 scores, packed in the cache's type, and their sum in fp32.
template <bool F16>
__device__ __forceinline__ float exp_block(const uint32_t (&s)[2][32], float scale_log2, float off,
                                           uint32_t (&pk)[32]) {
  const uint64_t sc = pack_f32x2(__float_as_uint(scale_log2), __float_as_uint(scale_log2));
  const uint64_t mo = pack_f32x2(__float_as_uint(-off), __float_as_uint(-off));
  uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    const uint64_t x = pack_f32x2(s[e >> 4][(2 * e) & 31], s[e >> 4][(2 * e + 1) & 31]);
    const float2 a = unpack_f32x2(fma_f32x2(x, sc, mo));
    const float p0 = exp2_mufu(a.x), p1 = exp2_mufu(a.y);
    // P in the cache's type, rounded by up to 2^-8 (bf16) or 2^-11 (fp16) of itself, the largest one
    // too where the offset lags; the row sum takes the fp32 values (the rounded ones gave the same
    // error for a tenth more time)
    pk[e] = pack2<F16>(p0, p1);
    sum[e & 3] = add_f32x2(sum[e & 3], pack_f32x2(__float_as_uint(p0), __float_as_uint(p1)));
  }
  const float2 t = unpack_f32x2(add_f32x2(add_f32x2(sum[0], sum[1]), add_f32x2(sum[2], sum[3])));
  return t.x + t.y;
}

// A block of one row: S (64 columns at s_col) -> P over its first 32 columns.  `see`(c): which of
// the 32 keys of half c the row sees.  P = 2^(s * scale - m + shift) with the row's offset m, which
// moves only by more than kRescaleLog2; O and l follow it.  Behind a piece's first block (`has_o`) the
// exponentials do not wait for the maximum: they are taken with the old m, and once more where it
// moves, which is rare.  A row that has seen nothing yet has m = -inf and takes the offset 0.  `o_ready`
// waits until no product writes O; where that wait runs out (false, for the warp), O is left alone.
template <int D, bool F16, bool kMask, typename See, typename Ready>
__device__ __forceinline__ void softmax_block(uint32_t s_col, uint32_t o_col, float scale_log2,
                                             bool has_o, float &m_run, float &l_run, See see,
                                             Ready o_ready) {
  uint32_t r[2][32];
  tmem_ld_32x32(s_col, r[0]);
  tmem_ld_32x32(s_col + 32, r[1]);
  tmem_wait_ld();
  if constexpr (kMask) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t bits = see(c);
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (!((bits >> e) & 1)) r[c][e] = 0xff800000u;  // -inf
    }
  }
  uint32_t pk[32];
  float sum = 0.f;
  if (has_o) sum = exp_block<F16>(r, scale_log2, p_offset<F16, kRescaleLog2>(m_run), pk);
  float m4[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) m4[e] = fmaxf(__uint_as_float(r[0][e]), __uint_as_float(r[1][e]));
#pragma unroll
  for (int e = 4; e < 32; ++e)
    m4[e & 3] = max3(m4[e & 3], __uint_as_float(r[0][e]), __uint_as_float(r[1][e]));
  const float top = row_max(fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]), scale_log2);
  const bool grow = top - m_run > kRescaleLog2;
  if (!has_o || __any_sync(0xffffffffu, grow)) {
    const float alpha = grow ? exp2_mufu(m_run - top) : 1.f;
    if (grow) m_run = top;
    sum = exp_block<F16>(r, scale_log2, p_offset<F16, kRescaleLog2>(m_run), pk);
    l_run *= alpha;
    if (has_o && o_ready()) {
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        tmem_ld16(o_col + c * 16, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
        tmem_st16(o_col + c * 16, o);
      }
    }
  }
  l_run += sum;
  tmem_st32(s_col, pk);
  tmem_wait_st();
}

// 64 bytes of this thread's row (null: it has none); rows are 16-byte aligned
__device__ __forceinline__ void store_rows(uint8_t *dst, const uint32_t (&v)[16]) {
  if (!dst) return;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    reinterpret_cast<uint4 *>(dst)[q] = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
}

}  // namespace

template <int D, int NT, bool F16>
__global__ void __launch_bounds__(32 * kSoftmaxWarp + 128 * NT, 1)
    attn_paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q,
                         const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const Params p, int box_shift) {
  using C = Cfg<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem =
      reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = smem + NT * C::kQTile;
  uint64_t *full = reinterpret_cast<uint64_t *>(ring + C::kSlots * C::kTile);
  uint64_t *empty = full + C::kSlots;
  uint64_t *q_full = empty + C::kSlots;
  uint64_t *q_empty = q_full + 1;
  uint64_t *s_full = q_empty + 1;       // [tile][stage], like the next two
  uint64_t *p_ready = s_full + 2 * NT;
  uint64_t *o_done = p_ready + 2 * NT;  // PV of the stage's P
  Walk *start = reinterpret_cast<Walk *>(o_done + 2 * NT);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(start + 1);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2 * NT; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 128);
      mbar_init(&o_done[i], 1);
    }
    fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  pdl_wait();
  pdl_launch_dependents();
  if (warp >= 2) prefetch_page_table(p, threadIdx.x - 64, C::kThreads - 64);
  if (warp == 0) {
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

  if (warp == 0 || warp == 3) {
    // ---------------- producers: warp 0 brings Q and K, warp 3 V; one lane issues the boxes (page x
    // 64 columns).  TMA takes its operands from uniform registers: boxes of several lanes would be
    // issued one by one all the same, at 100 to 200 clocks each.
    const bool v = warp == 3;
    const int box = 1 << box_shift;
    const uint32_t box_bytes = box * 128;
    PageFeed feed;
    // one tile: the keys are first to leave L2 (attention_paged.cu; 39.1 -> 37.2 us for 8-token trees).
    // With two, units share a sequence's keys: it gained nothing.
    uint64_t policy = 0;
    if constexpr (NT == 1) policy = l2_policy_evict_first();
    int base = 0, pieces = 0;  // ring index of the piece's first load
    int last = -1;             // ring index of this warp's last load
    bool ok = true;
    while (w.pos < w.end) {
      const int e = piece_end(w);
      const int nblk = e - w.blk;
      const int end = kv_end(p, w.T, w.ctx, w.i);
      const int tok0 = w.i * p.tpt;
      feed.begin(p, w.b, w.blk * kKeys, min(end, e * kKeys));
      if (!v) {
        const bool has_b = NT > 1 && tok0 + p.tile_tok < w.T;
        ok = mbar_wait_warp(q_empty, (pieces & 1) ^ 1);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t bytes = p.tile_tok * p.group * D * 2;
          mbar_arrive_expect_tx(q_full, has_b ? 2 * bytes : bytes);
          for (int x = 0; x < (has_b ? 2 : 1); ++x)
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_4d(smem + x * C::kQTile + c * kQChunk, &tm_q, q_full, 64 * c, w.h * p.group,
                          w.q0 + tok0 + x * p.tile_tok, 0);
        }
      }
      for (int j = 0; j < nblk; ++j) {
        const int at = base + (v ? v_at(j, nblk) : k_at(j));
        const int s = at % C::kSlots;
        const int key0 = (w.blk + j) * kKeys;
        const int nbox = (min(kKeys, end - key0) + box - 1) >> box_shift;
        feed.advance(p, key0);
        ok = mbar_wait_warp(&empty[s], ((at / C::kSlots) & 1) ^ 1);
        if (!ok) break;
        const bool lead = elect_one();
        if (lead) mbar_arrive_expect_tx(&full[s], nbox * box_bytes * (D / 64));
        const CUtensorMap *map = v ? &tm_v : &tm_k;
        for (int i = 0; i < nbox; ++i) {
          const int key = key0 + (i << box_shift);
          const int page = feed.page(p, key), slot = key & ((1 << p.page_shift) - 1);
          if (lead) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              if constexpr (NT == 1)
                tma_load_4d_hint(ring + s * C::kTile + c * kChunk + i * box_bytes, map, &full[s],
                                 64 * c, slot, w.h, page, policy);
              else
                tma_load_4d(ring + s * C::kTile + c * kChunk + i * box_bytes, map, &full[s], 64 * c,
                            slot, w.h, page);
          }
        }
        last = at;
      }
      if (!ok) break;
      base += 2 * nblk;
      ++pieces;
      next_unit<kKeys>(p, w, e);
    }
    if (!ok && lane == 0) report_status(p.status, kStatusTmaWait);
    // No TMA write may still be in flight when the CTA exits.  Every load is waited for by an issuer;
    // after a wait that ran out, give this warp's own (a slot has been given back only when its load
    // was complete, so a phase that is not there any more costs the limit and no more).
    if (!ok && last >= 0)
      for (int i = max(0, last - C::kSlots + 1); i <= last; ++i)
        mbar_wait(&full[i % C::kSlots], (i / C::kSlots) & 1, kMbarLimitNs / 64);
    if (!ok && !v && pieces) mbar_wait(q_full, (pieces - 1) & 1, kMbarLimitNs / 64);
  } else if (warp == 1) {
    // ---------------- QK issuer (one thread)
    if (lane == 0) {
      constexpr uint32_t idesc = F16 ? idesc_f16_f32(128, kKeys) : idesc_bf16_f32(128, kKeys);
      const uint64_t dq = sdesc_kmajor_sw128(smem_u32(smem));
      const uint64_t dk = sdesc_kmajor_sw128(smem_u32(ring));
      int base = 0, pieces = 0;   // ring index of the piece's first load; pieces
      uint32_t done[2] = {0, 0};  // blocks of each tile so far (a piece may lack the second)
      bool ok = true;
      while (w.pos < w.end && ok) {
        const int e = piece_end(w);
        const int n = e - w.blk;
        const int nx = NT > 1 && w.i * p.tpt + p.tile_tok < w.T ? 2 : 1;
        ok = mbar_wait(q_full, pieces & 1, kMbarLimitNs);
        for (int j = 0; j < n && ok; ++j) {
          const int at = (base + k_at(j)) % C::kSlots;
          ok = mbar_wait(&full[at], ((base + k_at(j)) / C::kSlots) & 1, kMbarLimitNs);
          const uint64_t k = dk + at * (C::kTile >> 4);
          for (int x = 0; x < nx && ok; ++x) {
            const uint32_t c = done[x]++, stage = c & 1;
            // S overwrites the P of the tile's block before last
            if (c >= 2) ok = mbar_wait(&o_done[2 * x + stage], ((c >> 1) - 1) & 1, kMbarLimitNs);
            if (!ok) break;
            tc_fence_after();
            const uint64_t q = dq + ((x * C::kQTile) >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)  // 16 columns of D per step, 64 per chunk
              umma_bf16(tmem + 256 * x + 64 * stage, q + (((kk >> 2) * kQChunk + (kk & 3) * 32) >> 4),
                        k + (((kk >> 2) * kChunk + (kk & 3) * 32) >> 4), idesc, kk > 0);
            umma_commit(&s_full[2 * x + stage]);
          }
          if (ok) umma_commit(&empty[at]);
        }
        if (ok) umma_commit(q_empty);
        base += 2 * n;
        ++pieces;
        next_unit<kKeys>(p, w, e);
      }
      if (!ok) report_status(p.status, kStatusMmaWait);
    }
  } else if (warp == 2) {
    // ---------------- PV issuer (lane 0; the other lanes keep step: they zero the rows of V behind
    // the last key)
    constexpr uint32_t idesc =
        (F16 ? idesc_f16_f32(128, D) : idesc_bf16_f32(128, D)) | (1u << 16);  // B (V) MN-major
    const uint64_t dv = sdesc_mnmajor_sw128(smem_u32(ring));
    int base = 0;
    uint32_t done[2] = {0, 0};
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t parity) { return ok = mbar_wait_warp(bar, parity); };
    while (w.pos < w.end && ok) {
      const int e = piece_end(w);
      const int n = e - w.blk;
      const int end = kv_end(p, w.T, w.ctx, w.i);
      const int nx = NT > 1 && w.i * p.tpt + p.tile_tok < w.T ? 2 : 1;
      for (int j = 0; j < n; ++j) {
        const int at = (base + v_at(j, n)) % C::kSlots;
        const int z0 = end - (w.blk + j) * kKeys;  // keys of the block that are there
        if (!wait(&full[at], ((base + v_at(j, n)) / C::kSlots) & 1)) break;
        if (z0 < kKeys) {
          // V rows behind the last key may be anything (stale or never written memory, whose
          // infinities a zero probability would not cancel): zero them
          const uint32_t vt = smem_u32(ring + at * C::kTile);
          for (int u = lane; u < (kKeys - z0) * (D / 8); u += 32) {
            const int key = z0 + u / (D / 8), c16 = u % (D / 8);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             vt + (c16 >> 3) * kChunk + key * 128 + (c16 & 7) * 16),
                         "r"(0)
                         : "memory");
          }
          fence_proxy_async_shared();
          __syncwarp();
        }
        const uint64_t v = dv + at * (C::kTile >> 4);
        for (int x = 0; x < nx; ++x) {
          const uint32_t c = done[x]++, stage = c & 1;
          if (!wait(&p_ready[2 * x + stage], (c >> 1) & 1)) break;
          tc_fence_after();
          if (lane == 0) {
#pragma unroll
            for (int kk = 0; kk < kKeys / 16; ++kk)  // 16 keys (8 columns of P) per step
              umma_ts(tmem + 256 * x + 128, tmem + 256 * x + 64 * stage + kk * 8,
                      v + ((kk * 2048) >> 4), idesc, j > 0 || kk > 0);
            umma_commit(&o_done[2 * x + stage]);
          }
        }
        if (!ok) break;
        if (lane == 0) umma_commit(&empty[at]);
      }
      base += 2 * n;
      next_unit<kKeys>(p, w, e);
    }
    if (!ok && lane == 0) report_status(p.status, kStatusMmaWait);
  } else if (warp >= kSoftmaxWarp) {
    // ---------------- softmax, epilogue: 128 threads per tile, thread = row
    const int x = (warp - kSoftmaxWarp) >> 2;
    const int quad = warp & 3;  // TMEM lane quadrant of this warp
    const int row = quad * 32 + lane;
    const uint32_t s_col = tmem + (static_cast<uint32_t>(quad * 32) << 16) + 256 * x;
    const uint32_t o_col = s_col + 128;
    const int rt = row / p.group, rg = row - rt * p.group;
    int mine = 0;  // blocks of this tile so far
    bool ok = true;
    while (w.pos < w.end) {
      const int e = piece_end(w);
      const int nblk = e - w.blk;
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
          const int c = mine + j, stage = c & 1;  // blocks of this tile before this one
          ok = mbar_wait_warp(&s_full[2 * x + stage], (c >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (any_row) {
            // PV of the block before (that of the one before it is complete: this S came after it).
            // Where it does not come, O stays untouched and the warp leaves after this block; nothing is
            // stored.
            auto o_ready = [&] {
              ok = mbar_wait_warp(&o_done[2 * x + (stage ^ 1)], ((c - 1) >> 1) & 1);
              tc_fence_after();
              return ok;
            };
            if (key0 + kKeys > hidden_from)
              softmax_block<D, F16, true>(
                  s_col + 64 * stage, o_col, p.scale_log2, j > 0, m_run, l_run,
                  [&](int q) { return visible32(p, row_mask, w.T, t, key0 + q * 32 - w.ctx); }, o_ready);
            else
              softmax_block<D, F16, false>(s_col + 64 * stage, o_col, p.scale_log2, j > 0, m_run, l_run,
                                           [](int) { return 0u; }, o_ready);
          }
          tc_fence_before();
          mbar_arrive(&p_ready[2 * x + stage]);
        }
        mine += nblk;
        if (ok) ok = mbar_wait_warp(&o_done[2 * x + ((mine - 1) & 1)], ((mine - 1) >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        if (any_row) {
          const bool whole = w.blk == 0 && e == w.nblk;
          if (whole) {
            const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
            uint16_t *out = p.out + (w.q0 + t) * p.ldo + static_cast<long>(w.h * p.group + rg) * D;
            uint32_t r[2][32], v[16];
            tmem_ld_32x32(o_col, r[0]);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              tmem_wait_ld();
              if (c + 1 < D / 32) tmem_ld_32x32(o_col + (c + 1) * 32, r[(c + 1) & 1]);
#pragma unroll
              for (int q = 0; q < 16; ++q)
                v[q] = pack2<F16>(__uint_as_float(r[c & 1][2 * q]) * inv,
                                  __uint_as_float(r[c & 1][2 * q + 1]) * inv);
              store_rows(row_ok ? reinterpret_cast<uint8_t *>(out + c * 32) : nullptr, v);
            }
          } else {
            // O of a piece lies in 16-byte columns [D / 4][rows][4]: a warp's 32 rows side by side
            // (row by row, each store touched 32 lines and a piece's end took 8000 clocks)
            const int slot = w.blk == 0, sr = x * 128 + row;
            float4 *po = reinterpret_cast<float4 *>(slot_o(p, blockIdx.x, slot)) + sr;
            if (row_ok) {
              float *ml = slot_ml(p, blockIdx.x, slot);
              ml[sr] = m_run;
              ml[p.rows + sr] = l_run;
            }
            uint32_t r[2][32];
            tmem_ld_32x32(o_col, r[0]);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              tmem_wait_ld();
              if (c + 1 < D / 32) tmem_ld_32x32(o_col + (c + 1) * 32, r[(c + 1) & 1]);
              const uint32_t(&v)[32] = r[c & 1];
              if (row_ok) {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                  po[(c * 8 + q) * p.rows] =
                      make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]),
                                  __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3]));
              }
            }
          }
        }
      }
      const bool goes_on = w.blk == 0 && e < w.nblk;
      if (threadIdx.x == 32 * kSoftmaxWarp && goes_on) p.desc[blockIdx.x] = split_desc(p, w);
      next_unit<kKeys>(p, w, e);
      // the piece that goes on is this CTA's last
      if (threadIdx.x == 32 * kSoftmaxWarp && w.pos >= w.end && !goes_on)
        p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    if (threadIdx.x == 32 * kSoftmaxWarp && (start->pos >= start->end || !ok))
      p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    if (!ok && lane == 0) report_status(p.status, kStatusEpiWait);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// ------------------------------------------------------------------ joining split units
// CTA (c, y, z) joins slot rows 32 y .. and columns z D / 4 .. of the unit that CTA c of the attention
// kernel began and later ones went on with: a lane per row, a warp per D / 16 columns,
// O = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k.
template <int D, bool F16>
__global__ void __launch_bounds__(128) combine_tc_kernel(const Params p) {
  constexpr int kCols = D / 64;  // 16-byte columns of a lane
  constexpr int kAhead = 4;      // pieces loaded at a time
  pdl_wait();
  const int c = blockIdx.x;
  const int4 d = p.desc[c];
  if (d.w < 2) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sr = blockIdx.y * 32 + lane, col = (blockIdx.z * 4 + warp) * kCols;
  const int tile = sr >> 7, rt = (sr & 127) / p.group, rg = (sr & 127) - rt * p.group;
  const int tok = tile * p.tile_tok + rt;
  if (rt >= p.tile_tok || tok >= d.y) return;
  // running maximum over the groups of pieces
  float mx = -INFINITY, total = 0.f;
  float4 acc[kCols];
#pragma unroll
  for (int q = 0; q < kCols; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < d.w; k0 += kAhead) {
    float m[kAhead], l[kAhead];
    float4 v[kAhead][kCols];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int k = k0 + u;
      m[u] = -INFINITY;
      if (k >= d.w) continue;
      const float *ml = slot_ml(p, c + k, k == 0);
      m[u] = ml[sr];
      l[u] = ml[p.rows + sr];
      const float4 *o = reinterpret_cast<const float4 *>(slot_o(p, c + k, k == 0)) + sr;
#pragma unroll
      for (int q = 0; q < kCols; ++q) v[u][q] = o[(col + q) * p.rows];
    }
    float top = mx;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) top = fmaxf(top, m[u]);
    const float off = top == -INFINITY ? 0.f : top;
    const float keep = exp2_mufu(mx - off);
    mx = top;
    total *= keep;
#pragma unroll
    for (int q = 0; q < kCols; ++q)
      acc[q] = make_float4(acc[q].x * keep, acc[q].y * keep, acc[q].z * keep, acc[q].w * keep);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (k0 + u >= d.w) continue;
      const float f = exp2_mufu(m[u] - off);
      total += f * l[u];
#pragma unroll
      for (int q = 0; q < kCols; ++q) {
        acc[q].x += f * v[u][q].x;
        acc[q].y += f * v[u][q].y;
        acc[q].z += f * v[u][q].z;
        acc[q].w += f * v[u][q].w;
      }
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  uint16_t *out = p.out + (d.x + tok) * p.ldo + static_cast<long>(d.z * p.group + rg) * D + col * 4;
#pragma unroll
  for (int q = 0; q < kCols; ++q)
    *reinterpret_cast<uint2 *>(out + q * 4) = make_uint2(pack2<F16>(acc[q].x * inv, acc[q].y * inv),
                                                         pack2<F16>(acc[q].z * inv, acc[q].w * inv));
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
  launch_pdl(kern, dim3(ctas), C::kThreads, C::kSmem, stream, false, tm_q, maps.k, maps.v, p, box_shift);
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
  auto *kern = p.D == 128 ? (f16 ? combine_tc_kernel<128, true> : combine_tc_kernel<128, false>)
                          : (f16 ? combine_tc_kernel<64, true> : combine_tc_kernel<64, false>);
  launch_pdl(kern, dim3(ctas, p.rows / 32, 4), 128, 0, stream, true, p);
}

}  // namespace paged
}  // namespace krb
