// Attention of new tokens over the paged K/V cache: the form for few query rows (a token or a
// small draft per sequence) on mma.sync, the kernel that joins split units, and the host side.
//
// Few rows are bound by reading K and V once: a 64-key block of one KV head is 32 KB at head_dim 128,
// 0.75 us of one SM's share of HBM bandwidth, against 0.14 us of mma.sync for a 16-row tile.  So the
// kernel is a ring of TMA loads (two CTAs of two 32 KB stages per SM; a third only deepens the queue
// at the memory, which then serves the SMs less evenly: 110.6 us against 108.3 in the first case
// below), the rows of all query heads that share a KV head go through the tensor cores together, and
// the four warps of a CTA split the keys, so that a block costs each a quarter.
// Measured (calls in a graph, three sets of inputs in turn): 64 sequences of 2 to 8 thousand positions,
// 28 query heads over 4 KV heads of 128, 106 us, 97 % of the copy's rate for 659 MB; 2 sequences of 98 and
// 131 thousand, 77 us, 94 %.  One call after the other through the Python wrapper: 109 and 78.6 us.
#include <algorithm>
#include <string>

#include "attention_paged.cuh"

namespace krb {
namespace paged {

namespace {

constexpr int kKeys = 64;        // keys of a block
constexpr int kThreads = 160;    // 4 consumer warps, 1 producer warp
constexpr int kConsumers = 128;

template <int D>
struct Cfg {
  static constexpr int kHalf = kKeys * 128;             // 64 keys x 64 elements, bytes
  static constexpr int kTile = kKeys * D * 2;           // K or V block
  static constexpr int kStages = D == 128 ? 2 : 4;      // 64 KB of ring: see the top
  static constexpr int kMergeLane = D / 16 * 4 + 4;     // floats per lane: half of O, m and l
  static constexpr int kMerge = kMergeLane * 32 * 4;    // bytes per sending warp
  static constexpr int kBars = 2 * kStages * 8;
  static constexpr int kSmem =
      2 * kStages * kTile + 2 * kMerge + kBars + 5 * int(sizeof(Walk)) + 16 + 1024;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
        " {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
        " {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// byte offset of 16-byte chunk `chunk` of key row `key` in a block (128-byte swizzle)
template <int D>
__device__ __forceinline__ uint32_t tile_off(int key, int chunk) {
  return (chunk >> 3) * Cfg<D>::kHalf + key * 128 + (((chunk & 7) ^ (key & 7)) << 4);
}

}  // namespace

// Warp (wm, wn) of the WM x (4 / WM) consumer warps (WM 1 or 2): rows 16 wm .. +15 of the unit, keys
// wn * 16 WM .. of every block.  A lane holds rows g = lane / 4 and g + 8 (mma fragments).
template <int D, int WM, bool F16>
__global__ void __launch_bounds__(kThreads, 2)
    attn_paged_kernel(const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const Params p, int box_shift) {
  using C = Cfg<D>;
  constexpr int WN = 4 / WM;
  constexpr int kWarpKeys = kKeys / WN;
  constexpr int NT = kWarpKeys / 8;  // 8-key score tiles of a warp
  constexpr int DT = D / 8;          // 8-column output tiles
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem =
      reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *merge = reinterpret_cast<float *>(smem + 2 * C::kStages * C::kTile);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + 2 * C::kStages * C::kTile + 2 * C::kMerge);
  uint64_t *empty = full + C::kStages;
  Walk *start = reinterpret_cast<Walk *>(empty + C::kStages);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    fence_mbar_init();
  }
  pdl_wait();
  pdl_launch_dependents();
  if (warp < 4) prefetch_page_table(p, threadIdx.x, kConsumers);
  if (warp == 4) {
    const Walk s = find_start<kKeys>(p, blockIdx.x, gridDim.x);
    if (lane == 0) *start = s;
  }
  __syncthreads();

  if (warp == 4) {
    Walk w = *start;
    // ---------------- producer: one lane issues a stage's boxes (page x 64 columns, K and V).  A
    // box per lane would be slower: TMA takes its operands from uniform registers, so the lanes'
    // copies are issued one by one all the same, at 100 to 200 clocks each.
    const int box = 1 << box_shift;
    const uint32_t box_bytes = box * 128;
    PageFeed feed;
    // The keys are first to leave L2.  Without / with: 64 decoding sequences 108.1 / 104.6 us, two long
    // ones 77.5 / 76.1, 64 sequences that share 2000, 8000 or 32000 positions 99.9 / 98.2, 114.1 / 112.0
    // and 390.6 / 381.4, 16 of 4000 (131 MB) 30.1 / 28.0; caches that stay in L2 between calls, alone or
    // beside 30 to 120 MB of other reads, take the same or less.
    const uint64_t policy = l2_policy_evict_first();
    int n = 0;  // blocks issued
    bool ok = true;
    while (w.pos < w.end && ok) {
      const int e = piece_end(w);
      const int end = kv_end(p, w.T, w.ctx, w.i);
      feed.begin(p, w.b, w.blk * kKeys, min(end, e * kKeys));
      for (int blk = w.blk; blk < e; ++blk, ++n) {
        const int s = n % C::kStages;
        const int key0 = blk * kKeys;
        const int nbox = (min(kKeys, end - key0) + box - 1) >> box_shift;
        feed.advance(p, key0);
        ok = mbar_wait_warp(&empty[s], ((n / C::kStages) & 1) ^ 1);
        if (!ok) break;
        uint8_t *stage = smem + s * 2 * C::kTile;
        const bool lead = elect_one();
        if (lead) mbar_arrive_expect_tx(&full[s], nbox * box_bytes * (D / 64 * 2));
        for (int i = 0; i < nbox; ++i) {
          const int key = key0 + (i << box_shift);
          const int page = feed.page(p, key), slot = key & ((1 << p.page_shift) - 1);
          uint8_t *to = stage + i * box_bytes;
          if (lead) {
#pragma unroll
            for (int half = 0; half < D / 64; ++half) {
              tma_load_4d_hint(to + half * C::kHalf, &tm_k, &full[s], half * 64, slot, w.h, page,
                               policy);
              tma_load_4d_hint(to + C::kTile + half * C::kHalf, &tm_v, &full[s], half * 64, slot, w.h, page,
                               policy);
            }
          }
        }
      }
      if (ok) next_unit<kKeys>(p, w, e);
    }
    if (!ok && lane == 0) report_status(p.status, kStatusTmaWait);
    // no TMA write may still be in flight when the CTA exits
    for (int i = max(0, n - C::kStages); i < n; ++i)
      mbar_wait(&full[i % C::kStages], (i / C::kStages) & 1, kMbarLimitNs / 4);
    return;
  }

  // ---------------- consumers
  const int wm = warp % WM, wn = warp / WM;
  const int g = lane >> 2, c2 = (lane & 3) * 2;
  const uint32_t base = smem_u32(smem);
  // the walk lies in shared memory, a copy per warp: the block loop wants the registers
  volatile Walk *vw = start + 1 + warp;
  auto load_walk = [&] {
    Walk w;
    w.b = vw->b, w.h = vw->h, w.i = vw->i, w.q0 = vw->q0, w.T = vw->T, w.ctx = vw->ctx;
    w.blk = vw->blk, w.nblk = vw->nblk, w.pos = vw->pos, w.end = vw->end, w.per = vw->per;
    return w;
  };
  auto store_walk = [&](const Walk &w) {
    __syncwarp();
    if (lane == 0) {
      vw->b = w.b, vw->h = w.h, vw->i = w.i, vw->q0 = w.q0, vw->T = w.T, vw->ctx = w.ctx;
      vw->blk = w.blk, vw->nblk = w.nblk, vw->pos = w.pos, vw->end = w.end, vw->per = w.per;
    }
    __syncwarp();
  };
  store_walk(*start);
  int n = 0;
  bool ok = true;
  while (vw->pos < vw->end) {
    int e, end, first_hidden;  // piece's end; unit's last key + 1; first key that a row may not see
    uint32_t qf[D / 16][4];
    {
      const Walk w = load_walk();
      e = piece_end(w);
      end = kv_end(p, w.T, w.ctx, w.i);
      const int tok0 = w.i * p.tpt;
      first_hidden = w.ctx + (p.mask ? 0 : tok0 + 1);
      const int nrows = min(p.tpt, w.T - tok0) * p.group;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        // rows g and g + 8 of this warp's tile
        const int r = wm * 16 + g + 8 * x;
        const bool there = r < nrows;
        const uint16_t *q = p.q + (w.q0 + tok0 + r / p.group) * p.ldq +
                            static_cast<long>(w.h * p.group + r % p.group) * D + c2;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          qf[ks][x] = there ? __ldg(reinterpret_cast<const uint32_t *>(q + ks * 16)) : 0u;
          qf[ks][2 + x] = there ? __ldg(reinterpret_cast<const uint32_t *>(q + ks * 16 + 8)) : 0u;
        }
      }
    }
    float o[DT][4];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[d][x] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int blk = vw->blk; blk < e; ++blk, ++n) {
      const int s = n % C::kStages;
      if (ok) ok = mbar_wait_warp(&full[s], (n / C::kStages) & 1);
      if (!ok) continue;  // leave the waits, keep the CTA's barriers in step
      const int k0 = blk * kKeys + wn * kWarpKeys;  // this warp's first key
      const uint32_t kt = base + s * 2 * C::kTile, vt = kt + C::kTile;
      const bool wrote = k0 + kWarpKeys > end;
      if (wrote) {
        // V rows behind the last key may be anything (stale or never written memory, whose
        // infinities a zero probability would not cancel): zero them
        const int z0 = max(k0, end) - blk * kKeys, z1 = (wn + 1) * kWarpKeys;
        for (int u = lane; u < (z1 - z0) * (D / 8); u += 32) {
          const int key = z0 + u / (D / 8);
          const uint32_t at = vt + tile_off<D>(key, u % (D / 8));
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
        }
        __syncwarp();
      }
      if (k0 < end) {
        float sc[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[t][x] = 0.f;
        // fragments are fetched a step ahead: two warps per scheduler do not hide ldmatrix
        const int krow = wn * kWarpKeys + (lane >> 4) * 8 + (lane & 7);
        uint32_t kb[2][NT / 2][4];
        auto load_k = [&](int ks) {
#pragma unroll
          for (int t = 0; t < NT; t += 2)
            ldsm4(kt + tile_off<D>(krow + t * 8, 2 * ks + ((lane >> 3) & 1)), kb[ks & 1][t / 2]);
        };
        load_k(0);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          if (ks + 1 < D / 16) load_k(ks + 1);
#pragma unroll
          for (int t = 0; t < NT; ++t)
            mma16816<F16>(sc[t], qf[ks], kb[ks & 1][t / 2][(t & 1) * 2], kb[ks & 1][t / 2][(t & 1) * 2 + 1]);
        }
        if (k0 + kWarpKeys > first_hidden) {
          const int T = vw->T, ctx = vw->ctx, tok0 = vw->i * p.tpt;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int t = tok0 + (wm * 16 + g + 8 * x) / p.group;
            const uint32_t *row_mask =
                p.mask ? p.mask + (vw->q0 + (t < T ? t : tok0)) * p.ldm : nullptr;
#pragma unroll
            for (int k = 0; k < kWarpKeys; k += 32) {
              const uint32_t see = visible32(p, row_mask, T, t, k0 + k - ctx);
#pragma unroll
              for (int t8 = k / 8; t8 < NT && t8 < k / 8 + 4; ++t8)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                  if (!((see >> (t8 * 8 - k + c2 + y)) & 1)) sc[t8][2 * x + y] = -INFINITY;
            }
          }
        }
        constexpr int kVSteps = D / 32;  // steps of 16 keys x 32 columns
        const int vrow = wn * kWarpKeys + ((lane >> 3) & 1) * 8 + (lane & 7);
        uint32_t vb[2][2][4];
        auto load_v = [&](int i) {
#pragma unroll
          for (int d = 0; d < 2; ++d)
            ldsm4_t(vt + tile_off<D>(vrow + i / kVSteps * 16, (i % kVSteps) * 4 + d * 2 + (lane >> 4)),
                    vb[i & 1][d]);
        };
        load_v(0);
        float mx[2] = {m[0], m[1]};
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          top[0] = fmaxf(top[0], fmaxf(sc[t][0], sc[t][1]));
          top[1] = fmaxf(top[1], fmaxf(sc[t][2], sc[t][3]));
        }
        float off[2], alpha[2];
        bool moved = false;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
          top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2));
          m[x] = fmaxf(m[x], row_max(top[x], p.scale_log2));
          // a row that has seen nothing yet has no maximum: any offset gives its zeros
          off[x] = m[x] == -INFINITY ? 0.f : m[x];
          alpha[x] = exp2_mufu(mx[x] - off[x]);
          moved |= m[x] != mx[x];
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int x = 0; x < 2; ++x) l[x] *= alpha[x];
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            o[d][0] *= alpha[0];
            o[d][1] *= alpha[0];
            o[d][2] *= alpha[1];
            o[d][3] *= alpha[1];
          }
        }
        // P enters the second product in the cache's type, rounded by up to 2^-8 (bf16) or 2^-11
        // (fp16) of itself; a row's largest is a power of two, so exact.  The row sum takes the
        // fp32 values.
        uint32_t pf[NT / 2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) off[x] = p_offset<F16, 0>(m[x]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float p0 = exp2_mufu(fmaf(sc[t][2 * x], p.scale_log2, -off[x]));
            const float p1 = exp2_mufu(fmaf(sc[t][2 * x + 1], p.scale_log2, -off[x]));
            l[x] += p0 + p1;
            pf[t / 2][(t & 1) * 2 + x] = pack2<F16>(p0, p1);
          }
        }
#pragma unroll
        for (int i = 0; i < NT / 2 * kVSteps; ++i) {
          if (i + 1 < NT / 2 * kVSteps) load_v(i + 1);
          const int ks = i / kVSteps, d0 = i % kVSteps * 4;
#pragma unroll
          for (int d = 0; d < 4; ++d)
            mma16816<F16>(o[d0 + d], pf[ks], vb[i & 1][d / 2][(d & 1) * 2], vb[i & 1][d / 2][(d & 1) * 2 + 1]);
        }
      }
      if (wrote) fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
    }

    if constexpr (WN > 1) {
      // the warps that share rows join: O in two halves (one fragment register of all lanes side
      // by side, so no bank conflicts), wn 2, 3 -> 0, 1, then 1 -> 0 (WN = 2: 1 -> 0)
      float fa[2][2], fb[2][2];  // per step and row: factors of the own and of the received O
      auto send = [&](float *buf, int h) {
#pragma unroll
        for (int d = 0; d < DT / 2; ++d)
          reinterpret_cast<float4 *>(buf)[d * 32 + lane] =
              make_float4(o[h * DT / 2 + d][0], o[h * DT / 2 + d][1], o[h * DT / 2 + d][2],
                          o[h * DT / 2 + d][3]);
        reinterpret_cast<float4 *>(buf)[DT / 2 * 32 + lane] = make_float4(m[0], m[1], l[0], l[1]);
      };
      auto take = [&](const float *buf, int h, int step) {
        if (h == 0) {
          const float4 v = reinterpret_cast<const float4 *>(buf)[DT / 2 * 32 + lane];
          const float vm[2] = {v.x, v.y}, vl[2] = {v.z, v.w};
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float mm = fmaxf(m[x], vm[x]);
            const float off = mm == -INFINITY ? 0.f : mm;
            fa[step][x] = exp2_mufu(m[x] - off);
            fb[step][x] = exp2_mufu(vm[x] - off);
            m[x] = mm;
            l[x] = l[x] * fa[step][x] + vl[x] * fb[step][x];
          }
        }
#pragma unroll
        for (int d = 0; d < DT / 2; ++d) {
          const float4 v = reinterpret_cast<const float4 *>(buf)[d * 32 + lane];
          float(&t)[4] = o[h * DT / 2 + d];
          t[0] = t[0] * fa[step][0] + v.x * fb[step][0];
          t[1] = t[1] * fa[step][0] + v.y * fb[step][0];
          t[2] = t[2] * fa[step][1] + v.z * fb[step][1];
          t[3] = t[3] * fa[step][1] + v.w * fb[step][1];
        }
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float *buf = merge + (warp & 1) * (C::kMerge / 4);
        float *buf1 = merge + C::kMerge / 4;
        named_bar_sync(1, kConsumers);  // the buffers' last readers are done
        if (warp >= 2) send(buf, h);
        named_bar_sync(1, kConsumers);
        if (warp < 2) take(buf, h, 0);
        if constexpr (WN == 4) {
          if (warp == 1) send(buf1, h);
          named_bar_sync(1, kConsumers);
          if (warp == 0) take(buf1, h, 1);
        }
      }
    }

    Walk w = load_walk();
    if (wn == 0 && ok) {
      const bool whole = w.blk == 0 && e == w.nblk;
      const int tok0 = w.i * p.tpt;
      const int nrows = min(p.tpt, w.T - tok0) * p.group;
      const int slot = w.blk == 0;
      float *ml = slot_ml(p, blockIdx.x, slot);
      float *po = slot_o(p, blockIdx.x, slot);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = wm * 16 + g + 8 * x;
        if (r >= nrows) continue;
        if (whole) {
          const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
          uint16_t *out = p.out + (w.q0 + tok0 + r / p.group) * p.ldo +
                          static_cast<long>(w.h * p.group + r % p.group) * D + c2;
#pragma unroll
          for (int d = 0; d < DT; ++d)
            *reinterpret_cast<uint32_t *>(out + d * 8) =
                pack2<F16>(o[d][2 * x] * inv, o[d][2 * x + 1] * inv);
        } else {
          if ((lane & 3) == 0) {
            ml[r] = m[x];
            ml[p.rows + r] = l[x];
          }
#pragma unroll
          for (int d = 0; d < DT; ++d)
            *reinterpret_cast<float2 *>(po + r * D + d * 8 + c2) =
                make_float2(o[d][2 * x], o[d][2 * x + 1]);
        }
      }
    }
    const bool goes_on = w.blk == 0 && e < w.nblk;
    if (threadIdx.x == 0 && goes_on) p.desc[blockIdx.x] = split_desc(p, w);
    next_unit<kKeys>(p, w, e);
    // the piece that goes on is this CTA's last
    if (threadIdx.x == 0 && w.pos >= w.end && !goes_on) p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    store_walk(w);
  }
  if (start->pos >= start->end && threadIdx.x == 0) p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
  if (!ok && lane == 0) report_status(p.status, kStatusEpiWait);
}

// ------------------------------------------------------------------ joining split units
// CTA (c, r) joins row r of the unit that CTA c of the attention kernel began and later ones went on
// with: each of its warps takes every fourth piece (a long sequence over few units is cut into
// dozens; one warp alone took 12 us for 37 pieces), then their sums in order;
// O = sum_k 2^(m_k - M) O_k / sum_k 2^(m_k - M) l_k.
template <int D, bool F16>
__global__ void __launch_bounds__(128) combine_kernel(const Params p) {
  constexpr int V = D / 32;  // columns of a lane
  constexpr int KW = 4, kUnroll = 4;
  __shared__ float part[KW][32][V + 1];
  pdl_wait();
  const int c = blockIdx.x;
  const int4 d = p.desc[c];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.y;
  if (d.w < 2 || r >= d.y * p.group) return;
  const int tok = r / p.group, g = r - tok * p.group;
  const int pieces = d.w;
  float mx = -INFINITY;
  for (int k = lane; k < pieces; k += 32) mx = fmaxf(mx, slot_ml(p, c + k, k == 0)[r]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float off = mx == -INFINITY ? 0.f : mx;
  float total = 0.f, acc[V];
#pragma unroll
  for (int x = 0; x < V; ++x) acc[x] = 0.f;
  for (int k0 = warp; k0 < pieces; k0 += KW * kUnroll) {
    float f[kUnroll], l[kUnroll], v[kUnroll][V];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = k0 + u * KW;
      if (k >= pieces) continue;
      const float *ml = slot_ml(p, c + k, k == 0);
      f[u] = ml[r];
      l[u] = ml[p.rows + r];
      const float *o = slot_o(p, c + k, k == 0) + static_cast<long>(r) * D + lane * V;
      if constexpr (V == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(o);
        v[u][0] = t.x, v[u][1] = t.y, v[u][2] = t.z, v[u][3] = t.w;
      } else {
        const float2 t = *reinterpret_cast<const float2 *>(o);
        v[u][0] = t.x, v[u][1] = t.y;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (k0 + u * KW >= pieces) continue;
      const float w = exp2_mufu(f[u] - off);
      total += w * l[u];
#pragma unroll
      for (int x = 0; x < V; ++x) acc[x] += w * v[u][x];
    }
  }
#pragma unroll
  for (int x = 0; x < V; ++x) part[warp][lane][x] = acc[x];
  part[warp][lane][V] = total;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int k = 1; k < KW; ++k) {
#pragma unroll
    for (int x = 0; x < V; ++x) acc[x] += part[k][lane][x];
    total += part[k][lane][V];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  uint16_t *out = p.out + (d.x + tok) * p.ldo + static_cast<long>(d.z * p.group + g) * D + lane * V;
  if constexpr (V == 4)
    *reinterpret_cast<uint2 *>(out) = make_uint2(pack2<F16>(acc[0] * inv, acc[1] * inv),
                                                 pack2<F16>(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t *>(out) = pack2<F16>(acc[0] * inv, acc[1] * inv);
}

// ------------------------------------------------------------------ host side
static void launch_combine(const Params &p, int ctas, bool f16, cudaStream_t stream) {
  auto *kern = p.D == 128 ? (f16 ? combine_kernel<128, true> : combine_kernel<128, false>)
                          : (f16 ? combine_kernel<64, true> : combine_kernel<64, false>);
  launch_pdl(kern, dim3(ctas, std::min(p.tpt, p.max_q) * p.group), 128, 0, stream, true, p);
}

KvMaps make_kv_maps(const krb_kv_cache &c, int layer, int keys) {
  KvMaps r;
  r.box = std::min(c.page_size, keys);
  const uint64_t dims[4] = {uint64_t(c.head_dim), uint64_t(c.page_size), uint64_t(c.heads),
                            uint64_t(c.pages)};
  auto make = [&](const void *mem, const int64_t *st) {
    // an axis of length 1 is never stepped along: any legal stride will do
    const uint64_t s[3] = {uint64_t(st[3]), c.heads > 1 ? uint64_t(st[2]) : 8,
                           c.pages > 1 ? uint64_t(st[1]) : 8};
    return make_tmap_4d_2byte(static_cast<const uint16_t *>(mem) + (c.layers > 1 ? layer * st[0] : 0),
                              dims, s, r.box);
  };
  r.k = make(c.k, c.k_stride);
  r.v = make(c.v, c.v_stride);
  return r;
}

static size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

size_t workspace_bytes(int ctas, int rows, int D) {
  return align256(ctas * sizeof(int4)) + align256(size_t(ctas) * 4 * rows * sizeof(float)) +
         size_t(ctas) * 2 * rows * D * sizeof(float);
}

void carve_workspace(Params &p, int ctas, void *ws) {
  uint8_t *b = static_cast<uint8_t *>(ws);
  p.desc = reinterpret_cast<int4 *>(b);
  b += align256(ctas * sizeof(int4));
  p.ml = reinterpret_cast<float *>(b);
  b += align256(size_t(ctas) * 4 * p.rows * sizeof(float));
  p.o = reinterpret_cast<float *>(b);
}

template <int D, int WM, bool F16>
static void launch(const Params &p, const KvMaps &maps, int ctas, int device, cudaStream_t stream) {
  auto *kern = attn_paged_kernel<D, WM, F16>;
  static bool configured[64] = {false};
  if (!configured[device & 63]) {
    KRB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
    configured[device & 63] = true;
  }
  int box_shift = 0;
  while ((1 << box_shift) < maps.box) ++box_shift;
  launch_pdl(kern, dim3(ctas), kThreads, Cfg<D>::kSmem, stream, false, maps.k, maps.v, p, box_shift);
}

template <int D, bool F16>
static void launch_wm(int wm, const Params &p, const KvMaps &maps, int ctas, int device,
                      cudaStream_t stream) {
  if constexpr (D == 64)
    if (wm == 2) return launch<D, 2, F16>(p, maps, ctas, device, stream);
  launch<D, 1, F16>(p, maps, ctas, device, stream);
}

CUtensorMap make_tmap_rows(const void *q, int N, int HQ, int D, long ldq, int tok, int heads) {
  const uint64_t dims[4] = {uint64_t(D), uint64_t(HQ), uint64_t(N), 1};
  const uint64_t strides[3] = {uint64_t(D), uint64_t(ldq), 8};
  return make_tmap_4d_2byte(q, dims, strides, heads, tok);
}

// The kernel of a call, from the most rows that a unit can have: mma.sync on 16 wm rows, or
// tcgen05 on nt tiles of 128.  From 17 rows on tcgen05 wins although it pads them: 32 query heads
// over 8 KV heads of 128, 16 sequences of 1 to 4 thousand positions, mma.sync against tcgen05: 16
// rows 38.8 us : 39.3, 32 rows 44.6 : 39.8, 48 rows 54.5 : 41.0, 64 rows 56.4 : 42.5 (mma.sync's
// warps are bound by the latency of ldmatrix and mma chains, two per scheduler).  At head_dim 64 a
// block has half the work: 28 rows 14.6 : 17.1, 56 rows 17.6 : 17.2.
struct Plan {
  int wm, nt, rows, ctas, tile_tok, tpt;
};
static Plan plan_of(int group, int max_q, int D, int device) {
  const long rows = long(max_q) * group;
  Plan r{};
  if (rows <= (D == 64 ? 32 : 16)) {
    r.wm = rows <= 16 ? 1 : 2;
    r.rows = 16 * r.wm;
    r.ctas = 2 * sm_count(device);
    r.tpt = r.tile_tok = r.rows / group;
  } else {
    r.tile_tok = 128 / group;
    r.nt = max_q > r.tile_tok ? 2 : 1;
    r.rows = 128 * r.nt;
    r.ctas = sm_count(device);
    r.tpt = r.nt * r.tile_tok;
  }
  return r;
}

static int group_of(const krb_kv_cache &c, int HQ, int max_q) {
  if (HQ <= 0 || HQ % c.heads) throw CudaError("attention_paged: HQ must be a multiple of the cache's heads");
  if (HQ / c.heads > 64) throw CudaError("attention_paged: more than 64 query heads per KV head");
  if (max_q < 0 || max_q > (1 << 24)) throw CudaError("attention_paged: bad max_q");
  return HQ / c.heads;
}

}  // namespace paged

size_t attention_paged_workspace(const krb_kv_cache &c, int HQ, int max_q) {
  const int group = paged::group_of(c, HQ, max_q);
  int device = 0;
  KRB_CUDA(cudaGetDevice(&device));
  const paged::Plan pl = paged::plan_of(group, std::max(max_q, 1), c.head_dim, device);
  return paged::workspace_bytes(pl.ctas, pl.rows, c.head_dim);
}

void attention_paged(const krb_kv_cache &c, int layer, const PagedAttnArgs &a, cudaStream_t stream) {
  using namespace paged;
  if (a.N < 0 || a.B < 0) throw CudaError("attention_paged: negative size");
  const int group = group_of(c, a.HQ, a.max_q);
  if (a.N == 0 || a.B == 0) return;
  if (a.max_q == 0) throw CudaError("attention_paged: bad max_q (0 with rows and sequences)");
  if (!a.q || !a.out || !a.page_table || !a.kv_lens || !a.q_starts)
    throw CudaError("attention_paged: null pointer");
  const long width = static_cast<long>(a.HQ) * c.head_dim;
  if (a.ldq < width || a.ldo < width || a.ldq % 8 || a.ldo % 8)
    throw CudaError("attention_paged: row pitch too small or not a multiple of 8");
  check_aligned({a.q, a.out, a.workspace}, 16, "attention_paged: pointers must be 16-byte aligned");
  check_aligned({a.page_table, a.kv_lens, a.q_starts, a.mask, a.status}, 4,
                "attention_paged: table, lengths, starts, mask and status must be 4-byte aligned");
  if (a.max_pages <= 0 || a.ldp < a.max_pages)
    throw CudaError("attention_paged: page table narrower than its rows");
  if (int64_t(a.max_pages) * c.page_size > (int64_t(1) << 30))
    throw CudaError("attention_paged: max_pages * page_size above 2^30");
  if (!(a.scale > 0.f) || a.scale > 1e30f) throw CudaError("attention_paged: scale must be positive");
  if (a.mask && (a.mask_words <= 0 || a.ldm < a.mask_words || long(a.mask_words) * 32 < a.max_q))
    throw CudaError("attention_paged: mask rows narrower than max_q");
  if (rows_overlap(a.q, a.ldq, width, a.out, a.ldo, width, a.N))
    throw CudaError("attention_paged: out overlaps q");
  int device = 0;
  KRB_CUDA(cudaGetDevice(&device));
  const Plan pl = plan_of(group, a.max_q, c.head_dim, device);
  if (!a.workspace || a.workspace_bytes < workspace_bytes(pl.ctas, pl.rows, c.head_dim))
    throw CudaError("attention_paged: workspace too small");

  Params p{};
  p.q = static_cast<const uint16_t *>(a.q);
  p.out = static_cast<uint16_t *>(a.out);
  p.ldq = a.ldq;
  p.ldo = a.ldo;
  p.page_table = a.page_table;
  p.kv_lens = a.kv_lens;
  p.q_starts = a.q_starts;
  p.mask = a.mask;
  p.ldp = a.ldp;
  p.ldm = a.ldm;
  p.N = a.N;
  p.HQ = a.HQ;
  p.HKV = c.heads;
  p.group = group;
  p.D = c.head_dim;
  p.B = a.B;
  p.max_q = a.max_q;
  p.max_pages = a.max_pages;
  p.pages = c.pages;
  while ((1 << p.page_shift) < c.page_size) ++p.page_shift;
  p.mask_words = a.mask_words;
  p.rows = pl.rows;
  p.tpt = pl.tpt;
  p.tile_tok = pl.tile_tok;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = a.status;
  carve_workspace(p, pl.ctas, a.workspace);

  const bool f16 = c.dtype == 1;
  if (pl.nt) {
    launch_tc(c, layer, p, pl.ctas, device, stream);
  } else {
    const KvMaps maps = make_kv_maps(c, layer, kKeys);
    if (p.D == 128 && f16) launch_wm<128, true>(pl.wm, p, maps, pl.ctas, device, stream);
    else if (p.D == 128) launch_wm<128, false>(pl.wm, p, maps, pl.ctas, device, stream);
    else if (f16) launch_wm<64, true>(pl.wm, p, maps, pl.ctas, device, stream);
    else launch_wm<64, false>(pl.wm, p, maps, pl.ctas, device, stream);
    launch_combine(p, pl.ctas, f16, stream);
  }
}

}  // namespace krb
