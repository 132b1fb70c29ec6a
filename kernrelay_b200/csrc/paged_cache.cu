// Operators that write the paged K/V cache: append (with the per-head norms and the rotation),
// page copies and the commit of a draft's accepted tokens.  All three move bytes: every kernel
// here is bound by HBM bandwidth at size and by its launch when small.
#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

#include "paged.h"
#include "ptx.cuh"

namespace krb {

// ------------------------------------------------------------------ arguments
[[noreturn]] static void refuse(const char *what, const char *why) {
  throw CudaError(std::string(what) + ": " + why);
}

static void check_strides(const int64_t *st, const krb_kv_cache &c, const char *what) {
  const int64_t n[4] = {c.layers, c.pages, c.heads, c.page_size};
  int order[4] = {0, 1, 2, 3};
  std::sort(order, order + 4, [&](int a, int b) { return st[a] < st[b]; });
  int64_t span = c.head_dim;  // extent of the axes with smaller strides, in elements
  for (int i : order) {
    if (n[i] == 1) continue;  // never stepped along
    if (st[i] % 8) refuse(what, "cache strides must be multiples of 8 elements");
    if (st[i] < span) refuse(what, "cache strides overlap");
    if (st[i] > (int64_t(1) << 38)) refuse(what, "cache stride too large");
    span = st[i] * (n[i] - 1) + span;
  }
}

void check_cache(const krb_kv_cache *c, int layer, const char *what) {
  if (!c) refuse(what, "no cache");
  if (!c->k || !c->v) refuse(what, "cache without K or V");
  if (c->k == c->v) refuse(what, "K and V are the same array");
  if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16)
    refuse(what, "K and V must be 16-byte aligned");
  if (c->dtype != 0 && c->dtype != 1) refuse(what, "cache dtype must be bf16 or fp16");
  if (c->layers <= 0 || c->pages <= 0 || c->heads <= 0)
    refuse(what, "cache without layers, pages or heads");
  if (c->head_dim != 64 && c->head_dim != 128) refuse(what, "head_dim must be 64 or 128");
  if (c->page_size < 8 || c->page_size > (1 << 20) || (c->page_size & (c->page_size - 1)))
    refuse(what, "page_size must be a power of two from 8 on");
  if (layer < 0 || layer >= c->layers) refuse(what, "no such layer");
  check_strides(c->k_stride, *c, what);
  check_strides(c->v_stride, *c, what);
}

void check_aligned(std::initializer_list<const void *> ps, size_t bytes, const char *why) {
  for (const void *p : ps)
    if (reinterpret_cast<uintptr_t>(p) % bytes) throw CudaError(why);
}

bool rows_overlap(const void *a, long la, long wa, const void *b, long lb, long wb, int n) {
  using i128 = __int128;  // pitches are the caller's
  const i128 a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  const i128 pa = i128(la) * 2, pb = i128(lb) * 2, ra = i128(wa) * 2, rb = i128(wb) * 2;
  const i128 last = n - 1;
  if (a0 + last * pa + ra <= b0 || b0 + last * pb + rb <= a0) return false;
  if (n > 1 && pa == pb) {  // columns of one buffer, maybe
    const i128 d = ((b0 - a0) % pa + pa) % pa;
    return d < ra || d + rb > pa;
  }
  for (i128 i = 0, j = 0; i < n && j < n;) {
    const i128 ea = a0 + i * pa + ra, eb = b0 + j * pb + rb;
    if (ea - ra < eb && eb - rb < ea) return true;
    if (ea <= eb) ++i;
    else ++j;
  }
  return false;
}

namespace {

int ilog2(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

// ------------------------------------------------------------------ append
struct AppendArgs {
  const uint16_t *qkv;
  long ldqkv;
  uint16_t *q_out;
  long ldq;
  uint16_t *k, *v;                               // this layer
  long k_page, k_head, k_slot, v_page, v_head, v_slot;  // strides in elements
  const int64_t *positions, *slots;
  const __nv_bfloat16 *cos_tab, *sin_tab, *q_norm, *k_norm;
  int N, HQ, HKV, max_pos, page_shift;
  int64_t total_slots;
  float eps;
  uint32_t *status;
};

// eight 2-byte values as four pairs of fp32, and back
template <bool F16>
__device__ __forceinline__ void unpack8(const uint4 &w, uint64_t (&f)[4]) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (F16) {
      const float2 t = unpack2<true>(ws[e]);
      f[e] = pack_f32x2(__float_as_uint(t.x), __float_as_uint(t.y));
    } else {
      f[e] = pack_f32x2(ws[e] << 16, ws[e] & 0xffff0000u);
    }
  }
}

template <bool F16>
__device__ __forceinline__ uint4 pack8(const uint64_t (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 t = unpack_f32x2(f[e]);
    w[e] = pack2<F16>(t.x, t.y);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 ldg4(const void *p) {
  return __ldg(reinterpret_cast<const uint4 *>(p));
}

// One thread = 8 rotation pairs (elements j..j+7 and D/2+j..D/2+j+7) of one head of one token; the
// D/16 threads of a head are neighbours in a warp and share its sum of squares.
//   x^ = x * rsqrt(mean(x^2) + eps) * w;  y_lo = x_lo cos_lo - x_hi sin_lo,
//   y_hi = x_hi cos_hi + x_lo sin_hi
// in fp32 from the stored values to the one rounding of the store.
//
// Bound: HBM at size (every value read and written once), a launch when small.  What it takes is
// loads in flight, and that is warps: the halves are rotated one after the other, in paired fp32, so
// that forty warps are resident, and the rows, read once, leave L1 to the tables.  Measured (calls in a
// graph, three sets of inputs in turn): 8192 tokens of 32 + 2 x 8 heads of 128 with norms, 203 MB, 42 us,
// 0.75 of the copy's rate (rows through L1 the same); 2400 of them 11.3 us, 0.83 (13.6).  Before rows went
// past L1: unpaired, with 32 / 40 / 48 warps, 48.8 / 44.2 / 45.6 us, paired 43.
// Tried: several heads per warp with the table products in registers (54 us), whole rows by bulk copies
// into shared memory (42.2 us, and twice the time at 14 + 2 x 2 heads of 64), stores that leave L2 first
// (__stcs: 39.5 us by itself, 11.9 for 2400 tokens, but the attention behind it pays: append and
// attention of 8 prompts, 101 / 201 MB of output, 175.0 / 468 us with plain stores, 176.4 / 472 with
// those; between a QKV and an output GEMM of a layer 727.5 / 1577 and 729 / 1577, 32 prompts 659.7 /
// 1357.6 and 659.5 / 1360).
template <int D, bool F16>
__global__ void __launch_bounds__(128, 10) append_kernel(const AppendArgs a) {
  constexpr int HALF = D / 2;
  constexpr int kLanes = HALF / 8;
  pdl_wait();
  const uint32_t gt = blockIdx.x * 128u + threadIdx.x;
  const uint32_t nh = a.HQ + 2 * a.HKV;
  const uint32_t item = gt / kLanes;
  const int j = static_cast<int>(gt % kLanes) * 8;
  const int n = static_cast<int>(item / nh);
  if (n >= a.N) return;  // whole heads only
  const int h = static_cast<int>(item - n * nh);
  const uint16_t *p = a.qkv + n * a.ldqkv + h * D + j;
  // read once: kept out of the way of the tables (coherent loads: q_out may be the q columns of qkv)
  const uint4 wlo = __ldcs(reinterpret_cast<const uint4 *>(p));
  const uint4 whi = __ldcs(reinterpret_cast<const uint4 *>(p + HALF));
  const int64_t pos = a.positions[n];
  const bool pos_ok = pos >= 0 && pos < a.max_pos;
  if (!pos_ok && h == 0 && j == 0) report_status(a.status, kStatusBadIndex);

  auto store = [&](uint16_t *to, const uint4 &w) { *reinterpret_cast<uint4 *>(to) = w; };
  uint16_t *dst;
  if (h < a.HQ) {
    dst = a.q_out + n * a.ldq + h * D + j;
  } else {
    const int64_t slot = a.slots[n];
    const bool slot_ok = slot >= 0 && slot < a.total_slots;
    if (!slot_ok && slot != -1 && h == a.HQ && j == 0) report_status(a.status, kStatusBadIndex);
    // the D/16 threads of this head leave together (n and h are theirs alike)
    if (!slot_ok || !pos_ok) return;
    const long page = static_cast<long>(slot >> a.page_shift);
    const long off = static_cast<long>(slot & ((int64_t(1) << a.page_shift) - 1));
    if (h < a.HQ + a.HKV) {
      dst = a.k + page * a.k_page + (h - a.HQ) * a.k_head + off * a.k_slot + j;
    } else {
      dst = a.v + page * a.v_page + (h - a.HQ - a.HKV) * a.v_head + off * a.v_slot + j;
      store(dst, wlo);
      store(dst + HALF, whi);
      return;
    }
  }
  if (!pos_ok) {
    *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4 *>(dst + HALF) = make_uint4(0, 0, 0, 0);
    return;
  }
  const long t = pos * D + j;
  const uint4 tc0 = ldg4(a.cos_tab + t), ts0 = ldg4(a.sin_tab + t);
  const uint4 tc1 = ldg4(a.cos_tab + t + HALF), ts1 = ldg4(a.sin_tab + t + HALF);
  uint64_t lo[4], hi[4], f[4];
  unpack8<F16>(wlo, lo);
  unpack8<F16>(whi, hi);
  const __nv_bfloat16 *nw = h < a.HQ ? a.q_norm : a.k_norm;
  if (nw) {
    uint64_t sq = 0;  // two sums
#pragma unroll
    for (int e = 0; e < 4; ++e) sq = fma_f32x2(hi[e], hi[e], fma_f32x2(lo[e], lo[e], sq));
    const float2 s2 = unpack_f32x2(sq);
    float ss = s2.x + s2.y;
    const unsigned lane = threadIdx.x & 31;
    const unsigned mask = ((1u << kLanes) - 1u) << (lane & ~unsigned(kLanes - 1));
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    const uint32_t r = __float_as_uint(rsqrtf(ss * (1.0f / D) + a.eps));
    const uint64_t rr = pack_f32x2(r, r);
    unpack8<false>(ldg4(nw + j), f);
#pragma unroll
    for (int e = 0; e < 4; ++e) lo[e] = mul_f32x2(lo[e], mul_f32x2(rr, f[e]));
    unpack8<false>(ldg4(nw + HALF + j), f);
#pragma unroll
    for (int e = 0; e < 4; ++e) hi[e] = mul_f32x2(hi[e], mul_f32x2(rr, f[e]));
  }
  uint64_t y[4];
  unpack8<false>(tc0, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = mul_f32x2(lo[e], f[e]);
  unpack8<false>(make_uint4(ts0.x ^ 0x80008000u, ts0.y ^ 0x80008000u, ts0.z ^ 0x80008000u,
                            ts0.w ^ 0x80008000u), f);  // -sin
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = fma_f32x2(hi[e], f[e], y[e]);
  store(dst, pack8<F16>(y));
  unpack8<false>(tc1, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = mul_f32x2(hi[e], f[e]);
  unpack8<false>(ts1, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = fma_f32x2(lo[e], f[e], y[e]);
  store(dst + HALF, pack8<F16>(y));
}

template <int D, bool F16>
void launch_append(const AppendArgs &a, cudaStream_t stream) {
  const long threads = static_cast<long>(a.N) * (a.HQ + 2 * a.HKV) * (D / 16);
  if (threads > 0xffffff00L) throw CudaError("qk_norm_rope_paged: too many tokens");
  launch_pdl(append_kernel<D, F16>, dim3(static_cast<unsigned>((threads + 127) / 128)), 128, 0, stream, false, a);
}

// ------------------------------------------------------------------ page copies
// Pages travel to the kernel in its parameters: the host arrays are read before the call
// returns, and a captured launch keeps its own copy.
constexpr int kPairsPerLaunch = 448;

struct CopyArgs {
  uint4 *base[2];           // K, V
  long layer[2], page[2];   // strides in 16-byte units
  long outer[2], inner[2];  // strides of the runs inside a page
  int n_inner[2];           // runs per outer step
  int run[2];               // 16-byte units per contiguous run
  int units;                // 16-byte units of a page (all heads)
  int layers;
  int32_t src[kPairsPerLaunch], dst[kPairsPerLaunch];
};

constexpr int kCopyVec = 4;

// grid (chunks of a page, pairs, layers * 2): 256 threads move kCopyVec units each
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  const int kv = blockIdx.z & 1;
  const int layer = blockIdx.z >> 1;
  const long base = layer * a.layer[kv];
  uint4 *const mem = a.base[kv];
  const uint4 *src = mem + base + a.src[blockIdx.y] * a.page[kv];
  uint4 *dst = mem + base + a.dst[blockIdx.y] * a.page[kv];
  const int run = a.run[kv], ni = a.n_inner[kv];
  uint4 w[kCopyVec];
  long at[kCopyVec];
#pragma unroll
  for (int i = 0; i < kCopyVec; ++i) {
    const int u = (blockIdx.x * kCopyVec + i) * 256 + threadIdx.x;
    const int r = u / run;
    at[i] = u < a.units ? (r / ni) * a.outer[kv] + (r % ni) * a.inner[kv] + (u - r * run) : -1;
    if (at[i] >= 0) w[i] = src[at[i]];
  }
#pragma unroll
  for (int i = 0; i < kCopyVec; ++i)
    if (at[i] >= 0) dst[at[i]] = w[i];
}

// ------------------------------------------------------------------ commit
struct CommitArgs {
  uint16_t *k, *v;
  long k_layer, k_page, k_head, k_slot, v_layer, v_page, v_head, v_slot;
  const int32_t *page_table, *bases, *accepted, *counts;
  long ldp, lda;
  int max_pages, pages, A, page_shift, layers, heads;
  uint32_t *status;
};

// One CTA = one sequence and some of its (layer, K or V, head) rows.  It checks the sequence's
// whole list first (so that a refused one is left whole) and keeps page and slot of the moves in
// shared memory, kCommitList at a time; a thread moves one 16-byte column, kCommitChunk moves at a
// time: it reads their sources, then writes their targets.  accepted ascends strictly from >= 0,
// so target i <= source i < later sources: no source is overwritten before it is read, whatever the
// chunks.
constexpr int kCommitThreads = 256;
constexpr int kCommitChunk = 8;
constexpr int kCommitList = 256;

template <int D>
__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const CommitArgs a) {
  constexpr int kLanes = D / 8;
  __shared__ int4 s_move[kCommitList];  // source page, slot; target page, slot (source page -1: stays)
  pdl_wait();
  const int b = blockIdx.x;
  const int32_t *acc = a.accepted + b * a.lda;
  const int32_t *table = a.page_table + b * a.ldp;
  const int t = threadIdx.x;
  // the list's first entries come with the sizes, not behind them
  const int n = a.counts[b];
  const int64_t base = a.bases[b];
  const int first = t < a.A ? acc[t] : 0, before_first = t > 0 && t < a.A ? acc[t - 1] : -1;
  const int64_t room = static_cast<int64_t>(a.max_pages) << a.page_shift;
  const bool sizes_ok = n >= 0 && n <= a.A && base >= 0 && base <= room;
  const int slot_mask = (1 << a.page_shift) - 1;
  // the move of entry i = x, checked
  auto move = [&](int i, int64_t x, int64_t before, int4 &m) {
    if (x <= before || base + x >= room) return false;
    const int64_t from = base + x, to = base + i;
    m = make_int4(table[from >> a.page_shift], static_cast<int>(from) & slot_mask,
                  table[to >> a.page_shift], static_cast<int>(to) & slot_mask);
    if (m.x < 0 || m.x >= a.pages || m.z < 0 || m.z >= a.pages) return false;
    if (x == i) m.x = -1;
    return true;
  };
  bool bad = !sizes_ok;
  if (sizes_ok) {
    for (int i = t; i < n; i += kCommitThreads) {
      int4 m;
      if (!move(i, i == t ? first : acc[i], i == t ? before_first : acc[i - 1], m)) bad = true;
      else if (i < kCommitList) s_move[i] = m;
    }
  }
  if (__syncthreads_or(bad)) {
    if (t == 0 && blockIdx.y == 0) report_status(a.status, kStatusBadIndex);
    return;
  }
  const int rows = a.layers * 2 * a.heads;
  const int row = blockIdx.y * (kCommitThreads / kLanes) + threadIdx.x / kLanes;
  const int col = (threadIdx.x % kLanes) * 8;
  const int h = row % a.heads;
  const int kv = (row / a.heads) & 1;
  const int layer = row / (2 * a.heads);
  uint16_t *mem = (kv ? a.v + layer * a.v_layer + h * a.v_head : a.k + layer * a.k_layer + h * a.k_head) + col;
  const long ps = kv ? a.v_page : a.k_page, ss = kv ? a.v_slot : a.k_slot;
  for (int l0 = 0; l0 < n; l0 += kCommitList) {
    if (l0 > 0) {  // the next part of a long list
      __syncthreads();
      for (int i = l0 + threadIdx.x; i < min(n, l0 + kCommitList); i += kCommitThreads)
        move(i, acc[i], acc[i - 1], s_move[i - l0]);
      __syncthreads();
    }
    if (row >= rows) continue;
    const int m = min(n - l0, kCommitList);
    for (int i0 = 0; i0 < m; i0 += kCommitChunk) {
      uint4 w[kCommitChunk];
#pragma unroll
      for (int i = 0; i < kCommitChunk; ++i)
        if (i0 + i < m && s_move[i0 + i].x >= 0)
          w[i] = *reinterpret_cast<const uint4 *>(mem + s_move[i0 + i].x * ps + s_move[i0 + i].y * ss);
#pragma unroll
      for (int i = 0; i < kCommitChunk; ++i)
        if (i0 + i < m && s_move[i0 + i].x >= 0)
          *reinterpret_cast<uint4 *>(mem + s_move[i0 + i].z * ps + s_move[i0 + i].w * ss) = w[i];
    }
  }
}

}  // namespace

// ------------------------------------------------------------------ host side
void qk_norm_rope_paged(const krb_kv_cache &c, int layer, const void *qkv, long ldqkv, void *q_out,
                        long ldq, const int64_t *positions, const int64_t *slots, int N, int HQ,
                        const __nv_bfloat16 *cos_tab, const __nv_bfloat16 *sin_tab, int max_pos,
                        const __nv_bfloat16 *q_norm, const __nv_bfloat16 *k_norm, float eps,
                        uint32_t *status, cudaStream_t stream) {
  const int D = c.head_dim;
  const int nh = HQ + 2 * c.heads;
  if (N < 0 || HQ <= 0) throw CudaError("qk_norm_rope_paged: bad N or HQ");
  if (N == 0) return;
  if (!qkv || !q_out || !positions || !slots || !cos_tab || !sin_tab)
    throw CudaError("qk_norm_rope_paged: null pointer");
  if (!q_norm != !k_norm) throw CudaError("qk_norm_rope_paged: q_norm and k_norm, or neither");
  if (max_pos <= 0) throw CudaError("qk_norm_rope_paged: empty rope tables");
  if (ldqkv < static_cast<long>(nh) * D || ldq < static_cast<long>(HQ) * D || ldqkv % 8 || ldq % 8)
    throw CudaError("qk_norm_rope_paged: row pitch too small or not a multiple of 8");
  check_aligned({qkv, q_out, cos_tab, sin_tab, q_norm, k_norm}, 16,
                "qk_norm_rope_paged: pointers must be 16-byte aligned");
  check_aligned({positions, slots}, 8, "qk_norm_rope_paged: positions and slots must be 8-byte aligned");
  check_aligned({status}, 4, "qk_norm_rope_paged: status must be 4-byte aligned");
  if (!(q_out == qkv && (ldq == ldqkv || N == 1)) &&
      rows_overlap(qkv, ldqkv, static_cast<long>(nh) * D, q_out, ldq, static_cast<long>(HQ) * D, N))
    throw CudaError("qk_norm_rope_paged: q_out overlaps qkv, and is not its q columns");
  AppendArgs a{};
  a.qkv = static_cast<const uint16_t *>(qkv);
  a.ldqkv = ldqkv;
  a.q_out = static_cast<uint16_t *>(q_out);
  a.ldq = ldq;
  a.k = static_cast<uint16_t *>(c.k) + layer * c.k_stride[0];
  a.v = static_cast<uint16_t *>(c.v) + layer * c.v_stride[0];
  a.k_page = c.k_stride[1];
  a.k_head = c.k_stride[2];
  a.k_slot = c.k_stride[3];
  a.v_page = c.v_stride[1];
  a.v_head = c.v_stride[2];
  a.v_slot = c.v_stride[3];
  a.positions = positions;
  a.slots = slots;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.N = N;
  a.HQ = HQ;
  a.HKV = c.heads;
  a.max_pos = max_pos;
  a.page_shift = ilog2(c.page_size);
  a.total_slots = int64_t(c.pages) * c.page_size;
  a.eps = eps;
  a.status = status;
  if (D == 128 && c.dtype) launch_append<128, true>(a, stream);
  else if (D == 128) launch_append<128, false>(a, stream);
  else if (c.dtype) launch_append<64, true>(a, stream);
  else launch_append<64, false>(a, stream);
}

void kv_copy_pages(const krb_kv_cache &c, const int32_t *src, const int32_t *dst, int n,
                   cudaStream_t stream) {
  if (n < 0) throw CudaError("kv_copy_pages: negative count");
  if (n == 0) return;
  if (!src || !dst) throw CudaError("kv_copy_pages: null pointer");
  std::vector<int32_t> written;  // in order
  written.reserve(n);
  for (int i = 0; i < n; ++i) {
    for (const int32_t p : {src[i], dst[i]})
      if (p < 0 || p >= c.pages) throw CudaError("kv_copy_pages: no page " + std::to_string(p));
    if (src[i] != dst[i]) written.push_back(dst[i]);
  }
  std::sort(written.begin(), written.end());
  const auto twice = std::adjacent_find(written.begin(), written.end());
  if (twice != written.end())
    throw CudaError("kv_copy_pages: page " + std::to_string(*twice) + " is written twice");
  for (int i = 0; i < n; ++i)
    if (src[i] != dst[i] && std::binary_search(written.begin(), written.end(), src[i]))
      throw CudaError("kv_copy_pages: page " + std::to_string(src[i]) + " is read and written");
  CopyArgs a;
  const int64_t *strides[2] = {c.k_stride, c.v_stride};
  void *mem[2] = {c.k, c.v};
  const long d = c.head_dim / 8;
  a.units = static_cast<int>(d) * c.heads * c.page_size;
  if (static_cast<long>(a.units) != d * c.heads * c.page_size || a.units > (1 << 30))
    throw CudaError("kv_copy_pages: page too large");
  a.layers = c.layers;
  for (int kv = 0; kv < 2; ++kv) {
    a.base[kv] = static_cast<uint4 *>(mem[kv]);
    a.layer[kv] = strides[kv][0] / 8;
    a.page[kv] = strides[kv][1] / 8;
    const long head = strides[kv][2] / 8, slot = strides[kv][3] / 8;
    // runs of contiguous units: the inner axis (the one of smaller stride) joins the run when its
    // steps are dense, then the outer one when that is dense too
    const bool slots_inner = c.heads == 1 || (c.page_size > 1 && slot < head);
    const long in_stride = slots_inner ? slot : head, out_stride = slots_inner ? head : slot;
    const int in_n = slots_inner ? c.page_size : c.heads, out_n = slots_inner ? c.heads : c.page_size;
    a.run[kv] = static_cast<int>(d);
    a.n_inner[kv] = in_n;
    a.inner[kv] = in_stride;
    a.outer[kv] = out_stride;
    if (in_n == 1 || in_stride == d) {
      a.run[kv] = static_cast<int>(d) * in_n;
      a.n_inner[kv] = out_n;
      a.inner[kv] = out_stride;
      a.outer[kv] = 0;
      if (out_n == 1 || out_stride == a.run[kv]) {
        a.run[kv] = a.units;
        a.n_inner[kv] = 1;
        a.inner[kv] = 0;
      }
    }
  }
  if (c.layers > 32767) throw CudaError("kv_copy_pages: too many layers");
  for (int i = 0; i < n;) {
    int m = 0;
    for (; i < n && m < kPairsPerLaunch; ++i) {
      if (src[i] == dst[i]) continue;
      a.src[m] = src[i];
      a.dst[m++] = dst[i];
    }
    if (!m) break;
    const dim3 grid((a.units + 256 * kCopyVec - 1) / (256 * kCopyVec), m, 2 * c.layers);
    launch_pdl(copy_pages_kernel, grid, 256, 0, stream, false, a);
  }
}

void kv_commit(const krb_kv_cache &c, const int32_t *page_table, long ldp, int max_pages,
               const int32_t *bases, const int32_t *accepted, long lda, int A,
               const int32_t *counts, int B, uint32_t *status, cudaStream_t stream) {
  if (B < 0 || A < 0) throw CudaError("kv_commit: negative size");
  if (B == 0 || A == 0) return;
  if (!page_table || !bases || !accepted || !counts) throw CudaError("kv_commit: null pointer");
  if (max_pages <= 0 || ldp < max_pages || lda < A)
    throw CudaError("kv_commit: page table or accepted list narrower than its rows");
  check_aligned({page_table, bases, accepted, counts, status}, 4, "kv_commit: pointers must be 4-byte aligned");
  if ((int64_t(max_pages) << ilog2(c.page_size)) > (int64_t(1) << 30))
    throw CudaError("kv_commit: max_pages * page_size above 2^30");
  CommitArgs a{};
  a.k = static_cast<uint16_t *>(c.k);
  a.v = static_cast<uint16_t *>(c.v);
  a.k_layer = c.k_stride[0];
  a.k_page = c.k_stride[1];
  a.k_head = c.k_stride[2];
  a.k_slot = c.k_stride[3];
  a.v_layer = c.v_stride[0];
  a.v_page = c.v_stride[1];
  a.v_head = c.v_stride[2];
  a.v_slot = c.v_stride[3];
  a.page_table = page_table;
  a.bases = bases;
  a.accepted = accepted;
  a.counts = counts;
  a.ldp = ldp;
  a.lda = lda;
  a.max_pages = max_pages;
  a.pages = c.pages;
  a.A = A;
  a.page_shift = ilog2(c.page_size);
  a.layers = c.layers;
  a.heads = c.heads;
  a.status = status;
  const long rows = 2L * c.layers * c.heads;
  const int per = kCommitThreads / (c.head_dim / 8);
  const long gy = (rows + per - 1) / per;
  if (gy > 65535) throw CudaError("kv_commit: too many layers and heads");
  const dim3 grid(B, static_cast<unsigned>(gy));
  launch_pdl(c.head_dim == 128 ? commit_kernel<128> : commit_kernel<64>, grid, kCommitThreads, 0, stream,
             false, a);
}

}  // namespace krb
