// The paged K/V cache as the kernels see it, and the launchers of its operators.
#pragma once

#include <initializer_list>
#include <utility>

#include "common.h"
#include "kernrelay_b200.h"

namespace krb {

// Launch by programmatic dependent launch: `kern` waits for the work before it itself (pdl_wait, first
// thing).  The gap between launches on a stream falls from 2.3 to about 1 us.  `always`: in a
// capture, too (behind a kernel of the same call); else a captured launch takes plain dependencies,
// whatever the stream waits for.
template <typename... P, typename... A>
void launch_pdl(void (*kern)(P...), dim3 grid, int threads, int smem, cudaStream_t stream, bool always,
                A &&...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (!always) KRB_CUDA(cudaStreamIsCapturing(stream, &status));
  cfg.numAttrs = status == cudaStreamCaptureStatusNone ? 1 : 0;
  KRB_CUDA(cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...));
}

// Throws on a cache the operators do not take (null pointers, sizes, alignment, strides whose
// rows overlap); `layer` in [0, layers).
void check_cache(const krb_kv_cache *c, int layer, const char *what);

// Throws unless every address is a multiple of `bytes` (null is one).
void check_aligned(std::initializer_list<const void *> ps, size_t bytes, const char *why);

// Whether any of n rows of `wa` 2-byte elements at pitch `la` shares an element with any of n rows
// of `wb` at pitch `lb` (pitches no smaller than their rows).
bool rows_overlap(const void *a, long la, long wa, const void *b, long lb, long wb, int n);

struct PagedAttnArgs {
  const void *q;
  long ldq;
  void *out;
  long ldo;
  int N, HQ;
  const int32_t *page_table;
  long ldp;
  int max_pages;
  const int32_t *kv_lens, *q_starts;
  int B, max_q;
  const uint32_t *mask;
  long ldm;
  int mask_words;
  float scale;
  void *workspace;
  size_t workspace_bytes;
  uint32_t *status;
};

void qk_norm_rope_paged(const krb_kv_cache &c, int layer, const void *qkv, long ldqkv, void *q_out,
                        long ldq, const int64_t *positions, const int64_t *slots, int N, int HQ,
                        const __nv_bfloat16 *cos_tab, const __nv_bfloat16 *sin_tab, int max_pos,
                        const __nv_bfloat16 *q_norm, const __nv_bfloat16 *k_norm, float eps,
                        uint32_t *status, cudaStream_t stream);
size_t attention_paged_workspace(const krb_kv_cache &c, int HQ, int max_q);
void attention_paged(const krb_kv_cache &c, int layer, const PagedAttnArgs &a, cudaStream_t stream);
void kv_copy_pages(const krb_kv_cache &c, const int32_t *src, const int32_t *dst, int n,
                   cudaStream_t stream);
void kv_commit(const krb_kv_cache &c, const int32_t *page_table, long ldp, int max_pages,
               const int32_t *bases, const int32_t *accepted, long lda, int A,
               const int32_t *counts, int B, uint32_t *status, cudaStream_t stream);

}  // namespace krb
