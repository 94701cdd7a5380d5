// Attention of one new token per sequence over a paged key-value cache: out = softmax(scale * q K^T) V.
// One block per (sequence, query head); each warp walks every fourth token with the running maximum and sum of the
// softmax, and the warps' parts are joined at the end.
#include "paged_kv.cuh"

namespace wush {
namespace kv {

struct AttentionParams {
  wush_kv_pages kv;
  wush_kv_table table;
  wush_heads q, out;
  float* lse;
  const int32_t* seq_lens;
  const int32_t* pages;
  const int32_t* counts;
  int* status;
  float scale;
  int64_t window;
  int q_heads, top;
};

constexpr int WARPS = 4;

template <typename T, typename C>
__global__ void __launch_bounds__(WARPS * 32) attention_kernel(const AttentionParams p) {
  __shared__ float sm_m[WARPS], sm_l[WARPS];
  __shared__ float sm_o[WARPS][MAX_DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x % p.q_heads, group = p.q_heads / p.kv.heads, hk = h / group, d = p.kv.dim;
  const int64_t b = blockIdx.x / p.q_heads;
  const int len = clamp_length(p.seq_lens[b], p.table.width * p.kv.page_size, p.status);
  const int begin = p.window > 0 && len > p.window ? (int)(len - p.window) : 0;
  const int64_t entry = b * p.kv.heads + hk;
  const int64_t n = p.pages ? (int64_t)max(0, min(p.counts[entry], p.top)) * p.kv.page_size : len - begin;
  float q[8];
  const bool mine = lane * 8 < d;
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = 0.0f;
  if (mine) load8(reinterpret_cast<const T*>(p.q.data) + b * p.q.row + (int64_t)h * p.q.head + lane * 8, q);
  const float factor = p.scale * (sizeof(C) == 1 ? p.kv.k_scale[hk] : 1.0f);
  float m = -INFINITY, l = 0.0f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int64_t t = warp; t < n; t += WARPS) {
    int lp = (int)((p.pages ? t : begin + t) / p.kv.page_size);
    const int row = (int)((p.pages ? t : begin + t) - (int64_t)lp * p.kv.page_size);
    if (p.pages) {
      lp = p.pages[entry * p.top + lp];
      if (lp < 0 || lp >= p.table.width) {
        report_index(p.status);
        continue;
      }
      if ((int64_t)lp * p.kv.page_size + row >= len) continue;
    }
    const int page = lookup_page(p.table, b, lp, p.kv.num_pages, p.status);
    if (page < 0) continue;
    float k[8], v[8], s = 0.0f;
    if (mine) {
      load8(reinterpret_cast<const C*>(p.kv.k) + page * p.kv.k_page + row * p.kv.k_row + hk * p.kv.k_head + lane * 8, k);
      load8(reinterpret_cast<const C*>(p.kv.v) + page * p.kv.v_page + row * p.kv.v_row + hk * p.kv.v_head + lane * 8, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(q[j], k[j], s);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= factor;
    const float top = fmaxf(m, s);
    const float base = top == -INFINITY ? 0.0f : top;
    const float keep = expf(m - base), e = expf(s - base);
    m = top;
    l = l * keep + e;
    if (mine) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = o[j] * keep + e * v[j];
    }
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
  if (mine) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sm_o[warp][lane * 8 + j] = o[j];
  }
  __syncthreads();
  float top = sm_m[0], total = 0.0f, part[WARPS];
  for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm_m[w]);
  const float base = top == -INFINITY ? 0.0f : top;
  for (int w = 0; w < WARPS; ++w) {
    part[w] = expf(sm_m[w] - base);
    total += sm_l[w] * part[w];
  }
  const float scale = (sizeof(C) == 1 ? p.kv.v_scale[hk] : 1.0f) / (total == 0.0f ? 1.0f : total);
  if (warp == 0 && mine) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      r[j] = 0.0f;
      for (int w = 0; w < WARPS; ++w) r[j] += sm_o[w][lane * 8 + j] * part[w];
      r[j] *= scale;
    }
    store8(reinterpret_cast<T*>(p.out.data) + b * p.out.row + (int64_t)h * p.out.head + lane * 8, r);
  }
  if (threadIdx.x == 0 && p.lse) p.lse[b * p.q_heads + h] = total == 0.0f ? -INFINITY : base + logf(total);
}

}  // namespace kv
}  // namespace wush

using namespace wush;
using namespace wush::kv;

extern "C" size_t wush_kv_attention_workspace_bytes(const wush_kv_pages*, int) { return 0; }

extern "C" int wush_kv_attention(const wush_kv_pages* kv, const wush_kv_table* table, int type, const wush_heads* q, int q_heads,
                                 const wush_heads* out, float* lse, const int32_t* seq_lens, float scale, int64_t window,
                                 const int32_t* pages, const int32_t* counts, int top, void* workspace, size_t workspace_bytes,
                                 int* status, void* stream) {
  int rc = check_pages(kv, table, type);
  if (rc != 0) return rc;
  if (q_heads <= 0 || q_heads % kv->heads || window < 0) return WUSH_ERR_BAD_SHAPE;
  if ((pages == nullptr) != (counts == nullptr)) return WUSH_ERR_NULL_POINTER;
  if (pages && (top <= 0 || (int64_t)top * kv->page_size > INT32_MAX)) return WUSH_ERR_BAD_SHAPE;
  if (pages && window != 0) return WUSH_ERR_BAD_FLAG;
  if (table->seqs == 0) return WUSH_OK;
  if ((rc = check_heads(q, 2)) != 0 || (rc = check_heads(out, 2)) != 0) return rc;
  if (!seq_lens) return WUSH_ERR_NULL_POINTER;
  if (workspace_bytes < wush_kv_attention_workspace_bytes(kv, q_heads)) return WUSH_ERR_WORKSPACE_TOO_SMALL;
  if (table->seqs * q_heads > INT32_MAX) return WUSH_ERR_TOO_LARGE;
  if ((rc = require_sm100()) != 0) return rc;
  const AttentionParams p{*kv, *table, *q, *out, lse, seq_lens, pages, counts, status, scale, window, q_heads, top};
  auto go = [&](auto kern) {
    kern<<<(unsigned)(table->seqs * q_heads), WARPS * 32, 0, (cudaStream_t)stream>>>(p);
    return (int)cudaGetLastError();
  };
  if (type == WUSH_TYPE_BF16)
    return kv->type == WUSH_TYPE_E4M3 ? go(attention_kernel<__nv_bfloat16, __nv_fp8_e4m3>)
                                      : go(attention_kernel<__nv_bfloat16, __nv_bfloat16>);
  return kv->type == WUSH_TYPE_E4M3 ? go(attention_kernel<__half, __nv_fp8_e4m3>) : go(attention_kernel<__half, __half>);
}
