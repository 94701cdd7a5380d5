// Paged key-value cache: append with rotation, per-page bounds of the keys, selection of pages.
#include "paged_kv.cuh"

namespace wush {
namespace kv {

// ---- append --------------------------------------------------------------------------------------------------------
using AppendParams = wush_kv_append_args;

// One thread per unit of 16 channels of a head (two chunks of 8 that are rotated against each other, or two chunks that
// are only copied).
template <typename T, typename C>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  const int d = p.kv.dim, turned = p.rotary >> 4;
  const int per_head = turned + ((d - p.rotary + 15) >> 4), per_value = (d + 15) >> 4;
  const int rotated_heads = p.q_heads + p.kv.heads;
  const int64_t per_row = (int64_t)rotated_heads * per_head + (int64_t)p.kv.heads * per_value;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < p.rows * per_row; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per_row;
    int u = (int)(i - row * per_row);
    const int seq = p.seq_ids[row], pos = p.positions[row];
    if (seq < 0 || pos < 0) continue;
    if (seq >= p.table.seqs || pos >= p.table.width * p.kv.page_size || (p.rope && pos >= p.rope_rows)) {
      report_index(p.status);
      continue;
    }
    const int lp = pos / p.kv.page_size;
    const int page = lookup_page(p.table, seq, lp, p.kv.num_pages, p.status);
    if (page < 0) continue;
    const int at = pos - lp * p.kv.page_size;
    const bool value = u >= rotated_heads * per_head;
    if (value) u -= rotated_heads * per_head;
    int head = u / (value ? per_value : per_head);
    u -= head * (value ? per_value : per_head);
    const bool query = !value && head < p.q_heads;
    if (!value && !query) head -= p.q_heads;
    int ca, cb;                                             // first channels of the two chunks
    const bool turn = !value && u < turned;
    if (turn) {
      ca = p.interleaved ? u * 16 : u * 8;
      cb = p.interleaved ? ca + 8 : ca + p.rotary / 2;
    } else {
      ca = value ? u * 16 : p.rotary + (u - turned) * 16;
      cb = ca + 8;
    }
    const wush_heads& src = value ? p.v : (query ? p.q : p.k);
    const T* in = reinterpret_cast<const T*>(src.data) + row * src.row + head * src.head;
    const bool two = cb < d;
    float a[8], b[8];
    load8(in + ca, a);
    if (two) load8(in + cb, b);
    if (turn) {
      const float* c = p.rope + (int64_t)pos * p.rotary + u * 8;
      const float* s = c + p.rotary / 2;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float cj = c[j], sj = s[j];
        float& x = p.interleaved ? (j < 4 ? a[2 * j] : b[2 * j - 8]) : a[j];
        float& y = p.interleaved ? (j < 4 ? a[2 * j + 1] : b[2 * j - 7]) : b[j];
        const float nx = __fsub_rn(__fmul_rn(x, cj), __fmul_rn(y, sj));
        const float ny = __fadd_rn(__fmul_rn(y, cj), __fmul_rn(x, sj));
        x = nx;
        y = ny;
      }
    }
    if (query) {
      T* o = reinterpret_cast<T*>(p.q_out.data) + row * p.q_out.row + head * p.q_out.head;
      store8(o + ca, a);
      if (two) store8(o + cb, b);
      continue;
    }
    if (!value && p.k_out.data) {
      T* o = reinterpret_cast<T*>(p.k_out.data) + row * p.k_out.row + head * p.k_out.head;
      store8(o + ca, a);
      if (two) store8(o + cb, b);
    }
    C* o = value ? reinterpret_cast<C*>(p.kv.v) + page * p.kv.v_page + at * p.kv.v_row + head * p.kv.v_head
                 : reinterpret_cast<C*>(p.kv.k) + page * p.kv.k_page + at * p.kv.k_row + head * p.kv.k_head;
    if (sizeof(C) == 1) {
      const float scale = value ? p.kv.v_scale[head] : p.kv.k_scale[head];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] = __fdiv_rn(a[j], scale);
        b[j] = __fdiv_rn(b[j], scale);
      }
    }
    store8(o + ca, a);
    if (two) store8(o + cb, b);
  }
}

// ---- bounds --------------------------------------------------------------------------------------------------------
// minimum / maximum that keep a NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One warp per (sequence, page, head), lanes over the chunks of 8 channels.
template <typename C, typename B>
__global__ void __launch_bounds__(256) bounds_kernel(const wush_kv_pages kv, const wush_kv_table table, const int32_t* seq_lens,
                                                     int64_t new_tokens, int64_t most, int* status) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5), total = table.seqs * most * kv.heads;
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total; w += warps) {
    const int head = (int)(w % kv.heads);
    const int64_t seq = w / kv.heads / most;
    const int len = clamp_length(seq_lens[seq], table.width * kv.page_size, status);
    const int64_t first = len > new_tokens ? len - new_tokens : 0;
    const int64_t lp = first / kv.page_size + w / kv.heads % most;
    if (lp * kv.page_size >= len) continue;
    const int page = lookup_page(table, seq, (int)lp, kv.num_pages, status);
    if (page < 0) continue;
    const int rows = (int)min((int64_t)kv.page_size, len - lp * kv.page_size);
    if (lane * 8 >= kv.dim) continue;
    const C* k = reinterpret_cast<const C*>(kv.k) + page * kv.k_page + head * kv.k_head + lane * 8;
    float lo[8], hi[8], x[8];
    load8(k, lo);
    load8(k, hi);
    for (int r = 1; r < rows; ++r) {
      load8(k + r * kv.k_row, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = min_nan(lo[j], x[j]);
        hi[j] = max_nan(hi[j], x[j]);
      }
    }
    B* out = reinterpret_cast<B*>(kv.bounds) + ((int64_t)page * kv.heads + head) * 2 * kv.dim + lane * 8;
    store8(out, lo);
    store8(out + kv.dim, hi);
  }
}

// ---- selection -----------------------------------------------------------------------------------------------------
// A score as a 64-bit key with the same order; NaN counts as +infinity.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) s = __longlong_as_double(0x7ff0000000000000ll);
  const long long b = __double_as_longlong(s + 0.0);       // -0 + 0 = +0: equal numbers, equal keys
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

// One warp per (sequence, head, page): keys of the scores.
template <typename T, typename B>
__global__ void __launch_bounds__(256) score_kernel(const wush_kv_pages kv, const wush_kv_table table, const wush_heads q,
                                                    int group, const int32_t* seq_lens, int top, unsigned long long* keys,
                                                    int* status) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5), total = table.seqs * kv.heads * table.width;
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total; w += warps) {
    const int lp = (int)(w % table.width), head = (int)(w / table.width % kv.heads);
    const int64_t seq = w / table.width / kv.heads;
    const int len = clamp_length(seq_lens[seq], table.width * kv.page_size, status);
    const int n = (len + kv.page_size - 1) / kv.page_size;
    if (lp >= n || n <= top) continue;
    const int page = lookup_page(table, seq, lp, kv.num_pages, status);
    unsigned long long best = 0;
    if (page >= 0) {
      const B* bound = reinterpret_cast<const B*>(kv.bounds) + ((int64_t)page * kv.heads + head) * 2 * kv.dim;
      for (int g = 0; g < group; ++g) {
        const T* row = reinterpret_cast<const T*>(q.data) + seq * q.row + (int64_t)(head * group + g) * q.head;
        double s = 0.0;
        for (int c = lane * 8; c < kv.dim; c += 256) {
          float x[8], lo[8], hi[8];
          load8(row + c, x);
          load8(bound + c, lo);
          load8(bound + kv.dim + c, hi);
#pragma unroll
          for (int j = 0; j < 8; ++j) s += (double)max_nan(x[j] * lo[j], x[j] * hi[j]);   // 16-bit factors: exact products
        }
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const unsigned long long key = score_key(s);
        best = best < key ? key : best;
      }
    }
    if (lane == 0) keys[w] = best;
  }
}

// One block per (sequence, head).  The threshold key is built bit by bit from the top (the largest key that at least
// `want` pages reach), then the pages above it and the first ones equal to it are written in order.
__global__ void __launch_bounds__(1024) select_kernel(int page_size, int64_t width, int heads, const int32_t* seq_lens,
                                                      const unsigned long long* keys, int top, int sink, int recent,
                                                      int32_t* pages, int32_t* counts) {
  __shared__ int warp_sum[32];
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t item = blockIdx.x;
  const int len = (int)max((int64_t)0, min((int64_t)seq_lens[item / heads], width * page_size));
  const int n = (len + page_size - 1) / page_size;
  const unsigned long long* key = keys + item * width;
  int32_t* out = pages + item * top;
  const int count = min(n, top);
  if (tid == 0) counts[item] = count;
  for (int i = count + tid; i < top; i += blockDim.x) out[i] = -1;
  if (n <= top) {
    for (int i = tid; i < n; i += blockDim.x) out[i] = i;
    return;
  }
  const int begin = sink, end = n - recent, want = top - sink - recent;
  unsigned long long threshold = 0;
  for (int bit = 63; bit >= 0; --bit) {
    const unsigned long long trial = threshold | 1ull << bit;
    int mine = 0;
    for (int i = begin + tid; i < end; i += blockDim.x) mine += key[i] >= trial;
    // every thread gets the sum
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) warp_sum[tid >> 5] = mine;
    __syncthreads();
    const int sum = __reduce_add_sync(0xffffffffu, warp_sum[lane]);
    __syncthreads();
    if (sum >= want) threshold = trial;
  }
  // pages in ascending order: those above the threshold, and the first of those equal to it that are still wanted
  int above = 0;
  for (int i = begin + tid; i < end; i += blockDim.x) above += key[i] > threshold;
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) warp_sum[tid >> 5] = above;
  __syncthreads();
  const int ties = want - __reduce_add_sync(0xffffffffu, warp_sum[lane]);
  __syncthreads();
  __shared__ int taken_sum[32], equal_sum[32];
  int taken = 0, equals = 0;                               // running totals over the pages before this round
  for (int base = 0; base < n; base += blockDim.x) {
    const int i = base + tid;
    const bool forced = i < n && (i < begin || i >= end);
    const unsigned long long x = i >= begin && i < end && want > 0 ? key[i] : 0;
    const bool middle = i >= begin && i < end && want > 0;
    const bool over = middle && x > threshold, equal = middle && x == threshold;
    const unsigned em = __ballot_sync(0xffffffffu, equal);
    if (lane == 0) equal_sum[tid >> 5] = __popc(em);
    __syncthreads();
    int before = equals, all_equal = 0;
    for (int j = 0; j < 32; ++j) {
      before += j < (tid >> 5) ? equal_sum[j] : 0;
      all_equal += equal_sum[j];
    }
    const bool take = forced || over || (equal && before + __popc(em & ((1u << lane) - 1)) < ties);
    const unsigned tm = __ballot_sync(0xffffffffu, take);
    if (lane == 0) taken_sum[tid >> 5] = __popc(tm);
    __syncthreads();
    int slot = taken, all_taken = 0;
    for (int j = 0; j < 32; ++j) {
      slot += j < (tid >> 5) ? taken_sum[j] : 0;
      all_taken += taken_sum[j];
    }
    if (take) out[slot + __popc(tm & ((1u << lane) - 1))] = i;
    taken += all_taken;
    equals += all_equal;
    __syncthreads();
  }
}

}  // namespace kv
}  // namespace wush

using namespace wush;
using namespace wush::kv;

extern "C" int wush_kv_append(const wush_kv_append_args* args) {
  if (!args) return WUSH_ERR_NULL_POINTER;
  AppendParams p = *args;
  int rc = check_pages(&p.kv, &p.table, p.type);
  if (rc == 0) rc = check_heads(&p.k, 2);
  if (rc == 0) rc = check_heads(&p.v, 2);
  if (rc == 0 && p.q.data) rc = check_heads(&p.q, 2);
  if (rc == 0 && p.q.data) rc = check_heads(&p.q_out, 2);
  if (rc == 0 && p.k_out.data) rc = check_heads(&p.k_out, 2);
  if (rc != 0) return rc;
  if (p.rows < 0 || (p.q.data && (p.q_heads <= 0 || p.q_heads > 65535))) return WUSH_ERR_BAD_SHAPE;
  if (p.rope) {
    if (p.rope_rows <= 0 || p.rotary <= 0 || p.rotary % 16 || p.rotary > p.kv.dim) return WUSH_ERR_BAD_SHAPE;
    if (!aligned16(p.rope)) return WUSH_ERR_BAD_ALIGNMENT;
  } else {
    p.rotary = 0;
  }
  if (!p.q.data) p.q_heads = 0;
  if (p.rows == 0) return WUSH_OK;
  if (!p.seq_ids || !p.positions) return WUSH_ERR_NULL_POINTER;
  if ((rc = require_sm100()) != 0) return rc;
  const int64_t units = p.rows * (int64_t)(p.q_heads + 2 * p.kv.heads) * ((p.kv.dim + 15) / 16 + 1);
  const unsigned grid = (unsigned)min((units + 255) / 256, (int64_t)sm_count() * 32);
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, (cudaStream_t)p.stream>>>(p);
    return (int)cudaGetLastError();
  };
  if (p.type == WUSH_TYPE_BF16)
    return p.kv.type == WUSH_TYPE_E4M3 ? go(append_kernel<__nv_bfloat16, __nv_fp8_e4m3>) : go(append_kernel<__nv_bfloat16, __nv_bfloat16>);
  return p.kv.type == WUSH_TYPE_E4M3 ? go(append_kernel<__half, __nv_fp8_e4m3>) : go(append_kernel<__half, __half>);
}

extern "C" int wush_kv_bounds(const wush_kv_bounds_args* args) {
  if (!args) return WUSH_ERR_NULL_POINTER;
  const wush_kv_pages& kv = args->kv;
  const wush_kv_table& table = args->table;
  int rc = check_pages(&kv, &table, kv.type == WUSH_TYPE_FP16 ? WUSH_TYPE_FP16 : WUSH_TYPE_BF16);
  if (rc != 0) return rc;
  if (!kv.bounds) return WUSH_ERR_NULL_POINTER;
  if (args->new_tokens < 0) return WUSH_ERR_BAD_SHAPE;
  // the bounds hold stored keys exactly: their type is the cache's, or either 16-bit type for E4M3
  if (kv.type != WUSH_TYPE_E4M3 && kv.bounds_type != kv.type) return WUSH_ERR_BAD_FLAG;
  if (table.seqs == 0 || args->new_tokens == 0) return WUSH_OK;
  if (!args->seq_lens) return WUSH_ERR_NULL_POINTER;
  if ((rc = require_sm100()) != 0) return rc;
  const int64_t most = min(table.width, (args->new_tokens - 1) / kv.page_size + 2);   // pages that the last tokens can touch
  const int64_t warps = table.seqs * most * kv.heads;
  const unsigned grid = (unsigned)min((warps + 7) / 8, (int64_t)sm_count() * 32);
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, (cudaStream_t)args->stream>>>(kv, table, args->seq_lens, args->new_tokens, most, args->status);
    return (int)cudaGetLastError();
  };
  if (kv.type == WUSH_TYPE_BF16) return go(bounds_kernel<__nv_bfloat16, __nv_bfloat16>);
  if (kv.type == WUSH_TYPE_FP16) return go(bounds_kernel<__half, __half>);
  return kv.bounds_type == WUSH_TYPE_BF16 ? go(bounds_kernel<__nv_fp8_e4m3, __nv_bfloat16>) : go(bounds_kernel<__nv_fp8_e4m3, __half>);
}

extern "C" size_t wush_kv_select_workspace_bytes(int64_t seqs, int heads, int64_t width) {
  return seqs > 0 && heads > 0 && width > 0 ? (size_t)seqs * heads * width * 8 : 0;
}

extern "C" int wush_kv_select_pages(const wush_kv_select_args* args) {
  if (!args) return WUSH_ERR_NULL_POINTER;
  const wush_kv_select_args& a = *args;
  int rc = check_pages(&a.kv, &a.table, a.type);
  if (rc != 0) return rc;
  if (!a.kv.bounds) return WUSH_ERR_NULL_POINTER;
  if (a.q_heads <= 0 || a.q_heads % a.kv.heads || a.top <= 0 || a.sink < 0 || a.recent < 0 || a.sink > a.top || a.recent > a.top - a.sink)
    return WUSH_ERR_BAD_SHAPE;
  if (a.table.seqs == 0) return WUSH_OK;
  if ((rc = check_heads(&a.q, 2)) != 0) return rc;
  if (!a.seq_lens || !a.pages || !a.counts || !a.workspace) return WUSH_ERR_NULL_POINTER;
  if (!aligned16(a.workspace)) return WUSH_ERR_BAD_ALIGNMENT;
  if (a.workspace_bytes < wush_kv_select_workspace_bytes(a.table.seqs, a.kv.heads, a.table.width)) return WUSH_ERR_WORKSPACE_TOO_SMALL;
  if (a.table.seqs * a.kv.heads > INT32_MAX) return WUSH_ERR_TOO_LARGE;
  if ((rc = require_sm100()) != 0) return rc;
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(a.workspace);
  const int64_t warps = a.table.seqs * a.kv.heads * a.table.width;
  const unsigned grid = (unsigned)min((warps + 7) / 8, (int64_t)sm_count() * 32);
  cudaStream_t stream = (cudaStream_t)a.stream;
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, stream>>>(a.kv, a.table, a.q, a.q_heads / a.kv.heads, a.seq_lens, a.top, keys, a.status);
    return (int)cudaGetLastError();
  };
  if (a.type == WUSH_TYPE_BF16)
    rc = a.kv.bounds_type == WUSH_TYPE_BF16 ? go(score_kernel<__nv_bfloat16, __nv_bfloat16>) : go(score_kernel<__nv_bfloat16, __half>);
  else
    rc = a.kv.bounds_type == WUSH_TYPE_BF16 ? go(score_kernel<__half, __nv_bfloat16>) : go(score_kernel<__half, __half>);
  if (rc != 0) return rc;
  select_kernel<<<(unsigned)(a.table.seqs * a.kv.heads), 1024, 0, stream>>>(
      a.kv.page_size, a.table.width, a.kv.heads, a.seq_lens, keys, a.top, a.sink, a.recent, a.pages, a.counts);
  return (int)cudaGetLastError();
}
