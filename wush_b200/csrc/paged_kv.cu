// Paged key-value cache: append with rotation, per-page bounds of the keys, selection of pages.
#include <type_traits>

#include "paged_kv.cuh"

namespace wush {
namespace kv {

// ---- append --------------------------------------------------------------------------------------------------------
using AppendParams = wush_kv_append_args;

// 16 bytes that are read once, past the L1 (not through the read-only path: the outputs may be the inputs)
template <typename T>
__device__ __forceinline__ uint4 load_once(const T* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <typename T>
__device__ __forceinline__ void widen8(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = to_float2<T>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// One block per row and `span` heads.  A thread has one unit of 16 channels (two chunks of 8 that are turned against each
// other, or two that are only copied) of every `lanes`-th head, so that the angles of its unit are loaded once for all of them.
// A pure pass over memory: q, k and v once in, once out.  BATCH heads are under way while the row's position and page are
// looked up (position, then page and angles: a chain of two latencies that a block would otherwise wait for with nothing
// in flight).
constexpr int APPEND_BATCH = 5, APPEND_THREADS = 128;
template <typename T, typename C>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const AppendParams p, int span) {
  const int d = p.kv.dim, units = (d + 15) >> 4, lanes = APPEND_THREADS / units, turned = p.rotary >> 4;
  const int u = threadIdx.x % units, lane = threadIdx.x / units;
  if (lane >= lanes) return;
  // The first channels of the chunks: of a value, and of a query or key, whose first `turned` units are the rotary channels.
  // Neighbouring threads have neighbouring chunks (a thread with two neighbouring ones would touch every 32-byte sector twice:
  // 230 us instead of 200 for 25000 tokens).  Interleaved pairs lie within a chunk, so any two chunks do.
  const bool turn = u < turned;
  const int va = u * 8, vb = (u + units) * 8;
  const int ca = turn ? u * 8 : p.rotary + (u - turned) * 8, cb = turn ? ca + p.rotary / 2 : ca + (units - turned) * 8;
  const int q_heads = p.q_heads, first_head = blockIdx.y * span, all_heads = min(q_heads + 2 * p.kv.heads, first_head + span);
  uint4 in[APPEND_BATCH][2];
  auto load = [&](int64_t row, int h0) {
#pragma unroll
    for (int i = 0; i < APPEND_BATCH; ++i) {
      const int h = h0 + i * lanes;
      if (h >= all_heads) continue;
      const bool value = h >= q_heads + p.kv.heads;
      const wush_heads& src = h < q_heads ? p.q : (value ? p.v : p.k);
      const int head = h < q_heads ? h : h - q_heads - (value ? p.kv.heads : 0);
      const T* from = reinterpret_cast<const T*>(src.data) + row * src.row + head * src.head;
      const int a = value ? va : ca, b = value ? vb : cb;
      in[i][0] = load_once(from + a);
      in[i][1] = b < d ? load_once(from + b) : make_uint4(0, 0, 0, 0);
    }
  };
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    load(row, first_head + lane);
    const int seq = p.seq_ids[row], pos = p.positions[row];
    if (seq < 0 || pos < 0) continue;
    if (seq >= p.table.seqs || pos >= p.table.width * p.kv.page_size || (p.rope && pos >= p.rope_rows)) {
      report_index(p.status);
      continue;
    }
    const int lp = pos / p.kv.page_size, at = pos - lp * p.kv.page_size;
    const int page = lookup_page(p.table, seq, lp, p.kv.num_pages, p.status);
    if (page < 0) continue;
    float cosine[8], sine[8];
    if (turn) {
      // pairs (i, i + rotary/2): angles 8u to 8u + 7; interleaved: the four of the first chunk, then the second's
      const float4* c = reinterpret_cast<const float4*>(p.rope + (int64_t)pos * p.rotary + (p.interleaved ? u * 4 : u * 8));
      const float4* s = c + p.rotary / 8;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = p.interleaved ? i * (p.rotary / 16) : i;
        const float4 x = __ldg(c + j), y = __ldg(s + j);
        cosine[4 * i] = x.x, cosine[4 * i + 1] = x.y, cosine[4 * i + 2] = x.z, cosine[4 * i + 3] = x.w;
        sine[4 * i] = y.x, sine[4 * i + 1] = y.y, sine[4 * i + 2] = y.z, sine[4 * i + 3] = y.w;
      }
    }
    for (int h0 = first_head + lane; h0 < all_heads; h0 += lanes * APPEND_BATCH) {
      if (h0 != first_head + lane) load(row, h0);
#pragma unroll
      for (int i = 0; i < APPEND_BATCH; ++i) {
        const int h = h0 + i * lanes;
        if (h >= all_heads) continue;
        const bool query = h < q_heads, value = h >= q_heads + p.kv.heads;
        const int head = query ? h : h - q_heads - (value ? p.kv.heads : 0);
        const int ac = value ? va : ca, bc = value ? vb : cb;
        const bool two = bc < d;
        float a[8], b[8];
        widen8<T>(in[i][0], a);
        widen8<T>(in[i][1], b);
        if (turn && !value) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float& x = p.interleaved ? (j < 4 ? a[2 * j] : b[2 * j - 8]) : a[j];
            float& y = p.interleaved ? (j < 4 ? a[2 * j + 1] : b[2 * j - 7]) : b[j];
            const float nx = __fsub_rn(__fmul_rn(x, cosine[j]), __fmul_rn(y, sine[j]));
            const float ny = __fadd_rn(__fmul_rn(y, cosine[j]), __fmul_rn(x, sine[j]));
            x = nx;
            y = ny;
          }
        }
        if (query || (!value && p.k_out.data)) {
          const wush_heads& dst = query ? p.q_out : p.k_out;
          T* o = reinterpret_cast<T*>(dst.data) + row * dst.row + head * dst.head;
          store8(o + ac, a);
          if (two) store8(o + bc, b);
        }
        if (query) continue;
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
        store8(o + ac, a);
        if (two) store8(o + bc, b);
      }
    }
  }
}

// ---- bounds --------------------------------------------------------------------------------------------------------
// Packed minimum and maximum that keep a NaN, of bf16 pairs (bf16 pages) or fp16 pairs (fp16 pages, and E4M3 values widened).
template <typename C>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<C, __nv_bfloat16>::value) asm("min.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename C>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (std::is_same<C, __nv_bfloat16>::value) asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// A warp works on `span` consecutive pages of one (sequence, head), whose places its lanes look up together; a lane takes 16
// bytes of every n-th row, and the next BOUNDS_ROWS rows, of this page or the next, are under way while it compares those it
// has.  (A page a warp without that: 3.9 TB/s whatever the batch, every warp waiting for length, page and rows in turn.)
constexpr int BOUNDS_ROWS = 8, BOUNDS_SPAN = 8;
template <typename C, typename B>
__global__ void __launch_bounds__(128) bounds_kernel(const wush_kv_pages kv, const wush_kv_table table, const int32_t* seq_lens,
                                                     int64_t new_tokens, int64_t most, int span, int* status) {
  constexpr int CH = 16 / (int)sizeof(C), PAIRS = CH / 2;    // channels of a lane
  using P = typename std::conditional<std::is_same<C, __nv_bfloat16>::value, __nv_bfloat16, __half>::type;
  const int lane = threadIdx.x & 31;
  const int across = (kv.dim + CH - 1) / CH, down = 32 / across;   // lanes of a row, rows of a warp
  const int piece = lane % across, row0 = lane / across;
  const int64_t groups = (most + span - 1) / span, total = table.seqs * groups * kv.heads;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total; w += warps) {
    const int64_t slot = w / kv.heads, seq = slot / groups;
    const int head = (int)(w - slot * kv.heads);
    const int len = clamp_length(seq_lens[seq], table.width * kv.page_size, status);
    const int64_t first = (len > new_tokens ? len - new_tokens : 0) / kv.page_size + (slot - seq * groups) * span;
    const int64_t behind = min((int64_t)(len + kv.page_size - 1) / kv.page_size, first + span);   // one past the last page
    if (first >= behind) continue;
    const int pages = (int)(behind - first);
    const int my_page = lane < pages ? lookup_page(table, seq, (int)first + lane, kv.num_pages, status) : -1;
    const C* base = reinterpret_cast<const C*>(kv.k) + head * kv.k_head + piece * CH;
    auto rows_of = [&](int i) { return (int)min((int64_t)kv.page_size, len - (first + i) * kv.page_size); };
    uint4 v[BOUNDS_ROWS], ahead[BOUNDS_ROWS];
    auto load = [&](int i, int r0) {                         // rows r0, r0 + down, ... of page i; past the last: that again
      const int page = max(0, __shfl_sync(0xffffffffu, my_page, i)), rows = rows_of(i);
      const C* k = base + page * kv.k_page;
#pragma unroll
      for (int x = 0; x < BOUNDS_ROWS; ++x) ahead[x] = ld_nc_v4(k + min(row0 < down ? r0 + row0 + x * down : 0, rows - 1) * kv.k_row);
    };
    uint32_t lo[PAIRS], hi[PAIRS];
    load(0, 0);
    for (int i = 0, r0 = 0; i < pages;) {
      const int rows = rows_of(i), next_r = r0 + down * BOUNDS_ROWS;
      const bool start = r0 == 0, ends = next_r >= rows;
      const int page = __shfl_sync(0xffffffffu, my_page, i);
#pragma unroll
      for (int x = 0; x < BOUNDS_ROWS; ++x) v[x] = ahead[x];
      if (!ends) load(i, next_r);
      else if (i + 1 < pages) load(i + 1, 0);
#pragma unroll
      for (int y = 0; y < BOUNDS_ROWS; ++y) {
        const uint32_t word[4] = {v[y].x, v[y].y, v[y].z, v[y].w};
        uint32_t pair[PAIRS];
        if constexpr (sizeof(C) == 1) {
#pragma unroll
          for (int x = 0; x < 4; ++x) e4m3x4_to_f16x4(word[x], pair[2 * x], pair[2 * x + 1]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) pair[x] = word[x];
        }
#pragma unroll
        for (int x = 0; x < PAIRS; ++x) {
          lo[x] = start && y == 0 ? pair[x] : min2<C>(lo[x], pair[x]);
          hi[x] = start && y == 0 ? pair[x] : max2<C>(hi[x], pair[x]);
        }
      }
      i += ends;
      r0 = ends ? 0 : next_r;
      if (!ends) continue;
      uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<B*>(kv.bounds) + ((int64_t)max(page, 0) * kv.heads + head) * 2 * kv.dim + piece * CH);
      auto store = [&](int x, uint32_t l, uint32_t h) {        // pair x of the lane's piece
        if constexpr (std::is_same<P, B>::value) {
          out[x] = l;
          out[kv.dim / 2 + x] = h;
        } else {                                               // E4M3 values: exact in either type
          const float2 fl = to_float2<P>(l), fh = to_float2<P>(h);
          out[x] = pack2<B>(fl.x, fl.y);
          out[kv.dim / 2 + x] = pack2<B>(fh.x, fh.y);
        }
      };
      if ((across & (across - 1)) == 0) {
        // lanes of the same channels exchange halves of what they hold: 12 shuffles for 4 rows of 16 channels instead of 96
        int offset = 0, held = PAIRS;
        bool writes = true;
#pragma unroll
        for (int s = 0; s < 5; ++s) {
          if (1 << s >= down) break;
          const int half = PAIRS >> (s + 1), partner = across << s;
          const bool upper = lane & partner;
          if (half > 0) {
#pragma unroll
            for (int x = 0; x < half; ++x) {
              const uint32_t kl = upper ? lo[x + half] : lo[x], sl = upper ? lo[x] : lo[x + half];
              const uint32_t kh = upper ? hi[x + half] : hi[x], sh = upper ? hi[x] : hi[x + half];
              lo[x] = min2<C>(kl, __shfl_xor_sync(0xffffffffu, sl, partner));
              hi[x] = max2<C>(kh, __shfl_xor_sync(0xffffffffu, sh, partner));
            }
            offset += upper ? half : 0;
            held = half;
          } else {
            lo[0] = min2<C>(lo[0], __shfl_xor_sync(0xffffffffu, lo[0], partner));
            hi[0] = max2<C>(hi[0], __shfl_xor_sync(0xffffffffu, hi[0], partner));
            writes = writes && !upper;
          }
        }
        if (writes && page >= 0) {
#pragma unroll
          for (int x = 0; x < PAIRS; ++x)
            if (x < held) store(offset + x, lo[x], hi[x]);
        }
      } else {
        for (int g = 1; g < down; ++g) {                       // the other rows' lanes, one after another
#pragma unroll
          for (int x = 0; x < PAIRS; ++x) {
            lo[x] = min2<C>(lo[x], __shfl_sync(0xffffffffu, lo[x], g * across + piece));
            hi[x] = max2<C>(hi[x], __shfl_sync(0xffffffffu, hi[x], g * across + piece));
          }
        }
        if (row0 == 0 && page >= 0) {
#pragma unroll
          for (int x = 0; x < PAIRS; ++x) store(x, lo[x], hi[x]);
        }
      }
    }
  }
}

// ---- selection -----------------------------------------------------------------------------------------------------
// A score as a 64-bit key with the same order; one that is not finite counts as +infinity.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (!(fabs(s) <= 1.7976931348623157e308)) return ~0ull;
  const long long b = __double_as_longlong(s + 0.0);       // -0 + 0 = +0: equal numbers, equal keys
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

__device__ __forceinline__ void mma_f64(double (&d)[2], double a, double b) {
  asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};\n" : "+d"(d[0]), "+d"(d[1]) : "d"(a), "d"(b));
}

// Keys of the scores: sum_d max(q_d lower_d, q_d upper_d) = sum_d q+_d upper_d + q-_d lower_d, with q+ and q- the positive and
// negative parts: products [8 queries x 4 channels] . [4 channels x 8 pages] in 64 bits.  (A bound that is not finite makes
// one of its two terms infinite or NaN whatever the query is.)  As in the attention, a product does not care which channel
// is which, so a lane takes 8 neighbouring channels of a page with one load and feeds them to 8 products; the queries are
// laid out to match in shared memory.  A unit of work is 64 pages of one (sequence, key head), 16 a warp; the units of all
// sequences that have more than `top` pages are numbered through, and every block takes an equal run of them.
// The bounds are asked for before the queries are laid out (J: steps of 32 channels; 2 of them at a time).
constexpr int SCORE_WARPS = 4, SCORE_PAGES = 16 * SCORE_WARPS;
template <typename T, typename B, int J>
__global__ void __launch_bounds__(SCORE_WARPS * 32, J <= 4 ? 4 : 3) score_kernel(const wush_kv_select_args a, int group, unsigned long long* keys) {
  extern __shared__ double sm_q[];                           // [parts][channels / 32][8][8 queries][4]
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int d = a.kv.dim, heads = a.kv.heads;
  auto pages_of = [&](int64_t seq) {
    const int len = clamp_length(a.seq_lens[seq], a.table.width * a.kv.page_size, a.status);
    return (len + a.kv.page_size - 1) / a.kv.page_size;
  };
  auto units_of = [&](int64_t seq) -> int64_t {              // of one key head
    if (seq >= a.table.seqs) return 0;
    const int n = pages_of(seq);
    return n > a.top ? (n + SCORE_PAGES - 1) / SCORE_PAGES : 0;
  };
  int64_t total = 0;
  for (int64_t s0 = lane; s0 < a.table.seqs; s0 += 32) total += units_of(s0);
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  total *= heads;
  const int64_t per = (total + gridDim.x - 1) / gridDim.x, unit_end = min(total, (blockIdx.x + 1) * per);
  int64_t unit = blockIdx.x * per;
  if (unit >= unit_end) return;
  int64_t seq = 0, base = 0, units = 0;                      // the sequence the unit lies in, and its first unit
  for (int64_t s0 = 0;; s0 += 32) {
    units = units_of(s0 + lane);
    int64_t sum = units * heads;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned beyond = __ballot_sync(0xffffffffu, base + sum > unit);
    if (beyond) {
      const int at = __ffs(beyond) - 1;
      seq = s0 + at;
      units = __shfl_sync(0xffffffffu, units, at);
      base += __shfl_sync(0xffffffffu, sum, at) - units * heads;
      break;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  int laid_out = -1;                                         // key head whose queries are in shared memory
  for (; unit < unit_end; ++unit) {
    while (unit >= base + units * heads) {
      base += units * heads;
      units = units_of(++seq);
      laid_out = -1;
    }
    const int n = pages_of(seq), head = (int)((unit - base) / units), page0 = (int)((unit - base) % units) * SCORE_PAGES;
    const int64_t entry = seq * heads + head;
    const B* bound[2];                                         // of the lane's two pages
    bool known[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int lp = page0 + warp * 16 + x * 8 + r;
      const int page = lp < n ? lookup_page(a.table, seq, lp, a.kv.num_pages, a.status) : -1;
      known[x] = page >= 0;
      bound[x] = reinterpret_cast<const B*>(a.kv.bounds) + ((int64_t)max(page, 0) * heads + head) * 2 * d;
    }
    constexpr int HELD = 2;
    uint4 raw[HELD][2][2];                                     // [step][page][lower, upper]
    auto ask = [&](int j0) {
#pragma unroll
      for (int j = 0; j < HELD; ++j) {
        const int ch = ((j0 + j) * 4 + c) * 8;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            raw[j][x][y] = make_uint4(0, 0, 0, 0);
            if (known[x] && ch < d) raw[j][x][y] = __ldg(reinterpret_cast<const uint4*>(bound[x] + y * d + ch));
          }
      }
    };
    ask(0);
    double best[2][2] = {{-INFINITY, -INFINITY}, {-INFINITY, -INFINITY}};
    bool bad[2][2] = {{false, false}, {false, false}};         // a score that is not finite
    for (int g0 = 0; g0 < group; g0 += 8) {
      if (group > 8 || laid_out != head) {
        __syncthreads();
        for (int i = threadIdx.x; i < J * 32; i += SCORE_WARPS * 32) {   // 8 channels of one query
          const int row = i / (J * 4), piece = i % (J * 4);
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (g0 + row < group && piece * 8 < d)
          load8(reinterpret_cast<const T*>(a.q.data) + seq * a.q.row + (int64_t)(head * group + g0 + row) * a.q.head + piece * 8, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          double* at = sm_q + ((piece >> 2) * 8 + e) * 32 + row * 4 + (piece & 3);
          at[0] = x[e] > 0.0f ? (double)x[e] : 0.0;
          at[J * 256] = x[e] > 0.0f ? 0.0 : (double)x[e];      // (a NaN query lands here)
        }
      }
      laid_out = head;
      __syncthreads();
      }
      // eight chains: a 64-bit product takes about 200 cycles to come back
      double part[2][2][2][2] = {};                            // [page][sign][channel parity][element]
      for (int j0 = 0; j0 < J; j0 += HELD) {
        if (j0 > 0 || g0 > 0) ask(j0);
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
          const double* plus = sm_q + (j0 + j) * 256 + lane;
#pragma unroll
          for (int e2 = 0; e2 < 4; ++e2) {
            float2 lo[2], hi[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t l[4] = {raw[j][x][0].x, raw[j][x][0].y, raw[j][x][0].z, raw[j][x][0].w};
              const uint32_t h[4] = {raw[j][x][1].x, raw[j][x][1].y, raw[j][x][1].z, raw[j][x][1].w};
              lo[x] = to_float2<B>(l[e2]);
              hi[x] = to_float2<B>(h[e2]);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const double qp = plus[(2 * e2 + y) * 32], qm = plus[J * 256 + (2 * e2 + y) * 32];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                mma_f64(part[x][0][y], qp, (double)(y ? hi[x].y : hi[x].x));
                mma_f64(part[x][1][y], qm, (double)(y ? lo[x].y : lo[x].x));
              }
            }
          }
        }
      }
      double s[2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) s[x][y] = (part[x][0][0][y] + part[x][0][1][y]) + (part[x][1][0][y] + part[x][1][1][y]);
      // the lane has query g0 + r and pages 2c, 2c + 1 of each 8
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (g0 + r >= group) continue;
          bad[x][y] |= !(fabs(s[x][y]) <= 1.7976931348623157e308);
          best[x][y] = fmax(best[x][y], s[x][y]);
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        double top = best[x][y];
        unsigned any = bad[x][y];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
          any |= __shfl_xor_sync(0xffffffffu, any, o);
        }
        const bool known_page = __shfl_sync(0xffffffffu, known[x], (2 * c + y) * 4);
        const int lp = page0 + warp * 16 + x * 8 + 2 * c + y;
        // a page outside the pool comes last: the attention would leave it out
        if (r == 0 && lp < n) keys[entry * a.table.width + lp] = !known_page ? 0 : (any ? ~0ull : score_key(top));
      }
  }
}

// Exclusive sums over `count` <= 256 numbers in shared memory, by one warp; returns the total.
__device__ __forceinline__ int scan256(int* x, int count) {
  const int lane = threadIdx.x & 31;
  int mine[8], sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mine[i] = sum;
    sum += lane * 8 + i < count ? x[lane * 8 + i] : 0;
  }
  int before = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += y;
  }
  const int total = __shfl_sync(0xffffffffu, before, 31);
  before -= sum;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane * 8 + i < count) x[lane * 8 + i] = before + mine[i];
  return total;
}

// One block per (sequence, key head).  A radix selection from the first bit in which the keys differ: 8 bits at a time the
// keys that share the threshold's leading bits are counted by their next digit, until all of them are wanted or all bits are
// known; the last of them are then taken in the order of their pages.  A thread holds every blockDim-th key, up to ROWS of
// them (ROWS is 8, or 0 for more pages than that: then they are read again for every pass).
template <int ROWS>
__global__ void __launch_bounds__(1024) select_kernel(const wush_kv_select_args a, const unsigned long long* keys) {
  __shared__ int hist[256];
  __shared__ unsigned long long sm_low[32], sm_high[32];
  __shared__ int sm_digit, sm_need, sm_count;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
  const int64_t item = blockIdx.x;
  const int len = (int)max((int64_t)0, min((int64_t)a.seq_lens[item / a.kv.heads], a.table.width * a.kv.page_size));
  const int n = (len + a.kv.page_size - 1) / a.kv.page_size, top = a.top;
  int32_t* out = a.pages + item * top;
  const int count = min(n, top);
  if (tid == 0) a.counts[item] = count;
  for (int i = count + tid; i < top; i += threads) out[i] = -1;
  if (n <= top) {
    for (int i = tid; i < n; i += threads) out[i] = i;
    return;
  }
  const int begin = a.sink, end = n - a.recent;              // pages that compete
  const unsigned long long* from = keys + item * a.table.width;
  unsigned long long held[ROWS > 0 ? ROWS : 1];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int i = j * threads + tid;
    held[j] = i >= begin && i < end ? from[i] : 0;
  }
  const int rounds = ROWS > 0 ? ROWS : (n + threads - 1) / threads;
  auto key_of = [&](int j) { return ROWS > 0 ? held[ROWS > 0 ? j : 0] : from[j * threads + tid]; };
  auto competes = [&](int j) {
    const int i = j * threads + tid;
    return i >= begin && i < end;
  };

  // smallest and largest key: the bits before the first in which they differ need no passes
  unsigned long long low = ~0ull, high = 0;
#pragma unroll
  for (int j = 0; j < rounds; ++j)
    if (competes(j)) {
      const unsigned long long k = key_of(j);
      low = k < low ? k : low;
      high = k > high ? k : high;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long x = __shfl_xor_sync(0xffffffffu, low, o), y = __shfl_xor_sync(0xffffffffu, high, o);
    low = x < low ? x : low;
    high = y > high ? y : high;
  }
  if (lane == 0) {
    sm_low[warp] = low;
    sm_high[warp] = high;
  }
  __syncthreads();
  for (int w = 0; w < warps; ++w) {
    low = sm_low[w] < low ? sm_low[w] : low;
    high = sm_high[w] > high ? sm_high[w] : high;
  }
  int need = top - a.sink - a.recent, among = end - begin;   // wanted among the keys that match the prefix
  int shift = low == high ? 0 : 64 - __clzll(low ^ high);    // bits of a key that are not known
  unsigned long long prefix = shift == 64 ? 0 : high >> shift;
  auto matches = [&](unsigned long long k) { return shift == 64 || k >> shift == prefix; };
  while (need > 0 && need < among && shift > 0) {
    const int bits = min(8, shift), next = shift - bits;
    for (int i = tid; i < 256; i += threads) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < rounds; ++j)
      if (competes(j)) {
        const unsigned long long k = key_of(j);
        if (matches(k)) atomicAdd(&hist[(int)(k >> next) & ((1 << bits) - 1)], 1);
      }
    __syncthreads();
    if (warp == 0) {                                         // the digit that the need-th largest key has
      int mine[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += mine[i] = hist[255 - (lane * 8 + i)];
      int before = sum;
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      before -= sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (before < need && need <= before + mine[i]) {
          sm_digit = 255 - (lane * 8 + i);
          sm_need = need - before;
          sm_count = mine[i];
        }
        before += mine[i];
      }
    }
    __syncthreads();
    prefix = (shift == 64 ? 0 : prefix << bits) | (unsigned)sm_digit;
    need = sm_need;
    among = sm_count;
    shift = next;
  }

  // Take the keys above the prefix and the first `need` of those that match it; place them in the order of the pages, 8 rounds
  // at a time.  hist holds the counts of (round, warp): 8 * 32 at most.
  int taken_before = 0, equal_before = 0;
  for (int j0 = 0; j0 < rounds; j0 += 8) {
    unsigned equal = 0, take = 0;                            // one bit a round
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int j = j0 + x, i = j * threads + tid;
      const bool in = need > 0 && competes(j);
      const unsigned long long k = in ? key_of(ROWS > 0 ? x : j) : 0;
      equal |= (unsigned)(in && matches(k)) << x;
      take |= (unsigned)((i < n && (i < begin || i >= end)) || (in && shift < 64 && k >> shift > prefix)) << x;
    }
    if (need < among) {                                      // not all that match: by rank
      __syncthreads();
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const unsigned m = __ballot_sync(0xffffffffu, equal >> x & 1);
        if (lane == 0) hist[x * warps + warp] = __popc(m);
      }
      __syncthreads();
      if (warp == 0) {
        const int total = scan256(hist, 8 * warps);
        if (lane == 0) sm_count = total;
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const unsigned m = __ballot_sync(0xffffffffu, equal >> x & 1);
        if ((equal >> x & 1) && equal_before + hist[x * warps + warp] + __popc(m & ((1u << lane) - 1)) < need) take |= 1u << x;
      }
      equal_before += sm_count;
    } else {
      take |= equal;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const unsigned m = __ballot_sync(0xffffffffu, take >> x & 1);
      if (lane == 0) hist[x * warps + warp] = __popc(m);
    }
    __syncthreads();
    if (warp == 0) {
      const int total = scan256(hist, 8 * warps);
      if (lane == 0) sm_count = total;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const unsigned m = __ballot_sync(0xffffffffu, take >> x & 1);
      if (take >> x & 1) out[taken_before + hist[x * warps + warp] + __popc(m & ((1u << lane) - 1))] = (j0 + x) * threads + tid;
    }
    taken_before += sm_count;
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
  // All heads of a row in one block where every SM gets a row, and then four blocks an SM that walk over the rows (25000
  // tokens: 188 us, a block a row 200 us); one head a thread otherwise (one token: 2.8 us, all heads in one block 4.1 us).
  const int all_heads = p.q_heads + 2 * p.kv.heads, lanes = APPEND_THREADS / ((p.kv.dim + 15) / 16), sms = sm_count();
  const int span = p.rows >= sms ? all_heads : lanes;
  const dim3 grid((unsigned)min(p.rows, (int64_t)sms * 4), (all_heads + span - 1) / span);
  auto go = [&](auto kern) {
    kern<<<grid, APPEND_THREADS, 0, (cudaStream_t)p.stream>>>(p, span);
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
  // one page a warp until every SM has 16 warps
  const int sms = sm_count();
  const int span = (int)min((int64_t)BOUNDS_SPAN, max((int64_t)1, table.seqs * most * kv.heads / (16 * sms)));
  const int64_t warps = table.seqs * ((most + span - 1) / span) * kv.heads;
  const unsigned grid = (unsigned)min((warps + 3) / 4, (int64_t)sms * 64);
  auto go = [&](auto kern) {
    kern<<<grid, 128, 0, (cudaStream_t)args->stream>>>(kv, table, args->seq_lens, args->new_tokens, most, span, args->status);
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
  const int64_t units = a.table.seqs * a.kv.heads * ((a.table.width + SCORE_PAGES - 1) / SCORE_PAGES);
  // the kernels may be launched while the one before still runs, and wait for it before they read anything
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = (cudaStream_t)a.stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(SCORE_WARPS * 32);
  auto go = [&](auto kern, int steps) {
    cfg.gridDim = dim3((unsigned)min(units, (int64_t)sm_count() * (steps <= 4 ? 4 : 3)));
    cfg.dynamicSmemBytes = (size_t)steps * 512 * sizeof(double);
    return (int)cudaLaunchKernelEx(&cfg, kern, a, a.q_heads / a.kv.heads, keys);
  };
  auto by_dim = [&](auto t, auto b) {
    using T = decltype(t);
    using B = decltype(b);
    return a.kv.dim <= 64 ? go(score_kernel<T, B, 2>, 2) : (a.kv.dim <= 128 ? go(score_kernel<T, B, 4>, 4) : go(score_kernel<T, B, 8>, 8));
  };
  const __nv_bfloat16 bf = {};
  const __half hf = {};
  if (a.type == WUSH_TYPE_BF16) rc = a.kv.bounds_type == WUSH_TYPE_BF16 ? by_dim(bf, bf) : by_dim(bf, hf);
  else rc = a.kv.bounds_type == WUSH_TYPE_BF16 ? by_dim(hf, bf) : by_dim(hf, hf);
  if (rc != 0) return rc;
  // 8 keys a thread in registers while that is enough
  int threads = 128;
  while (threads < 1024 && threads * 8 < a.table.width) threads *= 2;
  cfg.gridDim = dim3((unsigned)(a.table.seqs * a.kv.heads));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = 0;
  if (threads * 8 >= a.table.width) return (int)cudaLaunchKernelEx(&cfg, select_kernel<8>, a, (const unsigned long long*)keys);
  return (int)cudaLaunchKernelEx(&cfg, select_kernel<0>, a, (const unsigned long long*)keys);
}
