// Paged key-value cache: append with rotation, per-page bounds of the keys, selection of pages.
#include <cfloat>
#include <type_traits>

#include "paged_kv.cuh"

namespace wush {
namespace kv {

// ---- append --------------------------------------------------------------------------------------------------------
using AppendParams = wush_kv_append_args;

// 16 bytes that are read once, past the L1.  Nothing here goes through the read-only path (ld.global.nc): outputs may be the
// inputs, and a kernel that is launched early is there while the one before it still writes what will be read.
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

// A block takes `span` heads of a row, and the grid walks over the rows.  A thread has one unit of 16 channels (two chunks of 8
// that are turned against each other, or two that are only copied) of every `lanes`-th head, so that the angles of its unit are
// loaded once for all of them.  A pure pass over memory: q, k and v once in, once out.  BATCH heads are under way while the
// row's position and page are looked up (position, then page and angles: a chain of two latencies that a block would otherwise
// wait for with nothing in flight).
constexpr int APPEND_BATCH = 5, APPEND_THREADS = 128;
template <typename T, typename C>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const AppendParams p, int span) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
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
        const float4 x = __ldca(c + j), y = __ldca(s + j);       // (plain loads: 25000 tokens 193 us, so 190)
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
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
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
    const int64_t behind = min((int64_t)pages_of_length(len, kv.page_size), first + span);   // one past the last page
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
      for (int x = 0; x < BOUNDS_ROWS; ++x) ahead[x] = load_once(k + min(row0 < down ? r0 + row0 + x * down : 0, rows - 1) * kv.k_row);
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
// The score of a page for a key head is max over its queries of sum_d max(q_d lower_d, q_d upper_d), and the choice has to be
// the one that exact scores give.  64-bit sums of all of them cost 35 us where their bounds can be read in 11 (64-bit products,
// on either pipe, were the limit), so the work is divided:
//   1. score_kernel computes every score on the tensor cores in fp32, with the sum of the terms' magnitudes;
//   2. select_kernel finds the k-th largest of them, and from the magnitudes an eps by which no score is off.  What is more
//      than 2 eps above the k-th largest is among the k best, what is more than 2 eps below it is not; the few pages between
//      are scored again in 64 bits and ranked.
// Error of an fp32 score: an m16n8k16 product of its own (nothing to add to) adds 16 exact products; if each addend and the
// result is cut to 24 bits at the scale of the largest, it is off by at most 17 * 2^-23 of its terms' magnitude.  The
// 4 * ceil(dim / 32) products of a score (a step of 32 channels makes two with the upper bounds and two with the lower) are
// added in fp32, 2^-24 of the magnitude each.  PTX leaves open how a product's sum is rounded; measured over terms of very
// mixed size the errors stay below an eighth of this bound (tests/test_paged_kv_contract_gpu.py holds them to it).  (Chained
// through the product's accumulator every product would add 18 * 2^-23 of the whole magnitude: 16 times as many pages lay
// between, and scoring them again took 5 to 10 us.)
struct Score {
  float value, magnitude;               // magnitude: infinity when fp32 does not hold the score
};

__device__ __forceinline__ uint32_t float_key(float x) {     // same order; equal numbers, equal keys
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// A 64-bit score as a key with the same order; one that is not finite counts as +infinity.
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (!(fabs(s) <= 1.7976931348623157e308)) return ~0ull;
  const long long b = __double_as_longlong(s + 0.0);         // -0 + 0 = +0: equal numbers, equal keys
  return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

// A pair of bounds in the queries' type; NaN where that is not exact (E4M3 keys are exact in both).
template <typename T, typename B>
__device__ __forceinline__ uint32_t as_query_type(uint32_t pair) {
  if constexpr (std::is_same<T, B>::value) {
    return pair;
  } else {
    const float2 f = to_float2<B>(pair);
    const uint32_t p = pack2<T>(f.x, f.y);
    const float2 back = to_float2<T>(p);
    return (p & (back.x == f.x ? 0xffffu : 0u)) | (back.x == f.x ? 0u : 0x7fffu) | (p & (back.y == f.y ? 0xffff0000u : 0u)) |
           (back.y == f.y ? 0u : 0x7fff0000u);
  }
}

// not 0 where one of a pair is infinite or NaN: the exponent's ones carry into the sign's place
template <typename B>
__device__ __forceinline__ uint32_t not_finite2(uint32_t pair) {
  return ((pair & 0x7fff7fffu) + (std::is_same<B, __half>::value ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}

// fp32 scores: products [16 pages x 16 channels] . [16 channels x 8 queries] of the upper bounds with the queries' positive
// parts, the lower bounds with their negative parts, and the larger magnitudes with their magnitudes.  As in the attention,
// a product does not care which channel is which: a lane takes 8 neighbouring channels of two pages with one load each.
// (A bound that is not finite makes one of its terms infinite or NaN whatever the query is.)  A unit of work is 16 pages of
// one (sequence, key head); the units of all sequences that have more than `top` pages are numbered through, and every warp
// takes an equal run of them.  J: steps of 32 channels.
constexpr int SCORE_WARPS = 4, SCORE_PAGES = 16, SCORE_BLOCKS = 3;
template <typename T, typename B, int J>
__global__ void __launch_bounds__(SCORE_WARPS * 32, J <= 4 ? SCORE_BLOCKS : 2) score_kernel(const wush_kv_select_args a, int group, Score* scores) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int d = a.kv.dim, heads = a.kv.heads;
  auto pages_of = [&](int64_t seq) {
    const int len = clamp_length(a.seq_lens[seq], a.table.width * a.kv.page_size, a.status);
    return pages_of_length(len, a.kv.page_size);
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
  const int64_t warps = (int64_t)gridDim.x * SCORE_WARPS, per = (total + warps - 1) / warps;
  int64_t unit = ((int64_t)blockIdx.x * SCORE_WARPS + (threadIdx.x >> 5)) * per;
  const int64_t unit_end = min(total, unit + per);
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
  // the pages of a unit are looked up one unit ahead
  struct Unit { int64_t seq; int head, page0, n, my_page; };
  auto find = [&](int64_t t) -> Unit {
    while (t >= base + units * heads) {
      base += units * heads;
      units = units_of(++seq);
    }
    Unit u{seq, (int)((uint64_t)(t - base) / (uint64_t)units), 0, pages_of(seq), -1};
    u.page0 = (int)(t - base - u.head * units) * SCORE_PAGES;
    const int lp = u.page0 + (lane & 15);
    if (lp < u.n) u.my_page = lookup_page(a.table, seq, lp, a.kv.num_pages, a.status);
    return u;
  };
  uint4 q[J];                                                // of the lane's query
  auto ask_queries = [&](const Unit& u, int g0) {
    const T* row = reinterpret_cast<const T*>(a.q.data) + u.seq * a.q.row + (int64_t)(u.head * group + min(g0 + r, group - 1)) * a.q.head;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int ch = (j * 4 + c) * 8;
      q[j] = ch < d ? *reinterpret_cast<const uint4*>(row + ch) : make_uint4(0, 0, 0, 0);
    }
  };
  Unit then = find(unit);
  int64_t held_seq = -1;
  int held_head = -1;
  for (; unit < unit_end; ++unit) {
    const Unit now = then;
    const int head = now.head;
    uint4 raw[J][2][2];                                      // [step][page r, r + 8][lower, upper]
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      // (a page that is not there reads the first page of the pool, whose scores are not kept)
      const int page = max(0, __shfl_sync(0xffffffffu, now.my_page, x * 8 + r));
      const B* bound = reinterpret_cast<const B*>(a.kv.bounds) + ((int64_t)page * heads + head) * 2 * d;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int ch = (j * 4 + c) * 8;
#pragma unroll
        for (int y = 0; y < 2; ++y) raw[j][x][y] = load_once(bound + y * d + (ch < d ? ch : 0));
      }
    }
    if (group > 8 || held_head != head || held_seq != now.seq) {
      ask_queries(now, 0);
      held_head = head;
      held_seq = now.seq;
    }
    if (unit + 1 < unit_end) then = find(unit + 1);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const bool in = (j * 4 + c) * 8 < d;
          uint4& v = raw[j][x][y];
          v = make_uint4(in ? as_query_type<T, B>(v.x) : 0, in ? as_query_type<T, B>(v.y) : 0, in ? as_query_type<T, B>(v.z) : 0,
                         in ? as_query_type<T, B>(v.w) : 0);
        }
    float best[2] = {-INFINITY, -INFINITY}, magnitude[2] = {0.0f, 0.0f};
    for (int g0 = 0; g0 < group; g0 += 8) {
      if (g0 > 0) ask_queries(now, g0);
      float s[4] = {}, m[4] = {};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const uint32_t qw[4] = {q[j].x, q[j].y, q[j].z, q[j].w};
        uint32_t lo[2][4], hi[2][4], big[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t l[4] = {raw[j][x][0].x, raw[j][x][0].y, raw[j][x][0].z, raw[j][x][0].w};
          const uint32_t h[4] = {raw[j][x][1].x, raw[j][x][1].y, raw[j][x][1].z, raw[j][x][1].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[x][i] = l[i];
            hi[x][i] = h[i];
            big[x][i] = max2<T>(lo[x][i] & 0x7fff7fffu, hi[x][i] & 0x7fff7fffu);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const uint32_t al[4] = {lo[0][i], lo[1][i], lo[0][i + 1], lo[1][i + 1]}, ah[4] = {hi[0][i], hi[1][i], hi[0][i + 1], hi[1][i + 1]};
          const uint32_t ab[4] = {big[0][i], big[1][i], big[0][i + 1], big[1][i + 1]};
          float plus[4] = {}, minus[4] = {};
          mma<T>(plus, ah[0], ah[1], ah[2], ah[3], max2<T>(qw[i], 0), max2<T>(qw[i + 1], 0));
          mma<T>(minus, al[0], al[1], al[2], al[3], min2<T>(qw[i], 0), min2<T>(qw[i + 1], 0));
#pragma unroll
          for (int x = 0; x < 4; ++x) s[x] += plus[x];
#pragma unroll
          for (int x = 0; x < 4; ++x) s[x] += minus[x];
          mma<T>(m, ab[0], ab[1], ab[2], ab[3], qw[i] & 0x7fff7fffu, qw[i + 1] & 0x7fff7fffu);
        }
      }
      // the lane has pages r and r + 8, and queries g0 + 2c and g0 + 2c + 1
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (g0 + 2 * c + y >= group) continue;
          const float v = s[2 * x + y], w = m[2 * x + y];
          best[x] = fmaxf(best[x], v);
          magnitude[x] = fabsf(v) <= FLT_MAX && w <= FLT_MAX ? fmaxf(magnitude[x], w) : INFINITY;
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        best[x] = fmaxf(best[x], __shfl_xor_sync(0xffffffffu, best[x], o));
        magnitude[x] = fmaxf(magnitude[x], __shfl_xor_sync(0xffffffffu, magnitude[x], o));
      }
      const int lp = now.page0 + x * 8 + r;
      const int page = __shfl_sync(0xffffffffu, now.my_page, x * 8 + r);
      const bool known = page >= 0;
      // A sum that is not finite: because a bound is not, then the score is +infinity and needs no second look (looked at as
      // one that 64 bits have to decide, it would take all other pages with it), or because fp32 does not hold it.
      if (__any_sync(0xffffffffu, magnitude[x] > FLT_MAX)) {
        const B* bound = reinterpret_cast<const B*>(a.kv.bounds) + ((int64_t)max(page, 0) * heads + head) * 2 * d;
        uint32_t odd = 0;
#pragma unroll 1
        for (int ch = c * 8; ch < 2 * d; ch += 32) {
          const uint4 v = load_once(bound + ch);
          odd |= not_finite2<B>(v.x) | not_finite2<B>(v.y) | not_finite2<B>(v.z) | not_finite2<B>(v.w);
        }
        odd |= __shfl_xor_sync(0xffffffffu, odd, 1);
        odd |= __shfl_xor_sync(0xffffffffu, odd, 2);
        if (odd) {
          best[x] = INFINITY;
          magnitude[x] = 0.0f;
        }
      }
      // a page outside the pool comes last (-infinity): the attention would leave it out
      if (c == 0 && lp < now.n)
        *reinterpret_cast<float2*>(scores + (now.seq * heads + head) * a.table.width + lp) =
            known ? make_float2(magnitude[x] <= FLT_MAX ? best[x] : 0.0f, magnitude[x]) : make_float2(-INFINITY, 0.0f);
    }
  }
}

// Exact key of a page (`lower`: its bounds) for one query, by one warp.
template <typename T, typename B>
__device__ __noinline__ unsigned long long exact_key(const T* q, const B* lower, int d) {
  double s = 0.0;
#pragma unroll 2
  for (int i = (threadIdx.x & 31) * 2; i < d; i += 64) {
    const float2 x = to_float2<T>(*reinterpret_cast<const uint32_t*>(q + i));
    const float2 l = to_float2<B>(*reinterpret_cast<const uint32_t*>(lower + i)), h = to_float2<B>(*reinterpret_cast<const uint32_t*>(lower + d + i));
    // (as two terms, one of them 0 times a bound: NaN when that is not finite)
    s = fma((double)fmaxf(x.x, 0.0f), (double)h.x, fma((double)fminf(x.x, 0.0f), (double)l.x, s));
    s = fma((double)fmaxf(x.y, 0.0f), (double)h.y, fma((double)fminf(x.y, 0.0f), (double)l.y, s));
    if (x.x != x.x || x.y != x.y) s = INFINITY;
  }
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return score_key(s);
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

constexpr int BORDER = 256;                                  // pages between that are ranked in shared memory
constexpr int FEW = 32;                                      // keys that a warp ranks (and as many warps at most)

struct SelectShared {
  int hist[256];
  unsigned long long low[32], high[32];
  int digit, need, count;
  int sums[2][32];
  float most[32];
  int few_count, border_count;
  uint32_t few[FEW], kth;
  int border[BORDER], border_page[BORDER];
  uint32_t taken[256];
  unsigned long long border_key[BORDER];
};

// What a radix selection found: the `need` first of the `among` keys that match the prefix, and all above it, are taken.
template <typename K>
struct Chosen {
  K prefix;
  int shift, need, among;
  __device__ bool matches(K k) const { return shift == (int)sizeof(K) * 8 || k >> shift == prefix; }
  __device__ bool above(K k) const { return shift < (int)sizeof(K) * 8 && k >> shift > prefix; }
};

template <typename K>
__device__ __forceinline__ K warp_min(K x) {
  if constexpr (sizeof(K) == 4) {
    return __reduce_min_sync(0xffffffffu, x);
  } else {
    for (int o = 16; o > 0; o >>= 1) {
      const K y = __shfl_xor_sync(0xffffffffu, x, o);
      x = y < x ? y : x;
    }
    return x;
  }
}
template <typename K>
__device__ __forceinline__ K warp_max(K x) {
  return ~warp_min<K>(~x);
}

// The `need` largest of `among` keys, from the first bit in which they differ: 8 bits at a time the keys that share the
// threshold's leading bits are counted by their next digit, until all of them are wanted, no more than `few` are left or all
// bits are known.
// key(j) is the thread's j-th key, valid(j) whether it has one; ROWS rounds, or `rounds` where that is 0.
template <typename K, int ROWS, class Key, class Valid>
__device__ Chosen<K> radix_select(SelectShared& sm, int rounds, int need, int among, int few, Key key, Valid valid) {
  constexpr int BITS = (int)sizeof(K) * 8;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
  const int end = ROWS > 0 ? ROWS : rounds;
  K low = ~(K)0, high = 0;
#pragma unroll
  for (int j = 0; j < end; ++j)
    if (valid(j)) {
      const K k = key(j);
      low = k < low ? k : low;
      high = k > high ? k : high;
    }
  low = warp_min<K>(low);
  high = warp_max<K>(high);
  __syncthreads();
  if (lane == 0) {
    sm.low[warp] = low;
    sm.high[warp] = high;
  }
  __syncthreads();
  low = warp_min<K>(lane < warps ? (K)sm.low[lane] : ~(K)0);
  high = warp_max<K>(lane < warps ? (K)sm.high[lane] : (K)0);
  Chosen<K> c;
  c.need = need;
  c.among = among;
  c.shift = low >= high ? 0 : 64 - __clzll((unsigned long long)low ^ (unsigned long long)high);   // bits that are not known
  c.prefix = c.shift == BITS ? 0 : high >> c.shift;
  while (c.need > 0 && c.need < c.among && c.among > few && c.shift > 0) {
    const int bits = min(8, c.shift), next = c.shift - bits;
    for (int i = tid; i < 256; i += threads) sm.hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < end; ++j)
      if (valid(j)) {
        const K k = key(j);
        if (c.matches(k)) atomicAdd(&sm.hist[(int)(k >> next) & ((1 << bits) - 1)], 1);
      }
    __syncthreads();
    if (warp == 0) {                                         // the digit that the need-th largest key has
      int mine[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += mine[i] = sm.hist[255 - (lane * 8 + i)];
      int before = sum;
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += y;
      }
      before -= sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (before < c.need && c.need <= before + mine[i]) {
          sm.digit = 255 - (lane * 8 + i);
          sm.need = c.need - before;
          sm.count = mine[i];
        }
        before += mine[i];
      }
    }
    __syncthreads();
    c.prefix = (c.shift == BITS ? 0 : c.prefix << bits) | (K)sm.digit;
    c.need = sm.need;
    c.among = sm.count;                                      // (written again two barriers from here)
    c.shift = next;
  }
  return c;
}

// Sums of two numbers over the block, for every thread (once a kernel: no barrier before).
__device__ __forceinline__ int2 block_sums(SelectShared& sm, int x, int y) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  x = __reduce_add_sync(0xffffffffu, x);
  y = __reduce_add_sync(0xffffffffu, y);
  if (lane == 0) {
    sm.sums[0][warp] = x;
    sm.sums[1][warp] = y;
  }
  __syncthreads();
  return make_int2(__reduce_add_sync(0xffffffffu, lane < warps ? sm.sums[0][lane] : 0),
                   __reduce_add_sync(0xffffffffu, lane < warps ? sm.sums[1][lane] : 0));
}

// Writes the taken pages in ascending order: those with take(j), and the first `need` of the `among` with equal(j).  R rounds
// at a time; hist holds the counts of (round, warp): 8 * 32 at most.
template <int R, class Take, class Equal>
__device__ void write_pages(SelectShared& sm, int rounds, int need, int among, Take take_of, Equal equal_of, int32_t* out) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
  int taken_before = 0, equal_before = 0;
  for (int j0 = 0; j0 < rounds; j0 += R) {
    unsigned equal = 0, take = 0;                            // one bit a round
#pragma unroll
    for (int x = 0; x < R; ++x) {
      equal |= (unsigned)equal_of(j0, x) << x;
      take |= (unsigned)take_of(j0, x) << x;
    }
    if (need < among) {                                      // not all that match: by rank
      __syncthreads();
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const unsigned m = __ballot_sync(0xffffffffu, equal >> x & 1);
        if (lane == 0) sm.hist[x * warps + warp] = __popc(m);
      }
      __syncthreads();
      if (warp == 0) {
        const int total = scan256(sm.hist, R * warps);
        if (lane == 0) sm.count = total;
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const unsigned m = __ballot_sync(0xffffffffu, equal >> x & 1);
        if ((equal >> x & 1) && equal_before + sm.hist[x * warps + warp] + __popc(m & ((1u << lane) - 1)) < need) take |= 1u << x;
      }
      equal_before += sm.count;
    } else {
      take |= equal;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < R; ++x) {
      const unsigned m = __ballot_sync(0xffffffffu, take >> x & 1);
      if (lane == 0) sm.hist[x * warps + warp] = __popc(m);
    }
    __syncthreads();
    if (warp == 0) {
      const int total = scan256(sm.hist, R * warps);
      if (lane == 0) sm.count = total;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < R; ++x) {
      const unsigned m = __ballot_sync(0xffffffffu, take >> x & 1);
      if (take >> x & 1) out[taken_before + sm.hist[x * warps + warp] + __popc(m & ((1u << lane) - 1))] = (j0 + x) * threads + tid;
    }
    taken_before += sm.count;
    __syncthreads();
  }
}

// One block per (sequence, key head).  A thread holds every blockDim-th score, up to ROWS of them (ROWS is 4 or 8, or 0 for
// more pages than that: then they are read again for every pass).  A chain of latencies: of barriers, and of instructions that
// come for the first time, so few of them count (scores and selection of 64 of 2047 pages in a captured graph: 12.7 us with
// all bits of the k-th found by counting, lengths before scores, three cases in every comparison and 8 scores a thread; 9.6 us
// as it is).
template <typename T, typename B, int ROWS>
__global__ void __launch_bounds__(1024) select_kernel(const wush_kv_select_args a, int group, Score* scores) {
  __shared__ SelectShared sm;
  // (no early launch of what follows: an attention that waits on the SMs slowed this kernel down by 1.5 us)
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
  const int64_t item = blockIdx.x;
  Score* mine = scores + item * a.table.width;
  auto page_of = [&](int j) { return j * threads + tid; };
  auto load = [&](int j) { return *reinterpret_cast<const float2*>(mine + page_of(j)); };
  float2 early[ROWS > 0 ? ROWS : 1];                         // (before the length is known: what lies behind it is not used)
  if (ROWS > 0)
#pragma unroll
    for (int j = 0; j < ROWS; ++j) early[ROWS > 0 ? j : 0] = *reinterpret_cast<const float2*>(mine + min((int64_t)page_of(j), a.table.width - 1));
  const int len = (int)max((int64_t)0, min((int64_t)a.seq_lens[item / a.kv.heads], a.table.width * a.kv.page_size));
  const int n = pages_of_length(len, a.kv.page_size), top = a.top;
  int32_t* out = a.pages + item * top;
  const int count = min(n, top);
  if (tid == 0) a.counts[item] = count;
  for (int i = count + tid; i < top; i += threads) out[i] = -1;
  if (n <= top) {
    for (int i = tid; i < n; i += threads) out[i] = i;
    return;
  }
  const int begin = a.sink, end = n - a.recent, want = top - a.sink - a.recent;   // pages that compete
  constexpr int R = ROWS > 0 ? ROWS : 8;
  const int rounds = ROWS > 0 ? ROWS : (n + threads - 1) / threads;
  auto competes = [&](int j) { return page_of(j) >= begin && page_of(j) < end; };
  auto forced = [&](int j) { return page_of(j) < n && !competes(j); };
  uint32_t held[ROWS > 0 ? ROWS : 1];
  float magnitude = 0.0f;
#pragma unroll
  for (int j = 0; j < (ROWS > 0 ? ROWS : rounds); ++j)
    if (competes(j)) {
      const float2 s = ROWS > 0 ? early[ROWS > 0 ? j : 0] : load(j);
      if (ROWS > 0) held[ROWS > 0 ? j : 0] = float_key(s.x);
      magnitude = fmaxf(magnitude, s.y);
    }
  auto key_of = [&](int j) { return ROWS > 0 ? held[ROWS > 0 ? j : 0] : float_key(load(j).x); };
  if (want == 0) {
    for (int i = tid; i < top; i += threads) out[i] = i < begin ? i : n - top + i;
    return;
  }
  if (tid == 0) sm.few_count = sm.border_count = 0;
  const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(magnitude));       // (not negative: ordered as they are)
  if (lane == 0) sm.most[warp] = __uint_as_float(most);
  const Chosen<uint32_t> c = radix_select<uint32_t, ROWS>(sm, rounds, want, end - begin, FEW, key_of, competes);   // (with barriers)
  magnitude = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? __float_as_uint(sm.most[lane]) : 0u));

  // the k-th largest: ranked among the few that are left, or the smallest of all that match
  uint32_t kth = ~0u;
#pragma unroll
  for (int j = 0; j < (ROWS > 0 ? ROWS : rounds); ++j)
    if (competes(j)) {
      const uint32_t k = key_of(j);
      if (!c.matches(k)) continue;
      if (c.among <= FEW) sm.few[atomicAdd(&sm.few_count, 1)] = k;
      else kth = min(kth, k);
    }
  if (c.among <= FEW) {
    __syncthreads();
    const uint32_t k = lane < c.among ? sm.few[lane] : 0u;
#pragma unroll 1
    for (int i = warp; i < c.among; i += warps) {
      const uint32_t x = sm.few[i];
      const int above = __popc(__ballot_sync(0xffffffffu, lane < c.among && k > x)), upto = __popc(__ballot_sync(0xffffffffu, lane < c.among && k >= x));
      if (lane == 0 && above < c.need && c.need <= upto) sm.kth = x;       // (equal keys: the same from every warp)
    }
    __syncthreads();
    kth = sm.kth;
  } else {
    // (`few`, which nobody reads on this way: the selection's own words may still be read by a warp that is behind)
    kth = __reduce_min_sync(0xffffffffu, kth);
    if (lane == 0) sm.few[warp] = kth;
    __syncthreads();
    kth = __reduce_min_sync(0xffffffffu, lane < warps ? sm.few[lane] : ~0u);
  }
  // (17 + products / 2) * 2^-23 of the magnitude, a sixteenth more for the magnitude's own rounding, and what numbers below the
  // smallest normal one may lose
  const float eps = magnitude * (float)(17 + 2 * ((a.kv.dim + 31) / 32)) * (1.0625f / 8388608.0f) + 1024.0f * FLT_MIN;
  // a magnitude that is not finite leaves everything between; where the k-th is a page outside the pool, all that are in it
  // are above, and where it is one with a bound that is not finite, those are between
  const float center = key_float(kth);
  float bottom = -INFINITY, roof = INFINITY;
  if (eps <= FLT_MAX) {
    bottom = center >= -FLT_MAX ? __fsub_rd(center, 2.0f * eps) : center;
    roof = center >= -FLT_MAX ? __fadd_ru(center, 2.0f * eps) : center;
  }
  auto is_above = [&](float v) { return v > roof; };
  auto is_between = [&](float v) { return v >= bottom && v <= roof; };
  int n_above = 0, n_upto = 0;                               // (and of those above or between)
#pragma unroll
  for (int j = 0; j < (ROWS > 0 ? ROWS : rounds); ++j)
    if (competes(j)) {
      const float v = key_float(key_of(j));
      n_above += v > roof;
      n_upto += v >= bottom;
    }
  const int2 sums = block_sums(sm, n_above, n_upto);
  const int need = want - sums.x, between = sums.y - sums.x;
  const int64_t seq = item / a.kv.heads;
  const int head = (int)(item - seq * a.kv.heads);
  const T* queries = reinterpret_cast<const T*>(a.q.data) + seq * a.q.row + (int64_t)head * group * a.q.head;
  auto exact = [&](int page, int g) {                        // 0 for a page outside the pool
    const B* lower = reinterpret_cast<const B*>(a.kv.bounds) + ((int64_t)max(page, 0) * a.kv.heads + head) * 2 * a.kv.dim;
    const unsigned long long k = exact_key<T, B>(queries + g * a.q.head, lower, a.kv.dim);
    return page < 0 ? 0ull : k;
  };
  const bool all_between = need == between;                  // the usual case: the k-th itself and nothing else
  if (!all_between && between <= BORDER) {
    // score the pages between again and rank them; the verdict is a bit of `taken`, or is left in place of the score
    const int per = min(group, max(1, warps / between));
    if (ROWS > 0)
      for (int i = tid; i < ROWS * warps; i += threads) sm.taken[i] = 0;
    for (int j0 = 0; j0 < rounds; j0 += R) {
      unsigned mine_between = 0;                             // one bit a round
#pragma unroll
      for (int x = 0; x < R; ++x)
        if (competes(j0 + x)) mine_between |= (unsigned)is_between(key_float(key_of(ROWS > 0 ? x : j0 + x))) << x;
#pragma unroll 1
      for (; mine_between != 0; mine_between &= mine_between - 1) {
        const int at = atomicAdd(&sm.border_count, 1), lp = page_of(j0 + __ffs(mine_between) - 1);
        sm.border[at] = lp;
        sm.border_key[at] = 0;
        sm.border_page[at] = lookup_page(a.table, seq, lp, a.kv.num_pages, a.status);
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = warp; i < between * per; i += warps) {      // `per` warps share the queries of a page
      unsigned long long k = 0;
#pragma unroll 1
      for (int g = i % per; g < group; g += per) {
        const unsigned long long x = exact(sm.border_page[i / per], g);
        k = k < x ? x : k;
      }
      if (lane == 0) atomicMax(&sm.border_key[i / per], k);
    }
    __syncthreads();
    for (int i = tid; i < between; i += threads) {
      int better = 0;
#pragma unroll 1
      for (int o = 0; o < between; ++o)
        better += sm.border_key[o] > sm.border_key[i] || (sm.border_key[o] == sm.border_key[i] && sm.border[o] < sm.border[i]);
      const int lp = sm.border[i];
      if (ROWS == 0) mine[lp].value = better < need ? INFINITY : -INFINITY;
      else if (better < need) atomicOr(&sm.taken[lp >> 5], 1u << (lp & 31));
    }
    __threadfence_block();
    __syncthreads();
  }
  if (all_between || between <= BORDER) {
    write_pages<R>(sm, rounds, 0, 0, [&](int j0, int x) {
      const int j = j0 + x;
      if (!competes(j)) return forced(j);
      const float v = key_float(key_of(ROWS > 0 ? x : j));   // (read again, without registers: the verdict already)
      if (v > roof || (all_between && v >= bottom)) return true;
      if (ROWS == 0) return v == INFINITY;
      return !all_between && v >= bottom && (sm.taken[page_of(j) >> 5] >> (tid & 31) & 1);
    }, [](int, int) { return false; }, out);
    return;
  }
  // many between (equal pages, or queries that are not finite): 64-bit keys in place of the scores, and another selection (not
  // fast: 2047 pages whose bounds are all 0, with 8 queries, 0.7 ms)
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(mine);
  for (int i = warp; i < n; i += warps) {
    if (i < begin || i >= end) continue;
    const float v = *(volatile float*)&mine[i].value;
    unsigned long long k = is_above(v) ? ~0ull : 0;
    if (is_between(v)) {
      const int page = lookup_page(a.table, seq, i, a.kv.num_pages, a.status);
      for (int g = 0; g < group; ++g) {
        const unsigned long long x = exact(page, g);
        k = k < x ? x : k;
      }
    }
    __syncwarp();
    if (lane == 0) keys[i] = k;
  }
  __threadfence_block();
  __syncthreads();
  const int all = (n + threads - 1) / threads;
  auto wide_key = [&](int j) { return *(volatile unsigned long long*)&keys[page_of(j)]; };
  const Chosen<unsigned long long> w = radix_select<unsigned long long, 0>(sm, all, want, end - begin, 0, wide_key, competes);
  write_pages<8>(sm, all, w.need, w.among, [&](int j0, int x) { return competes(j0 + x) ? w.above(wide_key(j0 + x)) : forced(j0 + x); },
              [&](int j0, int x) { return competes(j0 + x) && w.matches(wide_key(j0 + x)); }, out);
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
    return (int)cudaLaunchKernelEx(EarlyLaunch((cudaStream_t)p.stream).config(grid, APPEND_THREADS, 0), kern, p, span);
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
    return (int)cudaLaunchKernelEx(EarlyLaunch((cudaStream_t)args->stream).config(dim3(grid), 128, 0), kern, kv, table, args->seq_lens,
                                   args->new_tokens, most, span, args->status);
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
  Score* scores = reinterpret_cast<Score*>(a.workspace);
  const int64_t units = a.table.seqs * a.kv.heads * ((a.table.width + SCORE_PAGES - 1) / SCORE_PAGES);
  const int group = a.q_heads / a.kv.heads;
  EarlyLaunch early((cudaStream_t)a.stream);
  auto go = [&](auto t, auto b) {
    using T = decltype(t);
    using B = decltype(b);
    const int per_sm = a.kv.dim <= 128 ? SCORE_BLOCKS : 2;
    const dim3 grid((unsigned)min((units + SCORE_WARPS - 1) / SCORE_WARPS, (int64_t)sm_count() * per_sm));
    auto kern = a.kv.dim <= 64 ? score_kernel<T, B, 2> : (a.kv.dim <= 128 ? score_kernel<T, B, 4> : score_kernel<T, B, 8>);
    const cudaError_t e = cudaLaunchKernelEx(early.config(grid, SCORE_WARPS * 32, 0), kern, a, group, scores);
    if (e != cudaSuccess) return (int)e;
    // Up to 4 scores a thread in registers, with up to 512 threads as few as 2 (the warps share what is scored again: 64 items
    // of 1024 pages 17.9 us, with 256 threads 19.3), while all blocks are on the SMs together (1024 threads by registers);
    // else 8 (8 a thread: 24.5 us; 512 items of 2048 pages: 4 a thread 105.5, 8 102.5).  Times of scores and selection.
    const int64_t items = a.table.seqs * a.kv.heads;
    auto threads_for = [&](int rows, int from, int most) {
      while (from < most && (int64_t)from * rows < a.table.width) from *= 2;
      return from;
    };
    int threads = threads_for(4, threads_for(2, 128, 512), 1024);
    const bool four = (int64_t)threads * 4 >= a.table.width && items * threads <= (int64_t)sm_count() * 1024;
    if (!four) threads = threads_for(8, 128, 1024);
    const bool eight = (int64_t)threads * 8 >= a.table.width;
    auto select = four ? select_kernel<T, B, 4> : (eight ? select_kernel<T, B, 8> : select_kernel<T, B, 0>);
    return (int)cudaLaunchKernelEx(early.config(dim3((unsigned)items), threads, 0), select, a, group, scores);
  };
  const __nv_bfloat16 bf = {};
  const __half hf = {};
  if (a.type == WUSH_TYPE_BF16) return a.kv.bounds_type == WUSH_TYPE_BF16 ? go(bf, bf) : go(bf, hf);
  return a.kv.bounds_type == WUSH_TYPE_BF16 ? go(hf, bf) : go(hf, hf);
}
