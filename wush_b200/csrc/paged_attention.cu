// Attention of one new token per sequence over a paged key-value cache: out = softmax(scale * q K^T) V.
//
// The kernel reads every key and value once and does G multiply-adds with each (G = query heads that share a key head), so it
// is bound by HBM as long as the products run on the tensor cores and enough loads are in flight.
//
// Products.  All G queries of a key head are worked on together, with the tokens as the rows of m16n8k16 products:
//     S^T [16 tokens x 8 heads] = K [16 tokens x 16 channels] . Q^T,     O^T [16 channels x 8 heads] += V^T . P^T.
// A product does not care in which order its contracted index runs, nor which row is which channel, so a lane's fragment
// of K is a 16-byte piece of a key row and its fragment of V neighbouring channels of four tokens, each one load from shared
// memory, and the queries are loaded in the matching order.  P is turned from the layout of an accumulator into that of an
// operand by movmatrix, as two 16-bit terms: one alone is off by up to 2^-9 (bf16) or 2^-12 (fp16) of a weight, and where
// values cancel no rounding of the result hides that.  8-bit pages are widened to fp16 (exact).  (tcgen05.mma has at least 64
// rows and 8 columns, wants P in memory, and would be idle all the same: the tensor pipe is busy 14 % of the time, 27 % over
// 8-bit pages.)
//
// Copies.  Every warp has a ring of three tiles in shared memory, filled two tiles ahead by bulk tensor copies (16 rows of one
// head of a page are one box), so a warp needs one instruction for 2 KB and no registers for what is in flight.  Measured on
// 64 ragged sequences of up to 4096 tokens (364 MB), each with the work dealt as it was then: fragments straight into registers
// 110 us, per-lane 16-byte copies 90 us, boxes 70 us (now 67: 84 % of the copy bandwidth; one of 500 000 tokens comes at 6.5 TB/s).
//
// Work.  The tokens of all (sequence, key head, chunk of queries) items are cut into units of 4 tiles (one per warp), the
// units of all items are numbered through, and every block of a grid that fills the GPU exactly once takes an equal run
// of them, teams of blocks the same run for neighbouring key heads; lengths are read on the device.  A block that holds a
// whole item writes its result; a part of an item goes to the workspace, and a second kernel joins the parts (every block has
// at most two: its first and its last item).
#include <type_traits>

#include "paged_kv.cuh"
#include "sm100.cuh"

namespace wush {
namespace kv {

constexpr int WARPS = 4;
// Units that an item is worth beyond its tokens (64 ragged sequences up to 4096: 1 81 us, 2 75 us, 4 and 6 70 us).
constexpr int START = 4;
// Smallest number of units a block takes while others idle (a window of 1000 over 19 sequences: 1 13.1 us, 2 14.1 us).
constexpr int MIN_UNITS = 1;
// Items of at most this many units are not split: one launch instead of two (8 sequences of 512 tokens, 8 units: whole 9.3 us,
// split 12.0 us; one of 1024, 16 units: whole 14.3 us, split 10.5 us).  Twice as many where every SM has an item (64 of 1024:
// whole 47 us, split 52 us), but not over selected pages (24 sequences with 128 of 16 tokens: 69 and 64 us).
constexpr int WHOLE_UNITS = 8;

struct AttentionParams {
  wush_kv_pages kv;
  wush_kv_table table;
  wush_heads q, out;
  float* lse;
  const int32_t* seq_lens;
  const int32_t* pages;
  const int32_t* counts;
  float* part_o;                        // [slots][heads of a chunk][DP]
  float* part_ml;                       // [slots][heads of a chunk][2]
  int4* splits;                         // [blocks][2]: the item that goes on in the next block
  int* status;
  float scale;
  int64_t window;
  int q_heads, group, chunks, top;
  int whole;                            // one block per item, no parts
  int team;                             // neighbouring blocks that walk the same tokens of as many key heads
  int64_t entries;                      // sequences, or (sequence, key head) pairs when pages are selected
};

// Tokens of a tile, and resident blocks per SM: by the rings of their warps (three tiles each) in 227 KB of shared memory,
// and by the registers where a key head has more than 8 queries.
__host__ __device__ constexpr int tile_tokens(int dp, int esize) { return dp < 256 && (esize == 1 || dp == 64) ? 32 : 16; }
__host__ __device__ constexpr int blocks_per_sm(int dp, int esize, int nt) {
  const int fit = 18 * 1024 / (2 * tile_tokens(dp, esize) * dp * esize);
  return nt == 2 && fit > 3 ? 3 : fit;
}

// ---- shape of an instantiation -----------------------------------------------------------------------------------------
// T: queries and result; C: pages; DP: channels, rounded up to 64, 128 or 256; NT: tiles of 8 query heads.
template <typename T, typename C, int DP, int NT>
struct Shape {
  static constexpr bool E8 = sizeof(C) == 1;
  // tokens of a warp's tile: 4 KB of keys and as much of values (128 channels)
  static constexpr int TT = tile_tokens(DP, (int)sizeof(C));
  static constexpr int MT = TT / 16;
  static constexpr int KJ = DP * (int)sizeof(C) / 64;       // 16-byte pieces of a key row per lane
  static constexpr int VC = E8 && DP >= 128 ? 16 : 8;       // channels of a lane's piece of a value row
  static constexpr int VB = VC * (int)sizeof(C);            // its bytes: 16, or 8 for short rows of 8-bit values
  static constexpr int VJ = DP / (8 * VC);                  // pieces per lane
  static constexpr int VI = VC / 2;                         // products of 16 channels they make
  // A tile in shared memory: for every 16 tokens the keys, then for every 16 tokens the values; 16 rows of at most 128
  // bytes make a box, the boxes of longer rows follow each other, and the 16-byte pieces of a box are swizzled
  static constexpr int PITCH_B = DP * (int)sizeof(C) < 128 ? DP * (int)sizeof(C) : 128;
  static constexpr int BOXES = DP * (int)sizeof(C) / PITCH_B, BOX = 16 * PITCH_B, GROUP = BOXES * BOX;
  static constexpr int STAGE = 2 * MT * GROUP;
  static constexpr int HEADS = NT * 8;
  static constexpr int UNIT = WARPS * TT;                   // tokens of a unit
  static constexpr int STAGES = 3;                          // tiles of a warp in shared memory or on the way there
  using M = typename std::conditional<E8, __half, T>::type; // operand type of the products
  static constexpr float RISE = 8.0f;                       // exponent that a weight may reach
  // fp16 weights are scaled by 2^7: the largest then are 2^15, and small ones stay normal numbers down to 2^-21
  static constexpr float BIAS = std::is_same<M, __half>::value ? 7.0f : 0.0f;
  static constexpr int BLOCKS = blocks_per_sm(DP, (int)sizeof(C), NT);
  static constexpr int PITCH = DP + 4;                      // floats of a head's row in shared memory
  static constexpr int RING = STAGES * STAGE;               // bytes of a warp
  static_assert(RING >= HEADS * PITCH * 4, "the ring also holds a warp's part of the result");
};

// Tiles of 8 query heads a block works on: two where a key head has more than 8 (16 queries a key head, 4096 tokens: two
// 55.3 us, one and every key read twice 58.7 us), one at 256 channels for the registers.
__host__ __device__ inline int pad_dim(int d) { return d <= 64 ? 64 : (d <= 128 ? 128 : 256); }
__host__ __device__ inline int head_tiles(int dp, int group) { return dp == 256 || group <= 8 ? 1 : 2; }

// ---- instructions ------------------------------------------------------------------------------------------------------
// asynchronous copy of a 16-byte piece into shared memory; zeros when !ok
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// box of 16 rows of one head of one page
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(page), "r"(bar)
      : "memory");
}

// place of a byte of a box: the swizzle exchanges the 16-byte pieces of a line of 128 bytes (64 where rows are that short)
// by the line's number
template <int PITCH_B>
__device__ __forceinline__ constexpr int swizzled(int at) {
  return at ^ ((at >> 3) & (PITCH_B == 128 ? 0x70 : 0x30));
}

// transpose of an 8 x 8 matrix of 16-bit numbers held by the warp (row = lane / 4, two columns per lane)
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

// 2^x to 2 units in the last place; 0 for -infinity
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// ---- numbering of the work ---------------------------------------------------------------------------------------------
// An item is worth START units for looking up its first pages, filling the ring and writing its result, and then one unit
// for each UNIT tokens.  Without START a block whose run held a dozen short sequences finished long after the others.
struct Work {
  int len;                              // tokens of the sequence
  int begin;                            // first position that counts (window); 0 when pages are selected
  int origin;                           // first position that is walked: begin, or the 16 tokens that hold it
  int tokens;                           // tokens to walk: positions, or rows of the selected pages
};

template <bool FAST>
__device__ __forceinline__ Work work_of(const AttentionParams& p, int64_t entry) {
  const int64_t b = p.pages ? entry / p.kv.heads : entry;
  Work w;
  w.len = clamp_length(p.seq_lens[b], p.table.width * p.kv.page_size, p.status);
  w.begin = p.window > 0 && w.len > p.window ? (int)(w.len - p.window) : 0;
  w.origin = FAST ? w.begin & ~15 : w.begin;
  w.tokens = p.pages ? clamp_length(p.counts[entry], p.top, p.status) * p.kv.page_size : w.len - w.origin;
  return w;
}

// an item without tokens has one unit: somebody has to write its zeros
template <bool FAST, int UNIT>
__device__ __forceinline__ int64_t units_of(const AttentionParams& p, int64_t entry) {
  return entry < p.entries ? max(1, (work_of<FAST>(p, entry).tokens + UNIT - 1) / UNIT) : 0;
}

struct Place {
  int64_t entry, base;                  // entry that holds a unit, and the number of its first unit
  int64_t units;                        // units of one item of the entry, without START
};

// Total number of units, by one warp.
template <bool FAST, int UNIT>
__device__ int64_t total_units(const AttentionParams& p, int copies) {
  const int lane = threadIdx.x & 31;
  int64_t sum = 0;
  for (int64_t e = lane; e < p.entries; e += 32) sum += START + units_of<FAST, UNIT>(p, e);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum * copies;
}

// The entry that unit t lies in, by one warp; `copies` items per entry.
template <bool FAST, int UNIT>
__device__ Place locate(const AttentionParams& p, int copies, int64_t t) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int64_t e0 = 0; e0 < p.entries; e0 += 32) {
    const int64_t u = units_of<FAST, UNIT>(p, e0 + lane);
    int64_t sum = e0 + lane < p.entries ? (START + u) * copies : 0;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned beyond = __ballot_sync(0xffffffffu, before + sum > t);
    if (beyond) {
      const int at = __ffs(beyond) - 1;
      const int64_t units = __shfl_sync(0xffffffffu, u, at);
      return {e0 + at, before + __shfl_sync(0xffffffffu, sum, at) - (START + units) * copies, units};
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return {p.entries, before, 1};
}

__device__ __forceinline__ int64_t units_per_block(int64_t total, int64_t blocks) {
  const int64_t per = (total + blocks - 1) / blocks;
  return per < START + MIN_UNITS ? START + MIN_UNITS : per;
}

struct Item {
  int64_t b;
  int hk, first_head, heads;            // key head; first query head and number of query heads of the chunk
};

template <int HEADS>
__device__ __forceinline__ Item item_of(const AttentionParams& p, int64_t entry, int64_t copy) {
  Item it;
  it.b = p.pages ? entry / p.kv.heads : entry;
  it.hk = p.pages ? (int)(entry % p.kv.heads) : (int)(copy / p.chunks);
  const int chunk = p.pages ? (int)copy : (int)(copy % p.chunks);
  it.first_head = it.hk * p.group + chunk * HEADS;
  it.heads = min(HEADS, p.group - chunk * HEADS);
  return it;
}

// ---- the kernel --------------------------------------------------------------------------------------------------------
// FAST: page_size is a multiple of 16, so that 16 consecutive tokens lie in one page: their rows come as boxes of a tensor
// map.  Otherwise the lanes copy them piece by piece, row by row.
template <typename T, typename C, int DP, int NT, bool FAST>
__global__ void __launch_bounds__(WARPS * 32, Shape<T, C, DP, NT>::BLOCKS)
    attention_kernel(const AttentionParams p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
  using S = Shape<T, C, DP, NT>;
  using M = typename S::M;
  constexpr int MT = S::MT, KJ = S::KJ, VJ = S::VJ, VI = S::VI, TT = S::TT, CB = (int)sizeof(C);
  constexpr unsigned FULL = TT == 32 ? 0xffffffffu : 0xffffu;
  // every warp's ring of tiles; between walks it holds the warp's part of the result, [HEADS][PITCH] floats
  extern __shared__ uint8_t smem_raw[];
  __shared__ float sm_m[WARPS * S::HEADS], sm_l[WARPS * S::HEADS];
  __shared__ __align__(8) uint64_t sm_bar[WARPS][S::STAGES];
  __shared__ uint32_t sm_abort;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  uint8_t* smem = smem_raw + ((1024 - (sm100::smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* ring = smem + warp * S::RING;
  const uint32_t ring_at = sm100::smem_u32(ring), bar_at = sm100::smem_u32(sm_bar[warp]);
  const int d = p.kv.dim, page_size = p.kv.page_size;
  const int copies = p.pages ? p.chunks : p.kv.heads * p.chunks;

  if (FAST) {
    if (threadIdx.x == 0) sm_abort = 0;
    if (lane == 0) {
      for (int i = 0; i < S::STAGES; ++i) sm100::mbar_init(bar_at + 8 * i, 1);
      sm100::mbar_init_fence();
    }
    __syncthreads();
  }
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");

  // Row r of a product is token token_row(r) of its 16 and lane 4 r + c reads piece piece_of(r) of a value row: with these
  // orders no two lanes that read together meet in a bank.
  const int token_row = (r >> 1) | (r & 1) << 2;                       // and token_row + 8; operand tokens c, c + 4, c + 8, c + 12
  const int piece = S::PITCH_B == 128 ? token_row : r;
  // byte offsets in a group of 16 tokens; 8 rows and a box further they repeat (short rows: computed apart)
  const int k_lo = swizzled<S::PITCH_B>(token_row * S::PITCH_B + c * 16), k_hi = swizzled<S::PITCH_B>((token_row + 8) * S::PITCH_B + c * 16);
  const int v_0 = swizzled<S::PITCH_B>(c * S::PITCH_B + piece * S::VB), v_4 = swizzled<S::PITCH_B>((c + 4) * S::PITCH_B + piece * S::VB);
  const int v_8 = swizzled<S::PITCH_B>((c + 8) * S::PITCH_B + piece * S::VB), v_12 = swizzled<S::PITCH_B>((c + 12) * S::PITCH_B + piece * S::VB);

  const int teams = p.whole ? copies : copies / p.team, member = p.whole ? 0 : blockIdx.x % p.team;   // teams' items an entry has
  int64_t t, t_end, t_first;
  Place at;
  if (p.whole) {
    const int64_t entry = blockIdx.x / copies;
    at = {entry, 0, units_of<FAST, S::UNIT>(p, entry)};
    t = t_first = (int64_t)(blockIdx.x % copies) * (START + at.units);
    t_end = t + START + at.units;
  } else {
    const int64_t total = total_units<FAST, S::UNIT>(p, teams);
    const int64_t per = units_per_block(total, gridDim.x / p.team);
    t = t_first = (int64_t)(blockIdx.x / p.team) * per;
    t_end = min(total, t + per);
    if (threadIdx.x == 0) p.splits[2 * blockIdx.x].w = 0;
    if (t >= t_end) return;
    at = locate<FAST, S::UNIT>(p, teams, t);
  }

  int stage = 0;                                             // of the ring, for the tile that is worked on next
  uint32_t parity = 0;
  for (int64_t t_next; t < t_end; t = t_next) {
    if (t >= at.base + (START + at.units) * teams) {         // the next entry
      at.base += (START + at.units) * teams;
      at.entry += 1;
      at.units = units_of<FAST, S::UNIT>(p, at.entry);
    }
    const int64_t its_team = (t - at.base) / (START + at.units), copy = p.whole ? its_team : its_team * p.team + member;
    const int64_t within = t - at.base - its_team * (START + at.units);
    t_next = t + min(START + at.units - within, t_end - t);
    const int64_t u0 = max((int64_t)0, within - START), u1 = within + (t_next - t) - START;
    if (u1 <= u0) continue;                                  // only the item's START: the next block has its first tokens
    const Work w = work_of<FAST>(p, at.entry);
    const Item it = item_of<S::HEADS>(p, at.entry, copy);
    const int s1 = (int)min((int64_t)w.tokens, u1 * S::UNIT);

    // -- where the tokens are --------------------------------------------------------------------------------------------
    const int32_t* list = p.pages ? p.pages + at.entry * p.top : nullptr;
    const int32_t* table = p.table.block_table + it.b * p.table.stride;
    constexpr int STEP = S::UNIT;
    const int first = (int)u0 * S::UNIT + warp * TT;         // the warp's tiles are first, first + STEP, ... below s1
    // A lookup goes in levels, each of which loads for the next: walked token -> logical page and row -> physical page.
    struct Row { int page, row, pos; };
    constexpr int NOTHING = INT32_MIN;                       // page of a token that is not there
    auto logical = [&](int v) -> Row {
      if (v >= s1) return {NOTHING, 0, 0};
      const int at_v = v + w.origin, li = at_v / page_size, row = at_v - li * page_size;
      if (!list) return {li, row, at_v};
      const int lp = list[li];
      if (lp < 0 || lp >= p.table.width) {
        report_index(p.status);
        return {NOTHING, 0, 0};
      }
      return {lp, row, lp * page_size + row};
    };
    // (a negative entry becomes -1, so that none of them is NOTHING)
    auto physical = [&](Row x) -> Row { return {x.page >= 0 && x.pos < w.len ? max(table[x.page], -1) : NOTHING, x.row, x.pos}; };
    // the current page (0 where there is none) and row, and the tokens that count: one, or with FAST the 16 from there
    int page = 0, page_row = 0;
    unsigned counts16 = 0;
    auto resolve = [&](Row x) {
      const bool ok = x.page >= 0 && x.page < p.kv.num_pages;
      if (!ok && x.page != NOTHING) report_index(p.status);
      page = ok ? x.page : 0;
      page_row = ok ? x.row : 0;
      const int lo = max(0, w.begin - x.pos), hi = min(16, w.len - x.pos);
      counts16 = !ok ? 0 : (FAST ? (0xffffu >> (16 - hi)) & (0xffffu << lo) : 1);
    };
    // FAST: lane i holds the warp's i-th group of 16 tokens of the current 32, the levels of the next 32 and of those after
    // them are under way.  Else: lane i holds the i-th token of the next tile.
    auto token_of = [&](int i) { return FAST ? first + i / MT * STEP + i % MT * 16 : first + i / TT * STEP + i % TT; };
    const int held = FAST ? lane : lane & (TT - 1), hold = FAST ? 32 : TT;
    Row next = physical(logical(token_of(held))), after = logical(token_of(hold + held));
    auto advance = [&](int i) {                              // make the lookups from i on the current ones
      resolve(next);
      next = physical(after);
      after = logical(token_of(i + 2 * hold + held));
    };

    // the copies of tile i into stage `to` of the ring; returns the tokens that count
    auto fetch = [&](int i, int to) -> unsigned {
      const uint32_t dst = ring_at + to * S::STAGE;
      unsigned mask = 0;
      if constexpr (FAST) {
        // the lanes that hold the tile's groups start their copies, whole boxes: rows that do not count are masked later
        if (i * MT % 32 == 0) advance(i * MT);
        const uint32_t bar = bar_at + 8 * to;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int from = (i * MT + mt) & 31;
          if (lane == from) {
            if (mt == 0) sm100::mbar_arrive_expect_tx(bar, S::STAGE);
#pragma unroll
            for (int x = 0; x < S::BOXES; ++x) {
              tma_load_4d(dst + mt * S::GROUP + x * S::BOX, &k_map, x * (S::PITCH_B / CB), page_row, it.hk, page, bar);
              tma_load_4d(dst + (MT + mt) * S::GROUP + x * S::BOX, &v_map, x * (S::PITCH_B / CB), page_row, it.hk, page, bar);
            }
          }
          mask |= __shfl_sync(0xffffffffu, counts16, from) << (16 * mt);
        }
      } else {
        advance(i * TT);
        mask = __ballot_sync(0xffffffffu, counts16 != 0) & FULL;
        const int64_t k_at = (page * p.kv.k_page + page_row * p.kv.k_row + it.hk * p.kv.k_head) * CB;
        const int64_t v_at = (page * p.kv.v_page + page_row * p.kv.v_row + it.hk * p.kv.v_head) * CB;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int row = half * 8 + r, tok = mt * 16 + row;
            const uint8_t* k = reinterpret_cast<const uint8_t*>(p.kv.k) + __shfl_sync(0xffffffffu, k_at, tok);
            const uint8_t* v = reinterpret_cast<const uint8_t*>(p.kv.v) + __shfl_sync(0xffffffffu, v_at, tok);
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
              const int x = (j * 4 + c) * 16;
              const bool in = x < d * CB, ok = in && (mask >> tok & 1);
              const uint32_t to_box = dst + mt * S::GROUP + x / S::PITCH_B * S::BOX + swizzled<S::PITCH_B>(row * S::PITCH_B + x % S::PITCH_B);
              copy16(to_box, k + (in ? x : 0), ok);
              copy16(to_box + MT * S::GROUP, v + (in ? x : 0), ok);
            }
          }
      }
      return mask;
    };

    // Tiles are fetched STAGES - 1 ahead of the one worked on; every warp has its own ring and barriers.
    unsigned seen[S::STAGES];                                // tokens that count of the tiles in the ring, oldest first
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; ++i) {
      seen[i] = 0;
      if (first + i * STEP < s1) seen[i] = fetch(i, (stage + i) % S::STAGES);
      if (!FAST) copy_commit();
    }

    // -- queries, in the order of the key fragments ----------------------------------------------------------------------
    uint32_t qf[NT][DP / 16][2];
    float factor[NT][2];                                     // logit -> exponent of 2, for the heads 2c and 2c + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + r;
      const T* row = reinterpret_cast<const T*>(p.q.data) + it.b * p.q.row + (int64_t)(it.first_head + h) * p.q.head;
      const float to_exp2 = p.scale * 1.4426950408889634f;
      if (!S::E8) {
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const int ch = (j * 4 + c) * 8;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (h < it.heads && ch < d) v = *reinterpret_cast<const uint4*>(row + ch);
          qf[nt][2 * j][0] = v.x;
          qf[nt][2 * j][1] = v.y;
          qf[nt][2 * j + 1][0] = v.z;
          qf[nt][2 * j + 1][1] = v.w;
        }
        factor[nt][0] = factor[nt][1] = to_exp2;
      } else {
        // fp16 operands: every query is scaled by a power of two that puts its largest element between 2^15 and 2^16, so that
        // nothing overflows, elements keep all their bits down to 2^-29 of it and what they lose below is 2^-40 of it
        float x[KJ][16];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const int ch = (j * 4 + c) * 16;
#pragma unroll
          for (int k = 0; k < 16; ++k) x[j][k] = 0.0f;
          if (h < it.heads && ch < d) {
            load8(row + ch, *reinterpret_cast<float(*)[8]>(&x[j][0]));
            load8(row + ch + 8, *reinterpret_cast<float(*)[8]>(&x[j][8]));
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) top = fmaxf(top, fabsf(x[j][k]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent field of the largest element, kept where both powers are normal numbers; infinities stay infinite
        const int e = min(max((int)(__float_as_uint(top) >> 23), 16), 254);
        const float in = __uint_as_float((uint32_t)(254 + 15 - e) << 23);
        const float up = __uint_as_float((uint32_t)(e - 15) << 23) * to_exp2 * p.kv.k_scale[it.hk];
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
          for (int k = 0; k < 8; ++k) qf[nt][j * 4 + (k >> 1)][k & 1] = pack2<__half>(x[j][2 * k] * in, x[j][2 * k + 1] * in);
        factor[nt][0] = __shfl_sync(0xffffffffu, up, 8 * c);         // lane 4 h holds head h
        factor[nt][1] = __shfl_sync(0xffffffffu, up, 8 * c + 4);
      }
    }

    // -- the walk --------------------------------------------------------------------------------------------------------
    float m[NT][2], l[NT][2], o[NT][VJ][VI][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int j = 0; j < VJ; ++j)
#pragma unroll
        for (int i = 0; i < VI; ++i) o[nt][j][i][0] = o[nt][j][i][1] = o[nt][j][i][2] = o[nt][j][i][3] = 0.0f;
    }
    int ahead = S::STAGES - 1;
    bool gave_up = false;
    for (int base = first; base < s1; base += STEP, ++ahead) {
      __syncwarp();                                          // the stage that is fetched into has been read by every lane
      seen[S::STAGES - 1] = 0;
      if (base + (S::STAGES - 1) * STEP < s1) seen[S::STAGES - 1] = fetch(ahead, stage == 0 ? S::STAGES - 1 : stage - 1);
      if (FAST) {
        const bool came = sm100::mbar_wait(bar_at + 8 * stage, parity >> stage & 1, &sm_abort);
        if (!__all_sync(0xffffffffu, came)) {
          gave_up = true;
          break;
        }
        parity ^= 1u << stage;
      } else {
        copy_commit();
        copy_wait<S::STAGES - 1>();
        __syncwarp();
      }
      const uint8_t* tile = ring + stage * S::STAGE;
      stage = stage + 1 == S::STAGES ? 0 : stage + 1;
      // logits; two sums where a single chain of products would be waited for
      constexpr int CHAINS = MT * NT == 1 ? 2 : 1;
      float s[MT][NT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float part[CHAINS][NT][4];
#pragma unroll
        for (int x = 0; x < CHAINS; ++x)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[x][nt][0] = part[x][nt][1] = part[x][nt][2] = part[x][nt][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          // piece 4 j + c of the rows; pieces 4 to 7 of a line lie in its other half
          const uint8_t* at_k = tile + mt * S::GROUP + (j >> 1) * S::BOX;
          const uint4 k0 = *reinterpret_cast<const uint4*>(at_k + (k_lo ^ (j & 1) << 6));
          const uint4 k1 = *reinterpret_cast<const uint4*>(at_k + (k_hi ^ (j & 1) << 6));
          const uint32_t lo[4] = {k0.x, k0.y, k0.z, k0.w}, hi[4] = {k1.x, k1.y, k1.z, k1.w};
          if constexpr (S::E8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16x4(lo[i], a0, a2);
              e4m3x4_to_f16x4(hi[i], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<M>(part[i % CHAINS][nt], a0, a1, a2, a3, qf[nt][j * 4 + i][0], qf[nt][j * 4 + i][1]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma<M>(part[i % CHAINS][nt], lo[2 * i], hi[2 * i], lo[2 * i + 1], hi[2 * i + 1], qf[nt][2 * j + i][0], qf[nt][2 * j + i][1]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[mt][nt][x] = CHAINS == 2 ? part[0][nt][x] + part[CHAINS - 1][nt][x] : part[0][nt][x];
      }

      // Softmax: weights relative to a reference per head, which is raised to the running maximum only when a logit passes it
      // by more than RISE; weights then stay below 2^RISE, and most tiles need no exchange between lanes.
      bool rises = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[mt][nt][x] *= factor[nt][x & 1];
      if (seen[0] != FULL) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (!(seen[0] >> (mt * 16 + (x >> 1) * 8 + token_row) & 1)) s[mt][nt][x] = -INFINITY;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
          for (int mt = 1; mt < MT; ++mt) x = fmaxf(x, fmaxf(s[mt][nt][e], s[mt][nt][2 + e]));
          rises |= x > m[nt][e] + S::RISE;
        }
      if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
            for (int mt = 1; mt < MT; ++mt) x = fmaxf(x, fmaxf(s[mt][nt][e], s[mt][nt][2 + e]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float top = fmaxf(m[nt][e], x);
            const float keep = top == m[nt][e] ? 1.0f : exp2_fast(m[nt][e] - top);
            l[nt][e] *= keep;
            m[nt][e] = top;
#pragma unroll
            for (int j = 0; j < VJ; ++j)
#pragma unroll
              for (int i = 0; i < VI; ++i) {
                o[nt][j][i][e] *= keep;
                o[nt][j][i][2 + e] *= keep;
              }
          }
      }
      uint32_t ph[MT][NT][2], pl[MT][NT][2];                 // weights as operands: tokens c, c + 4 (+8) of head r
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float base0 = (m[nt][0] == -INFINITY ? 0.0f : m[nt][0]) - S::BIAS;
        const float base1 = (m[nt][1] == -INFINITY ? 0.0f : m[nt][1]) - S::BIAS;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float p0 = exp2_fast(s[mt][nt][half * 2] - base0), p1 = exp2_fast(s[mt][nt][half * 2 + 1] - base1);
            l[nt][0] += p0;
            l[nt][1] += p1;
            const uint32_t hi = pack2<M>(p0, p1);
            ph[mt][nt][half] = transpose8(hi);
            const float2 back = to_float2<M>(hi);
            pl[mt][nt][half] = transpose8(pack2<M>(p0 - back.x, p1 - back.y));
          }
      }

      // values
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < VJ; ++j) {
          uint32_t w[4][4];                                  // the pieces of tokens c, c + 4, c + 8, c + 12
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint8_t* at_v = tile + (MT + mt) * S::GROUP + j * S::BOX + (x == 0 ? v_0 : (x == 1 ? v_4 : (x == 2 ? v_8 : v_12)));
            if constexpr (S::VB == 8) {
              const uint2 v = *reinterpret_cast<const uint2*>(at_v);
              w[x][0] = v.x;
              w[x][1] = v.y;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(at_v);
              w[x][0] = v.x;
              w[x][1] = v.y;
              w[x][2] = v.z;
              w[x][3] = v.w;
            }
            // values of tokens that do not count must not meet their zero weights as NaN
            if (FAST && seen[0] != FULL && !(seen[0] >> (mt * 16 + c + 4 * x) & 1)) w[x][0] = w[x][1] = w[x][2] = w[x][3] = 0;
          }
#pragma unroll
          for (int i = 0; i < VI; ++i) {
            uint32_t a0, a1, a2, a3;                         // channels 2i and 2i + 1 of the lane's piece
            if constexpr (S::E8) {
              const uint32_t sel = i & 1 ? 0x7362 : 0x5140;  // bytes of two tokens side by side
              const uint32_t x = __byte_perm(w[0][i >> 1], w[1][i >> 1], sel), y = __byte_perm(w[2][i >> 1], w[3][i >> 1], sel);
              e4m3x4_to_f16x4(x, a0, a1);
              e4m3x4_to_f16x4(y, a2, a3);
            } else {
              a0 = __byte_perm(w[0][i], w[1][i], 0x5410);
              a1 = __byte_perm(w[0][i], w[1][i], 0x7632);
              a2 = __byte_perm(w[2][i], w[3][i], 0x5410);
              a3 = __byte_perm(w[2][i], w[3][i], 0x7632);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma<M>(o[nt][j][i], a0, a1, a2, a3, ph[mt][nt][0], ph[mt][nt][1]);
              mma<M>(o[nt][j][i], a0, a1, a2, a3, pl[mt][nt][0], pl[mt][nt][1]);
            }
          }
        }
#pragma unroll
      for (int i = 0; i < S::STAGES - 1; ++i) seen[i] = seen[i + 1];
    }

    // -- join the warps --------------------------------------------------------------------------------------------------
    if (!FAST) copy_wait<0>();
    if (FAST && gave_up) {                                   // the copies in flight have to land before the block ends
      for (int i = 0; i < S::STAGES; ++i)
        for (int k = 0; k < (1 << 16) && !sm100::mbar_try_wait(bar_at + 8 * i, parity >> i & 1); ++k) __nanosleep(64);
    }
    __syncwarp();                                            // the ring has been read by every lane
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int h = nt * 8 + 2 * c + e;
        if (r == 0) {
          sm_m[warp * S::HEADS + h] = m[nt][e];
          sm_l[warp * S::HEADS + h] = x;
        }
        float* row = reinterpret_cast<float*>(ring) + h * S::PITCH + piece * S::VC;
#pragma unroll
        for (int j = 0; j < VJ; ++j)
#pragma unroll
          for (int i = 0; i < VI; i += 2)
            *reinterpret_cast<float4*>(row + j * 8 * S::VC + 2 * i) =
                make_float4(o[nt][j][i][e], o[nt][j][i][2 + e], o[nt][j][i + 1][e], o[nt][j][i + 1][2 + e]);
      }
    __syncthreads();
    const bool all = u0 == 0 && u1 == at.units;
    // Parts go to slot 0 (the block's first item) or 1 (its last).  The block with an item's first tokens leaves a note for
    // the join: sequence, first query head, key head, number of heads; number of parts and slot of the first one.
    const int64_t slot = 2 * (int64_t)blockIdx.x + (t > t_first ? 1 : 0);
    if (!all && u0 == 0 && threadIdx.x == 0) {
      const int64_t rest = at.units - u1, per = t_end - t_first;
      p.splits[2 * blockIdx.x] = make_int4((int)it.b, it.first_head, it.hk, it.heads);
      p.splits[2 * blockIdx.x + 1] = make_int4((int)(1 + (rest + per - 1) / per), (int)(slot & 1), 0, 0);
    }
    for (int x = threadIdx.x; x < S::HEADS * (DP / 8); x += WARPS * 32) {
      const int h = x / (DP / 8), ch = (x % (DP / 8)) * 8;
      if (h >= it.heads || ch >= d) continue;
      float top = sm_m[h];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) top = fmaxf(top, sm_m[k * S::HEADS + h]);
      float total = 0.0f, y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float mk = sm_m[k * S::HEADS + h];
        const float keep = mk == top ? 1.0f : exp2_fast(mk - top);
        total = fmaf(sm_l[k * S::HEADS + h], keep, total);
        const float* row = reinterpret_cast<const float*>(smem + k * S::RING) + h * S::PITCH + ch;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = fmaf(row[i], keep, y[i]);
      }
      if (all) {
        const float scale = (S::E8 ? p.kv.v_scale[it.hk] : 1.0f) / (total == 0.0f ? 1.0f : total);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= scale;
        store8(reinterpret_cast<T*>(p.out.data) + it.b * p.out.row + (int64_t)(it.first_head + h) * p.out.head + ch, y);
        if (ch == 0 && p.lse)
          p.lse[it.b * p.q_heads + it.first_head + h] =
              total == 0.0f ? -INFINITY : (top - S::BIAS + log2f(total)) * 0.6931471805599453f;
      } else {
        float* row = p.part_o + (slot * S::HEADS + h) * DP + ch;
        *reinterpret_cast<float4*>(row) = make_float4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<float4*>(row + 4) = make_float4(y[4], y[5], y[6], y[7]);
        if (ch == 0) {
          p.part_ml[(slot * S::HEADS + h) * 2] = top;
          p.part_ml[(slot * S::HEADS + h) * 2 + 1] = total;
        }
      }
    }
    if (FAST) asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");   // ... and before copies into it by the other proxy
    __syncthreads();                                         // the rings are free again
    if (FAST && sm_abort) {                                  // a copy never came: what was written is invalid
      if (threadIdx.x == 0 && p.status) atomicExch(p.status, 1);
      return;
    }
  }
}

// ---- join of the parts -------------------------------------------------------------------------------------------------
// Block (k, h) joins the parts of the item that block k of the attention left unfinished, for query head h of its chunk: the
// first part is block k's, the others are in slot 0 of the same member of the teams after it.  32 parts at a time, eight a
// warp, all loaded before the first is used: the kernel is a chain of latencies (note, parts, result).
constexpr int JOIN_WARPS = 4, JOIN_ROWS = 32 / JOIN_WARPS;
template <typename T, typename C, int DP, int NT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const AttentionParams p) {
  using S = Shape<T, C, DP, NT>;
  constexpr int E = DP / 64;                                 // pairs of channels of a lane
  __shared__ float2 sm_o[JOIN_WARPS][DP / 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = blockIdx.y;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");      // (every block: none may end before the parts are there)
  const int4 item = p.splits[2 * blockIdx.x], more = p.splits[2 * blockIdx.x + 1];
  if (h >= item.w) return;
  const int parts = more.x;
  auto slot_of = [&](int i) { return (2 * ((int64_t)blockIdx.x + i * p.team) + (i == 0 ? more.y : 0)) * S::HEADS + h; };
  float top = -INFINITY, total = 0.0f;
  float2 o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = make_float2(0.0f, 0.0f);
  for (int base = 0; base < parts; base += 32) {
    float2 row[JOIN_ROWS][E];
#pragma unroll
    for (int x = 0; x < JOIN_ROWS; ++x) {
      const int i = base + warp + x * JOIN_WARPS;
      if (i >= parts) break;
      const float2* from = reinterpret_cast<const float2*>(p.part_o + slot_of(i) * DP) + lane;
#pragma unroll
      for (int j = 0; j < E; ++j) row[x][j] = from[j * 32];
    }
    const bool mine = base + lane < parts;
    const float2 ml = mine ? *reinterpret_cast<const float2*>(p.part_ml + slot_of(base + lane) * 2) : make_float2(-INFINITY, 0.0f);
    float now = ml.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, x));
    now = fmaxf(now, top);
    const float keep = top == now ? 1.0f : exp2_fast(top - now);
    const float weight = !mine ? 0.0f : (ml.x == now ? 1.0f : exp2_fast(ml.x - now));
    top = now;
    float sum = mine ? ml.y * weight : 0.0f;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    total = fmaf(total, keep, sum);
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = make_float2(o[j].x * keep, o[j].y * keep);
#pragma unroll
    for (int x = 0; x < JOIN_ROWS; ++x) {
      const int i = warp + x * JOIN_WARPS;
      if (base + i >= parts) break;
      const float w = __shfl_sync(0xffffffffu, weight, i);
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = make_float2(fmaf(row[x][j].x, w, o[j].x), fmaf(row[x][j].y, w, o[j].y));
    }
  }
#pragma unroll
  for (int j = 0; j < E; ++j) sm_o[warp][j * 32 + lane] = o[j];
  __syncthreads();
  const float scale = (S::E8 ? p.kv.v_scale[item.z] : 1.0f) / (total == 0.0f ? 1.0f : total);
  for (int ch = threadIdx.x * 2; ch < p.kv.dim; ch += JOIN_WARPS * 64) {
    float2 y = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < JOIN_WARPS; ++w) y = make_float2(y.x + sm_o[w][ch / 2].x, y.y + sm_o[w][ch / 2].y);
    T* out = reinterpret_cast<T*>(p.out.data) + item.x * p.out.row + (int64_t)(item.y + h) * p.out.head + ch;
    *reinterpret_cast<uint32_t*>(out) = pack2<T>(y.x * scale, y.y * scale);
  }
  if (threadIdx.x == 0 && p.lse)
    p.lse[(int64_t)item.x * p.q_heads + item.y + h] = total == 0.0f ? -INFINITY : (top - S::BIAS + log2f(total)) * 0.6931471805599453f;
}

// Blocks of the persistent grid (also the number of pairs of workspace slots).
inline int grid_blocks(int dp, int esize, int nt) { return sm_count() * blocks_per_sm(dp, esize, nt); }

template <typename T, typename C, int DP, int NT, bool FAST>
static int launch(AttentionParams p, const CUtensorMap& k_map, const CUtensorMap& v_map, int64_t most_tokens, cudaStream_t stream) {
  using S = Shape<T, C, DP, NT>;
  constexpr int smem = WARPS * S::RING + 1024;
  auto kern = attention_kernel<T, C, DP, NT, FAST>;
  static PerDevice opted;
  if (const int rc = opt_in_smem(opted, kern, smem)) return rc;
  const int64_t items = p.entries * (p.pages ? p.chunks : p.kv.heads * p.chunks);
  const int64_t most_units = (most_tokens + S::UNIT - 1) / S::UNIT;
  p.whole = most_units <= (items >= sm_count() && !p.pages ? 2 * WHOLE_UNITS : WHOLE_UNITS);
  // Teams of up to 8 neighbouring key heads: their rows lie next to each other in token-major pages, and read together they
  // come faster (one sequence of 131071 in E4M3: 53 us, each head by itself 58 us).  Selected pages differ from head to head.
  p.team = 1;
  if (!p.pages && !p.whole)
    for (int g = 2; g <= 8; ++g)
      if (p.kv.heads * p.chunks % g == 0) p.team = g;
  const int64_t most_blocks = (items * most_units + MIN_UNITS - 1) / MIN_UNITS;
  int blocks = p.whole ? (int)items : (int)min((int64_t)grid_blocks(DP, (int)sizeof(C), NT), most_blocks);
  blocks -= blocks % p.team;                                 // (not 0: there are as many items as a team has members)
  // both launches overlap the end of the kernel before them, for which they wait
  EarlyLaunch early(stream);
  const cudaError_t e = cudaLaunchKernelEx(early.config(dim3(blocks), WARPS * 32, smem), kern, p, k_map, v_map);
  if (e != cudaSuccess || p.whole || blocks == p.team) return (int)e;
  return (int)cudaLaunchKernelEx(early.config(dim3(blocks - p.team, min(S::HEADS, p.group)), JOIN_WARPS * 32, 0), join_kernel<T, C, DP, NT>, p);
}

// Tensor map over a pool: boxes of 16 rows of at most 128 bytes of one head of one page.  (Lines are promoted to 128 bytes in
// the L2 and not to 256: 8-bit rows of 128 bytes with other heads' rows between them then took 70 us instead of 61.)
inline bool make_pool_map(CUtensorMap* map, const wush_kv_pages& kv, void* base, int64_t page, int64_t row, int64_t head, int box) {
  EncodeTiledFn encode = tensor_map_encoder();
  if (!encode) return false;
  const cuuint64_t e = element_bytes(kv.type);
  const cuuint64_t dims[4] = {(cuuint64_t)kv.dim, (cuuint64_t)kv.page_size, (cuuint64_t)kv.heads, (cuuint64_t)kv.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)row * e, (cuuint64_t)head * e, (cuuint64_t)page * e};
  const cuuint32_t boxes[4] = {(cuuint32_t)(box / e), 16, 1, 1}, steps[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle swizzle = box == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  return encode(map, e == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, boxes, steps,
                CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes where pages are made of whole groups of 16 tokens and a tensor map can describe the strides, rows piece by piece
// otherwise (64 sequences of 1024: boxes 52.1 us, pieces 54.5 us; 32 ragged ones 16.4 and 18.7 us).
template <typename T, typename C, int DP, int NT>
static int by_page(const AttentionParams& p, int64_t most_tokens, cudaStream_t stream) {
  CUtensorMap k_map{}, v_map{};
  constexpr int box = Shape<T, C, DP, NT>::PITCH_B;
  if (p.kv.page_size % 16 == 0 && make_pool_map(&k_map, p.kv, p.kv.k, p.kv.k_page, p.kv.k_row, p.kv.k_head, box) &&
      make_pool_map(&v_map, p.kv, p.kv.v, p.kv.v_page, p.kv.v_row, p.kv.v_head, box))
    return launch<T, C, DP, NT, true>(p, k_map, v_map, most_tokens, stream);
  return launch<T, C, DP, NT, false>(p, k_map, v_map, most_tokens, stream);
}

template <typename T, typename C>
static int dispatch(const AttentionParams& p, int64_t most_tokens, cudaStream_t stream) {
  const int dp = pad_dim(p.kv.dim), nt = head_tiles(dp, p.group);
  if (dp == 64) return nt == 1 ? by_page<T, C, 64, 1>(p, most_tokens, stream) : by_page<T, C, 64, 2>(p, most_tokens, stream);
  if (dp == 128) return nt == 1 ? by_page<T, C, 128, 1>(p, most_tokens, stream) : by_page<T, C, 128, 2>(p, most_tokens, stream);
  return by_page<T, C, 256, 1>(p, most_tokens, stream);
}

}  // namespace kv
}  // namespace wush

using namespace wush;
using namespace wush::kv;

extern "C" size_t wush_kv_attention_workspace_bytes(const wush_kv_pages* kv, int q_heads) {
  if (!kv || kv->heads <= 0 || q_heads <= 0 || kv->dim <= 0 || kv->dim > MAX_DIM || q_heads < kv->heads) return 0;
  const int dp = pad_dim(kv->dim), nt = head_tiles(dp, q_heads / kv->heads);
  return (size_t)2 * grid_blocks(dp, element_bytes(kv->type), nt) * (nt * 8 * (dp + 2) * sizeof(float) + sizeof(int4));
}

extern "C" int wush_kv_attention(const wush_kv_attention_args* args) {
  if (!args) return WUSH_ERR_NULL_POINTER;
  const wush_kv_attention_args& a = *args;
  const wush_kv_pages& kv = a.kv;
  const wush_kv_table& table = a.table;
  int rc = check_pages(&kv, &table, a.type);
  if (rc != 0) return rc;
  if (a.q_heads <= 0 || a.q_heads % kv.heads || a.window < 0) return WUSH_ERR_BAD_SHAPE;
  if ((a.pages == nullptr) != (a.counts == nullptr)) return WUSH_ERR_NULL_POINTER;
  if (a.pages && (a.top <= 0 || (int64_t)a.top * kv.page_size > MAX_TOKENS)) return WUSH_ERR_BAD_SHAPE;
  if (a.pages && a.window != 0) return WUSH_ERR_BAD_FLAG;
  if (table.seqs == 0) return WUSH_OK;
  if ((rc = check_heads(&a.q, 2)) != 0 || (rc = check_heads(&a.out, 2)) != 0) return rc;
  if (!a.seq_lens || !a.workspace) return WUSH_ERR_NULL_POINTER;
  if (!aligned16(a.workspace)) return WUSH_ERR_BAD_ALIGNMENT;
  if (a.workspace_bytes < wush_kv_attention_workspace_bytes(&kv, a.q_heads)) return WUSH_ERR_WORKSPACE_TOO_SMALL;
  if (table.seqs * a.q_heads > INT32_MAX) return WUSH_ERR_TOO_LARGE;
  if ((rc = require_sm100()) != 0) return rc;
  AttentionParams p{};
  p.kv = kv;
  p.table = table;
  p.q = a.q;
  p.out = a.out;
  p.lse = a.lse;
  p.seq_lens = a.seq_lens;
  p.pages = a.pages;
  p.counts = a.counts;
  p.status = a.status;
  p.scale = a.scale;
  p.window = a.window;
  p.q_heads = a.q_heads;
  p.group = a.q_heads / kv.heads;
  p.top = a.top;
  const int dp = pad_dim(kv.dim), nt = head_tiles(dp, p.group), heads = nt * 8;
  p.chunks = (p.group + heads - 1) / heads;
  p.entries = a.pages ? table.seqs * kv.heads : table.seqs;
  p.part_o = reinterpret_cast<float*>(a.workspace);
  const size_t slots = (size_t)2 * grid_blocks(dp, element_bytes(kv.type), nt);
  p.part_ml = p.part_o + slots * heads * dp;
  p.splits = reinterpret_cast<int4*>(p.part_ml + slots * heads * 2);
  int64_t most = a.pages ? (int64_t)a.top * kv.page_size : table.width * kv.page_size;   // tokens an item can have
  if (a.window > 0 && a.window + 15 < most) most = a.window + 15;                        // (from a multiple of 16 on)
  cudaStream_t s = (cudaStream_t)a.stream;
  if (a.type == WUSH_TYPE_BF16)
    return kv.type == WUSH_TYPE_E4M3 ? dispatch<__nv_bfloat16, __nv_fp8_e4m3>(p, most, s) : dispatch<__nv_bfloat16, __nv_bfloat16>(p, most, s);
  return kv.type == WUSH_TYPE_E4M3 ? dispatch<__half, __nv_fp8_e4m3>(p, most, s) : dispatch<__half, __half>(p, most, s);
}
