// Attention over whole prompts and what a prompt leaves behind (sm_100a):
//   prompt_attention   softmax(scale q K^T) V over packed sequences, causal, query heads in groups; the keys of a sequence may
//                      reach further back than its queries, and every sequence may see a prefix that all of them share
//   prompt_importance  probabilities of each sequence's last queries, summed over the heads
//   prefix_partial     the same attention for single tokens that share a prefix, not yet normalised (decode.cu joins it with the
//                      sequences' own caches)
#include "prompt.cuh"

#include <cudaTypedefs.h>

#include <limits.h>

#include <type_traits>

#include "tensor.cuh"

namespace hqkv {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ int start_of(const int* starts, int s, int total) { return min(max(__ldcg(starts + s), 0), total); }

// ------------------------------------------------------------------------------------------------
// Attention
// ------------------------------------------------------------------------------------------------
// A CTA takes blocks of 256 rows of queries - two tiles of 128 rows, a row being a (token, head of the group) - and walks the tiles of 128
// keys that any of them sees: first the prefix, then the sequence's own.  One pass, with the running maximum and sum of the softmax.
//   warps 0-3, 4-7   softmax of the first and second row tile, a row per thread
//   warps 8, 11      issue the matrix products of the first and second row tile
//   warp 9           looks up the items and requests their tiles of Q, K and V (one thread)
//   warp 10          looks after V tiles that not every row sees (below)
//   warps 12-15      write the output of an item, while the softmax of the next one has begun
// Tensor memory: S of both row tiles (128 columns each, overwritten by P in the type of V) and O of both.
// An item is a block of queries, a head group and a share of the keys.  The grid has a CTA per item, but one CTA per SM does the work: when
// warp 9 begins an item it asks for one that has not been launched yet, looks it up while the others are at work and leaves it in shared
// memory for them.  (Items in a fixed order per CTA: with four prompts of 4 k, some CTAs had 11 % more than their share.)
//   What bounds it.  Of 16 k tokens, 32 heads over 8: tensor cores 75 % of the cycles, special function units 74 %, issue slots 40 %, DRAM
// 3 %.  A tile of keys takes some 3000 cycles, 2048 of them products; a row tile's chain is S (512), softmax (2000: 128 columns at 8 cycles
// of the special function unit a warp, the maximum before, the last stores after), PV (512), and the other row tile's work lies in its
// softmax.  32 heads, us and TFLOP/s a call: 8 k tokens 415 and 1325, all of them seen 785 and 1400, 4 x 4 k 442 and 1245, 8 x 1000 85 and
// 770.  In a long run the power limit decides: 32 k tokens 7.3 ms, 1205 TFLOP/s at 1410 MHz and 990 W (a library product of 8192^3
// under the same limit 1409).
//   Why 256 rows: K and V of a tile are 64 KB from L2 for every CTA, 3.2 KB a cycle for all of them at this rate (3.7 with Q and what is read
// twice); with 128 rows it would be twice that.  Why heads of a group side by side: a block of four heads is 64 tokens long, so its
// last tiles are half as empty and its row tiles as long as each other, and eight tokens of 32 heads fill it.
//   P is rounded to V's type because it is the second product's left operand, which has to have the type of the right one; the sum that
// divides is taken before that, in fp32.
constexpr int TILE = 128;                                // keys per tile, rows per row tile
constexpr int TILE_BYTES = TILE * 128 * 2;               // 64 channels of all its tokens, then the other 64
constexpr int KV_STAGES = 5;
constexpr int PROMPT_THREADS = 512;
constexpr int PROMPT_CTAS = 148;                         // one per SM
constexpr int SHARE_TILES = 4;                           // fewest tiles of keys per share
constexpr unsigned TMEM_COLUMNS = 512;
constexpr float RESCALE_AT = 8.f;                        // powers of two that P may exceed 1 by

struct Place {   // a block of a sequence, and where the sequence's queries and keys are
  int q0, lq, k0, lk, block, rest;   // rest: head group and share
};
// an item of the attention kernel
struct Item {
  Place at;
  bool over;                               // there are no more
  int head0, kv, share, i0;                // i0: the block's first query in its sequence
  bool part, paired;                       // the result is a part of the rows'; one row tile of queries, on which both halves of the CTA work
  int before, seen_first, seen_last;       // tiles of the prefix; own keys that the block's first and last query see
  int lo, hi, hi0, hi1;                    // tiles of keys: [lo, hi), of which the row tiles see those below hi0 and hi1
  // The tiles that row tile a works on: all that it sees, or of a paired item every other one.
  __device__ __forceinline__ int first(int a) const { return lo + (paired ? a : 0); }
  __device__ __forceinline__ int end(int a) const { return a && !paired ? hi1 : hi0; }
  __device__ __forceinline__ int step() const { return paired ? 2 : 1; }
  // Own V tiles that hold keys which some rows of the block do not see.  0 x NaN is NaN in a matrix product, so infinities and NaN
  // of such keys are set to 0, and the rows that do see them add them at the end.
  __device__ __forceinline__ bool partly_seen(int tile) const { return tile >= before && (tile - before + 1) * TILE > seen_first; }
};
constexpr int ITEMS = 4;   // looked up at a time

struct LastCopies {   // a bit per stage: of the last copy into it
  unsigned q_phase, used, to_raw, raw_parity, full_parity;
};
struct PromptShared {
  unsigned long long item_full[ITEMS], item_empty[ITEMS], next_full, q_full, q_empty, kv_full[KV_STAGES], kv_empty[KV_STAGES], v_raw[KV_STAGES];
  unsigned long long s_full[2], p_first[2], p_rest[2], o_full[2], o_empty[2], turn[2], drained[2], ml_full, ml_empty;
  uint32_t tmem;
  LastCopies copies;
  alignas(16) uint4 next;   // answer to the request for an item
  Item items[ITEMS];
  float2 ml[2][TILE];       // (maximum, sum) of the rows
  int stop, odd[ITEMS];     // odd: the last item (by its number) with this place in which warp 10 found infinities or NaN
};
constexpr size_t PROMPT_SMEM = (2 + KV_STAGES) * static_cast<size_t>(TILE_BYTES) + sizeof(PromptShared);
static_assert(PROMPT_SMEM <= 227 * 1024, "one CTA per SM");

static __device__ unsigned g_waits_expired;

// own keys that query i of its sequence sees
__device__ __forceinline__ int keys_seen(const PromptArgs& A, int i, int lq, int lk) {
  return A.causal ? min(max(i + 1 + lk - lq, 0), lk) : lk;
}
__device__ __forceinline__ int tiles_of(int keys) { return (keys + TILE - 1) / TILE; }
// tiles of keys that the last of a sequence's blocks sees, and shares of `per` tiles that the keys of its blocks are divided into
__device__ __forceinline__ int most_tiles(const PromptArgs& A, int lq, int lk) { return tiles_of(A.prefix_len) + tiles_of(keys_seen(A, lq - 1, lq, lk)); }
__device__ __forceinline__ int shares_of(const PromptArgs& A, int per, int lq, int lk) {
  return A.shares == 1 ? 1 : max(1, (most_tiles(A, lq, lk) + per - 1) / per);
}
// Where the sizes of shares follow from the lengths, a block that begins at query i0 and has one row tile, of two that there may be,
// gets half as many tiles more (a tile of its keys takes 1.05 us, that of two row tiles 1.7).
__device__ __forceinline__ int longer(int per) { return per + per / 2; }
__device__ __forceinline__ bool is_longer(const PromptArgs& A, int i0, int lq) {
  return A.by_length && A.block_shift > A.row_shift && i0 + (1 << A.row_shift) >= lq;
}
// Tiles per share, for a warp that holds a sequence per lane (none: lq = 0): the fewest that make an item for every CTA at most, or
// two where that is faster - an item takes as long as its tiles and some three more.  Every lane tries another size.  us with one
// size chosen from the average length for three items per CTA, and with this, in graphs of repeated calls whose K and V the L2 holds
// in part (queries and keys up to, 32 heads over 8): 4 x 96, 16 k 73.4 and 67.3; 8 heads over 2: 5 x 81, 43 k 65.1 and 48.7, 30 x 60,
// 3 k 51 and 32, 12 x 243, 11 k 100 and 75.  Where one item per CTA leaves each a single short one it loses a little: 6 x 31, 11 k, 8 heads over 8
// 41.6 and 43.9, 8 x 50, 31 k, 8 over 2 47.4 and 48.3.
__device__ __forceinline__ int share_size(const PromptArgs& A, int lq, int lk) {
  constexpr unsigned all = 0xffffffffu;
  const int lane = threadIdx.x & 31, round = PROMPT_CTAS / A.groups;   // blocks of a head group that CTAs are there for
  const int tiles = lq > 0 ? most_tiles(A, lq, lk) : 0, blocks = min((lq + (1 << A.block_shift) - 1) >> A.block_shift, PROMPT_CTAS);
  const int shorter = blocks > 0 && is_longer(A, (blocks - 1) << A.block_shift, lq) ? 1 : 0, whole = blocks - shorter;
  const int least = max(SHARE_TILES, __reduce_max_sync(all, (tiles + A.shares - 1) / A.shares));   // (there is room for A.shares)
  const int most = max(least, __reduce_max_sync(all, tiles)), n = __reduce_add_sync(all, blocks);
  // Between work / per and work / (per - 1/3) + n items: a block of one row tile counts as two thirds of one of two, but longer(per) may be
  // 1/2 short of 3/2 per.  So work / (round - n) + 1/3 tiles are enough for one round at most; `high` adds 2 to the truncated quotient
  // for that third and for the quotient's own error (fp32: below 2/3 up to a million tiles, and only the number of items hangs on it: the
  // grid has two rounds).
  const float work = static_cast<float>(__reduce_add_sync(all, static_cast<unsigned>(3 * whole + 2 * shorter) * tiles)) * (1.f / 3.f);
  const int low = max(least, static_cast<int>(__fdividef(work, static_cast<float>(2 * round))));
  const int high = max(low, n < round ? min(most, static_cast<int>(__fdividef(work, static_cast<float>(round - n))) + 2) : most);
  const int per = low + (high - low) * lane / 31;
  const float by = __fdividef(1.f, static_cast<float>(per)), by_longer = __fdividef(1.f, static_cast<float>(longer(per)));
  int items = 0;
  for (int s = 0; s < A.n_seqs; ++s) {
    const float t = static_cast<float>(__shfl_sync(all, tiles, s));
    items += __shfl_sync(all, whole, s) * __float2int_ru(t * by) + __shfl_sync(all, shorter, s) * __float2int_ru(t * by_longer);
  }
  const unsigned in_one = __ballot_sync(all, items <= round) | 1u << 31, in_two = __ballot_sync(all, items <= 2 * round) | 1u << 31;
  const int one = __shfl_sync(all, per, __ffs(in_one) - 1), two = __shfl_sync(all, per, __ffs(in_two) - 1);
  return one <= 2 * two + 3 ? one : two;
}

// Walks the sequences in order, 32 at a time (a lane each), to the one that holds an item.  Items are asked for in rising order, mostly.
template <typename Count>
struct Walk {
  const PromptArgs& A;
  Count count;   // blocks of (lq, lk), items of each and of the last
  int lane, at = 0, q0 = 0, lq = 0, k0 = 0, lk = 0;
  long long before = 0, sum = 0;   // (what starts that are not in order add up to may be anything)
  __device__ __forceinline__ Walk(const PromptArgs& args, Count c) : A(args), count(c), lane(threadIdx.x & 31) {
    look();
    if constexpr (!Count::EVEN) {
      count.choose(lq, lk);
      add_up();
    }
  }
  __device__ __forceinline__ void look() {
    const int s = at + lane;
    q0 = lq = k0 = lk = 0;
    if (A.n_seqs == 0) lq = lane == 0 ? A.total_q : 0;   // a single sequence without keys of its own
    else if (s < A.n_seqs) {
      q0 = start_of(A.q_starts, s, A.total_q), k0 = start_of(A.k_starts, s, A.total_k);
      lq = max(start_of(A.q_starts, s + 1, A.total_q) - q0, 0), lk = max(start_of(A.k_starts, s + 1, A.total_k) - k0, 0);
    }
    add_up();
  }
  __device__ __forceinline__ void add_up() {
    const int blocks = count.blocks(lq, lk);
    sum = static_cast<long long>(blocks) * count.each(lq, lk);
    if constexpr (!Count::EVEN) sum += blocks > 0 ? count.last(lq, lk) - count.each(lq, lk) : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
  }
  // The last block of a sequence, which sees the most keys, comes first.  False: there are not as many items.
  __device__ __forceinline__ bool find(int item, Place& p) {
    unsigned past;
    if (item < before) {
      at = 0, before = 0;
      look();
    }
    while (!(past = __ballot_sync(0xffffffffu, item < before + sum))) {
      before += __shfl_sync(0xffffffffu, sum, 31);
      at += 32;
      if (at >= A.n_seqs) {
        sum = 0;   // (all that follow get the same answer)
        return false;
      }
      look();
    }
    const int from = __ffs(past) - 1;
    auto get = [&](int v) { return __shfl_sync(0xffffffffu, v, from); };
    p.q0 = get(q0), p.lq = get(lq), p.k0 = get(k0), p.lk = get(lk);
    const int each = count.each(p.lq, p.lk), blocks = count.blocks(p.lq, p.lk);
    long long items = static_cast<long long>(blocks) * each;
    if constexpr (!Count::EVEN) items += count.last(p.lq, p.lk) - each;
    const int i = item - static_cast<int>(before + __shfl_sync(0xffffffffu, sum, from) - items), at_block = Count::EVEN ? i / each : min(i / each, blocks - 1);
    p.block = blocks - 1 - at_block, p.rest = i - at_block * each;
    return true;
  }
};

template <bool BF16>
__device__ __forceinline__ bool odd_pair(uint32_t v) {   // an infinity or NaN in either half
  constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
  return (v & e) == e || (v >> 16 & e) == e;
}

template <bool BF16>
__device__ __forceinline__ uint32_t add_zeros(uint32_t sum, uint32_t v) {   // sum + v * 0, both halves
  uint32_t r;
  if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0u), "r"(sum));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(v), "r"(0u), "r"(sum));
  return r;
}

template <bool BY_LENGTH>   // (A.by_length, of which other calls have no instructions to fetch: inside one kernel it cost them 0.4 to 3 us)
struct ItemCount {
  static constexpr bool EVEN = !BY_LENGTH;   // all blocks of a sequence have as many items
  const PromptArgs& A;
  int per;   // tiles per share, where the lengths decide
  __device__ __forceinline__ void choose(int lq, int lk) { per = share_size(A, lq, lk); }
  __device__ __forceinline__ int blocks(int lq, int) const { return (lq + (1 << A.block_shift) - 1) >> A.block_shift; }
  __device__ __forceinline__ int size(int i0, int lq) const { return !BY_LENGTH ? A.per_share : is_longer(A, i0, lq) ? longer(per) : per; }
  __device__ __forceinline__ int each(int lq, int lk) const { return A.groups * shares_of(A, BY_LENGTH ? per : A.per_share, lq, lk); }
  __device__ __forceinline__ int last(int lq, int lk) const {
    return A.groups * shares_of(A, size((blocks(lq, lk) - 1) << A.block_shift, lq), lq, lk);
  }
};
// Items in front of those that are split: with A.split the ones of an unfilled last round, if they are at most half of one.  Each becomes
// two, of a row tile each, which both halves of a CTA work on in less than two thirds of the time.  Items and rounds of
// 32 heads over 8, us without and with: 9 x 300 behind 8192 (2.4 rounds) 324 and 304, 7 x 330 behind 3000 (2.3) 153 and 137,
// 16 x 256 behind 8192 (3.5) 497 and 465, 20 x 200 behind 500 (4.3) 59.8 and 57.5, 24 x 400 behind 1000 (9.1) 186.4 and 186.1, 3 x 400 behind
// 1000 (1.1) 38.2 and 38.4.
template <typename Count>
__device__ __forceinline__ int whole_items(const PromptArgs& A, const Walk<Count>& walk) {
  const int all = static_cast<int>(min(__shfl_sync(0xffffffffu, walk.sum, 31), static_cast<long long>(INT_MAX))), rest = all % PROMPT_CTAS;
  return A.split && rest <= PROMPT_CTAS / 2 ? all - rest : INT_MAX;
}
// false: there are fewer items
template <typename Count>
__device__ __forceinline__ bool look_up(const PromptArgs& A, Walk<Count>& walk, int whole, int item, Item& w) {
  w.over = false;
  const bool split = item >= whole;
  const int second = split ? (item - whole) & 1 : 0;   // of the two row tiles that a split item's block has
  if (split) item = whole + ((item - whole) >> 1);
  if (!walk.find(item, w.at)) return false;
  const int lq = w.at.lq, lk = w.at.lk, half = 1 << A.row_shift, block = 1 << A.block_shift, tokens = split ? half : block;
  // (where keys are shared out, the last block of a sequence comes last: with a single row tile it takes half as long as the others)
  if (A.shares > 1) w.at.block = ((lq + block - 1) >> A.block_shift) - 1 - w.at.block;
  w.share = A.shares == 1 ? 0 : w.at.rest / A.groups;
  const int group = w.at.rest - w.share * A.groups;
  w.head0 = group * A.group;
  w.kv = group / A.groups_per_kv;
  w.i0 = (w.at.block << A.block_shift) + second * half;
  const int per = walk.count.size(w.i0, lq);
  w.part = A.partial || shares_of(A, per, lq, lk) > 1;
  w.paired = tokens == half || w.i0 + half >= lq;
  w.before = tiles_of(A.prefix_len);
  w.seen_first = keys_seen(A, w.i0, lq, lk);
  w.seen_last = keys_seen(A, min(w.i0 + tokens, lq) - 1, lq, lk);
  const int n0 = w.i0 < lq ? w.before + tiles_of(keys_seen(A, min(w.i0 + half, lq) - 1, lq, lk)) : 0;
  const int n1 = !w.paired ? w.before + tiles_of(w.seen_last) : 0;
  w.lo = min(w.share * per, max(n0, n1));
  w.hi = min(w.lo + per, max(n0, n1));
  w.hi0 = min(w.hi, n0), w.hi1 = min(w.hi, n1);
  return true;
}

// Adds the infinities and NaN of keys that only some rows of the block see to query i's output.
template <bool BF16>
__device__ __noinline__ void add_odd_values(const PromptArgs& A, const Item& w, int i, float* part_to, std::conditional_t<BF16, __nv_bfloat16, __half>* to) {
  using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
  const int from = max(w.seen_first, (w.lo - w.before) * TILE), last = min(keys_seen(A, i, w.at.lq, w.at.lk), (w.hi - w.before) * TILE);
#pragma unroll 1
  for (int c = 0; c < 128; ++c) {
    float sum = 0.f;
#pragma unroll 1
    for (int j = from; j < last; ++j) {
      const float x = to_float(static_cast<const T*>(A.v)[(w.at.k0 + j) * A.v_token + w.kv * A.v_head + c]);
      if (!isfinite(x)) sum += x;
    }
    if (sum == 0.f) continue;
    if (w.part) part_to[c] += sum;
    else to[c] = static_cast<T>(to_float(to[c]) + sum);
  }
}

template <bool BF16, bool BY_LENGTH>
__global__ void __launch_bounds__(PROMPT_THREADS, 1) prompt_kernel(const __grid_constant__ PromptArgs A, const __grid_constant__ PromptMaps M) {
  using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
  extern __shared__ __align__(1024) unsigned char tiles[];
  PromptShared& sh = *reinterpret_cast<PromptShared*>(tiles + (2 + KV_STAGES) * TILE_BYTES);
  const uint32_t q_at = smem_u32(tiles), kv_at = q_at + 2 * TILE_BYTES;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int half = 1 << A.row_shift;   // tokens per row tile
  volatile int* const stop = &sh.stop;
  if (warp == 8) tmem_alloc(smem_u32(&sh.tmem), TMEM_COLUMNS);
  if (threadIdx.x == 0) {
    sh.stop = 0;
    for (int& o : sh.odd) o = -1;
    bar_init(smem_u32(&sh.q_full), 1);
    bar_init(smem_u32(&sh.q_empty), 2);
    for (int i = 0; i < KV_STAGES; ++i) {
      bar_init(smem_u32(&sh.kv_full[i]), 1);
      bar_init(smem_u32(&sh.kv_empty[i]), 2);
      bar_init(smem_u32(&sh.v_raw[i]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      bar_init(smem_u32(&sh.s_full[a]), 1);
      bar_init(smem_u32(&sh.p_first[a]), 4);
      bar_init(smem_u32(&sh.p_rest[a]), 4);
      bar_init(smem_u32(&sh.o_full[a]), 1);
      bar_init(smem_u32(&sh.o_empty[a]), 4);
      bar_init(smem_u32(&sh.turn[a]), 1);
      bar_init(smem_u32(&sh.drained[a]), 1);
    }
    for (int i = 0; i < ITEMS; ++i) {
      bar_init(smem_u32(&sh.item_full[i]), 1);
      bar_init(smem_u32(&sh.item_empty[i]), PROMPT_THREADS / 32 - 1);
    }
    bar_init(smem_u32(&sh.next_full), 1);
    bar_init(smem_u32(&sh.ml_full), 8);
    bar_init(smem_u32(&sh.ml_empty), 4);
    bar_init_fence();
  }
  if (warp == 9 && lane < 5) prefetch_map(lane == 0 ? &M.q : lane == 1 ? &M.k : lane == 2 ? &M.v : lane == 3 ? &M.pk : &M.pv);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = uniform(sh.tmem);
  // The next kernel may start (it waits for this one's end before it reads results) now that the tensor memory is there: a CTA of it
  // that shared the SM could take all of it, and would keep it while it waits.
  asm volatile("griddepcontrol.launch_dependents;");
  // (nothing before this reads or writes what an earlier kernel may still be working on)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // item number `round`, for the warps that work on it; null: there are no more, or a wait has run out
  auto item = [&](int round) -> const Item* {
    const int at = round % ITEMS;
    if (!bar_wait(smem_u32(&sh.item_full[at]), round / ITEMS & 1, stop)) return nullptr;
    return sh.items[at].over ? nullptr : &sh.items[at];
  };
  auto done = [&](int round) {
    __syncwarp();
    if (lane == 0) bar_arrive(smem_u32(&sh.item_empty[round % ITEMS]));
  };

  // 512 threads are launched with 128 registers each: 2 x 128 x 184 + 128 x 56 + 128 x 88 = 512 x 128
  if (warp < 8) more_registers<184>();
  else if (warp < 12) fewer_registers<56>();
  else fewer_registers<88>();
  if (warp < 8) {
    // ---- softmax
    const int a = warp >> 2, row = threadIdx.x & 127, token = row >> (7 - A.row_shift);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);   // (32 lanes a warp, in bits 16 and up)
    const uint32_t s_at = lanes + a * TILE, o_at = lanes + 2 * TILE + a * 128;
    const float scale = A.scale_log2;
    unsigned s_phase = 0, ml_phase = 1;
    bool ok = true;
#pragma unroll 1
    for (int round = 0; ok; ++round) {
      const Item* const item_at = item(round);
      if (!item_at) break;
      const Item& w = *item_at;
      const int i = w.i0 + token + (w.paired ? 0 : a * half), first = w.first(a), end = w.end(a), step = w.step(), before = w.before;
      const int seen = i < w.at.lq ? keys_seen(A, i, w.at.lq, w.at.lk) : w.at.lk;
      float ref = -INFINITY, sum = 0.f;
#pragma unroll 1
      for (int tile = first; tile < end; tile += step) {
        if (!(ok = bar_wait(smem_u32(&sh.s_full[a]), s_phase, stop))) break;
        s_phase ^= 1;
        fence_after();
        uint32_t s[TILE];
#pragma unroll
        for (int c = 0; c < TILE; c += 32) tmem_load32(s_at + c, s + c);
        wait_loads(s);
        const int limit = tile < before ? A.prefix_len - tile * TILE : seen - (tile - before) * TILE;
        if (__any_sync(0xffffffffu, limit < TILE)) {
#pragma unroll
          for (int c = 0; c < TILE; ++c)
            if (c >= limit) s[c] = 0xFF800000u;   // -inf
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < TILE; c += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(s[c + 2 * k]), __uint_as_float(s[c + 2 * k + 1]));
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * scale;   // NaN if any S is
        // O and the sum are scaled to the maximum only where it has grown enough to matter: P stays below 2^8
        const bool grown = !(top <= ref + RESCALE_AT);
        if (__any_sync(0xffffffffu, grown)) {
          const float f = grown ? exp2_approx(ref - top) : 1.f;
          if (grown) ref = top;
          sum *= f;
          if (tile > first) {
            // (the product with the tile before, which was issued before this S, is complete)
#pragma unroll 1
            for (int c = 0; c < 128; c += 32) {
              uint32_t o[32];
              tmem_load32(o_at + c, o);
              wait_loads(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_store32(o_at + c, o);
            }
          }
        }
        // (a row of which an S is infinite or NaN is NaN, as inf - inf is)
        const float shift = ref == -INFINITY ? 0.f : fmaf(0.f, ref, -ref);
        const uint64_t scale2 = pair(scale, scale), shift2 = pair(shift, shift);
        uint64_t sums[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < TILE; c += 32) {
          uint32_t p[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float x, y;
            const uint64_t e = pair_fma(pair(__uint_as_float(s[c + 2 * k]), __uint_as_float(s[c + 2 * k + 1])), scale2, shift2);
            unpair(e, x, y);
            x = exp2_approx(x), y = exp2_approx(y);
            sums[k & 1] = pair_add(sums[k & 1], pair(x, y));
            p[k] = narrow2<BF16>(x, y);
            if (c == TILE - 32 && k == 7) {
              wait_stores();
              fence_before();
              __syncwarp();
              if (lane == 0) bar_arrive(smem_u32(&sh.p_first[a]));
            }
          }
          tmem_store16(s_at + c / 2, p);
          if (c == TILE - 32) {
            wait_stores();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(&sh.p_rest[a]));
          }
        }
        float x, y;
        unpair(pair_add(sums[0], sums[1]), x, y);
        sum += x + y;
      }
      if (!ok) break;
      if (!(ok = bar_wait(smem_u32(&sh.ml_empty), ml_phase, stop))) break;
      ml_phase ^= 1;
      sh.ml[a][row] = make_float2(ref, sum);
      __syncwarp();
      if (lane == 0) bar_arrive(smem_u32(&sh.ml_full));
      done(round);
    }
  } else if (warp >= 12) {
    // ---- output: a row of each row tile per thread, or of a paired item the one row that both halves have worked on
    const int row = threadIdx.x & 127, token = row >> (7 - A.row_shift);
    const uint32_t o_at = tmem + (static_cast<uint32_t>(warp & 3) << 21) + 2 * TILE;
    const int64_t rows = static_cast<int64_t>(A.total_q) * A.nh_q;
    unsigned ml_phase = 0, o_phase[2] = {0, 0};
    bool ok = true;
#pragma unroll 1
    for (int round = 0; ok; ++round) {
      const Item* const item_at = item(round);
      if (!item_at) break;
      const Item& w = *item_at;
      if (!(ok = bar_wait(smem_u32(&sh.ml_full), ml_phase, stop))) break;
      ml_phase ^= 1;
      float2 ml[2] = {sh.ml[0][row], sh.ml[1][row]};
      __syncwarp();
      if (lane == 0) bar_arrive(smem_u32(&sh.ml_empty));
      float f[2] = {1.f, 1.f};
      if (w.paired) {
        const float top = fmaxf(ml[0].x, ml[1].x), base = top == -INFINITY ? 0.f : top;
        f[0] = exp2_approx(ml[0].x - base), f[1] = exp2_approx(ml[1].x - base);
        ml[0] = make_float2(top, f[0] * ml[0].y + f[1] * ml[1].y);
      }
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const bool any = w.end(a) > w.first(a);
        if (any) {
          if (!(ok = bar_wait(smem_u32(&sh.o_full[a]), o_phase[a], stop))) break;
          o_phase[a] ^= 1;
          fence_after();
        }
        if (w.paired && a == 0) continue;   // (its output comes with the other half's)
        const int half_a = w.paired ? 0 : a, i = w.i0 + token + half_a * half, head = w.head0 + (row & (A.group - 1));
        const bool live = i < w.at.lq, first = w.paired ? w.end(0) > w.first(0) : any, second = w.paired && any;
        const float ref = ml[half_a].x, sum = ml[half_a].y;
        const int64_t at = static_cast<int64_t>(w.at.q0 + i) * A.nh_q + head;
        if (live && w.part) A.part_ml[w.share * rows + at] = make_float2(ref, sum);
        else if (live) A.lse[static_cast<int64_t>(head) * A.total_q + w.at.q0 + i] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
        if (w.part && !first && !second) continue;   // (nobody reads a part whose sum is 0)
        const float by = w.part ? 1.f : sum == 0.f ? 0.f : 1.f / sum, f0 = f[0] * by, f1 = f[1] * by;
        float* const part_to = A.part_o + (w.share * rows + at) * 128;
        T* const to = static_cast<T*>(A.out) + at * 128;
        const bool part = w.part;
        // (Few instructions, gone through eight times: written out at length this took twice as long, most of it to fetch them.  The next
        // columns are on the way meanwhile: 17 tokens 7.1 / 6.9 us, 2048 41.1 / 40.5.)
        uint32_t o_next[16] = {}, x[16] = {};
        if (first) tmem_load16(o_at + half_a * 128, o_next);
#pragma unroll 1
        for (int c = 0; c < 128; c += 16) {
          uint32_t o[16];
          if (second) tmem_load16(o_at + 128 + c, x);
          wait_loads(o_next);
          wait_loads(x);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(x[k]), f1, __uint_as_float(o_next[k]) * f0));
          if (first && c < 112) tmem_load16(o_at + half_a * 128 + c + 16, o_next);
          if (!live) continue;
          if (part) {
            store_sector(part_to + c, o);
            store_sector(part_to + c + 8, o + 8);
          } else {
            uint32_t h[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) h[m] = narrow2<BF16>(__uint_as_float(o[2 * m]), __uint_as_float(o[2 * m + 1]));
            store_sector(to + c, h);
          }
        }
        fence_before();   // O has been read
        __syncwarp();
        if (lane == 0 && first) bar_arrive(smem_u32(&sh.o_empty[half_a]));
        if (lane == 0 && second) bar_arrive(smem_u32(&sh.o_empty[1]));
        if (live && *const_cast<volatile int*>(&sh.odd[round % ITEMS]) == round) add_odd_values<BF16>(A, w, i, part_to, to);
      }
      done(round);
    }
  } else if (warp == 8 || warp == 11) {
    // ---- matrix products of a row tile.  One warp for both was busy all the time with waiting (some 150 cycles for a barrier that is
    //      complete already) and issuing, and either softmax waited for it: 8 k tokens, all seen: 866 us with one, 832 with two.
    constexpr uint32_t kind_s = mma_kind(BF16, TILE, TILE, false), kind_o = mma_kind(BF16, TILE, 128, true);
    const int a = warp == 8 ? 0 : 1;
    const uint64_t k_operand = operand(kv_at, 16), v_operand = operand(kv_at, TILE_BYTES / 2);
    const uint32_t s_at = tmem + a * TILE, o_at = tmem + 2 * TILE + a * 128;
    const uint32_t s_full = smem_u32(&sh.s_full[a]), p_first = smem_u32(&sh.p_first[a]), p_rest = smem_u32(&sh.p_rest[a]), o_empty = smem_u32(&sh.o_empty[a]);
    uint64_t q_operand = 0;
    int stage = 0;
    unsigned kv_phase = 0, q_phase = 0, p_phase = 0, o_phase = 1, turn = a ^ 1;
    bool ok = true;
    auto wait = [&](uint32_t bar, unsigned parity) { return ok = ok && bar_wait(bar, parity, stop); };
    auto scores = [&] {   // S = Q K^T, 16 channels at a time
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int at = ((c >> 2) * (TILE_BYTES / 2) + (c & 3) * 32) >> 4;
          mma_shared(s_at, q_operand + at, k_operand + (stage * TILE_BYTES >> 4) + at, kind_s, c > 0);
        }
        mma_commit(s_full);
      }
    };
    auto commit = [&](unsigned long long& bar) {
      if (elect_one()) mma_commit(smem_u32(&bar));
    };
    auto advance = [&] {
      if (++stage == KV_STAGES) stage = 0, kv_phase ^= 1;
    };
    auto release = [&](int at, bool mine) {   // a stage, when the products issued so far have read it
      if (!elect_one()) return;
      if (mine) mma_commit(smem_u32(&sh.kv_empty[at]));
      else bar_arrive(smem_u32(&sh.kv_empty[at]));
    };
    // O += P V, 16 keys at a time, the first three quarters as soon as they are there
    auto values = [&](int v_stage, bool add) {
      auto product = [&](int c) {
        mma_tensor(o_at, s_at + c * 8, v_operand + (v_stage * TILE_BYTES >> 4) + c * (2048 >> 4), kind_o, add || c > 0);
      };
      if (!add) {   // (the output of the item before has been read)
        if (!wait(o_empty, o_phase)) return;
        o_phase ^= 1;
      }
      if (!wait(p_first, p_phase)) return;
      fence_after();
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < 6; ++c) product(c);
      }
      if (!wait(p_rest, p_phase)) return;
      p_phase ^= 1;
      fence_after();
      if (elect_one()) {
#pragma unroll
        for (int c = 6; c < 8; ++c) product(c);
      }
    };
#pragma unroll 1
    for (int round = 0; ok; ++round) {
      const Item* const item_at = item(round);
      if (!item_at) break;
      const Item& w = *item_at;
      const int lo = uniform(w.lo), hi = uniform(w.hi), end = uniform(w.end(a)), both = uniform(min(w.hi0, w.hi1));
      const bool paired = uniform(w.paired);
      done(round);
      if (hi <= lo) continue;
      if (!wait(smem_u32(&sh.q_full), q_phase)) break;
      q_phase ^= 1;
      if (paired) {
        // Tile by tile, and those of the other half of the CTA are let go.  Turns as below, given when the next S is under way: a half's
        // product waits for the other's S of a tile ahead, whose stages its own products have left by then.  (One prompt of 2048
        // tokens 42.4 us without, 40.4 with; 1500 27.5, 26.8; 4 x 512 22.0, 22.4; 300 and 1024, decodes behind prefixes the same.)
        q_operand = operand(q_at, 16);
        const int first = lo + a;
        int turns = (hi - lo) / 2;   // products that both halves have
        if (first >= end) commit(sh.q_empty);
#pragma unroll 1
        for (int i = lo; i < hi; ++i) {
          const bool mine = (i - first) % 2 == 0;
          if (!wait(smem_u32(&sh.kv_full[stage]), kv_phase)) break;
          if (mine) {
            scores();
            if (i > first && turns > 0) {
              --turns;
              if (elect_one()) bar_arrive(smem_u32(&sh.turn[a ^ 1]));
            }
            if (i + 2 >= end) commit(sh.q_empty);
          }
          release(stage, mine);
          advance();
          if (!wait(smem_u32(&sh.kv_full[stage]), kv_phase)) break;
          if (mine) {
            if (turns > 0) {
              if (!wait(smem_u32(&sh.turn[a]), turn)) break;
              turn ^= 1;
            }
            values(stage, i > first);
            if (!ok) break;
            if (i + 2 >= end) {
              commit(sh.o_full[a]);
              if (turns > 0 && elect_one()) bar_arrive(smem_u32(&sh.turn[a ^ 1]));
            }
          }
          release(stage, mine);
          advance();
        }
        continue;
      }
      q_operand = operand(q_at + a * TILE_BYTES, 16);
      if (!wait(smem_u32(&sh.kv_full[stage]), kv_phase)) break;
      if (lo < end) scores();
      release(stage, lo < end);
      if (lo + 1 >= end) commit(sh.q_empty);
      advance();
#pragma unroll 1
      for (int i = lo; i < hi; ++i) {   // (tiles that the other row tile alone sees are let go)
        const int v_stage = stage;
        if (!wait(smem_u32(&sh.kv_full[stage]), kv_phase)) break;
        advance();
        if (i + 1 < hi && !wait(smem_u32(&sh.kv_full[stage]), kv_phase)) break;
        if (i < end) {
          // The row tiles take turns.  Left alone they fall into step, and the tensor cores wait for both softmaxes, which share
          // the special function units: 4280 cycles a tile instead of 3300 (8 k tokens, all seen: 1132 us, 832).
          if (i < both) {
            if (!wait(smem_u32(&sh.turn[a]), turn)) break;
            turn ^= 1;
          }
          values(v_stage, i > lo);
          if (!ok) break;
          if (i + 1 < end) scores();
          else commit(sh.o_full[a]);
          if (i < both && elect_one()) bar_arrive(smem_u32(&sh.turn[a ^ 1]));
        }
        release(v_stage, i < end);
        if (i + 1 < hi) {
          release(stage, i < end);
          if (i + 2 == end) commit(sh.q_empty);
          advance();
        }
      }
    }
  } else if (warp == 9) {
    // ---- items, and their copies: Q, then K and V of one tile after the other
    Walk<ItemCount<BY_LENGTH>> walk(A, ItemCount<BY_LENGTH>{A, A.per_share});
    const int whole = BY_LENGTH ? INT_MAX : whole_items(A, walk);
    if (BY_LENGTH && lane == 0) *A.share_size = walk.count.per;   // (for the join; the same from every CTA)
    Item w;
    int stage = 0, round = 0, asked = 0;
    unsigned kv_phase = 1, q_phase = 1, to_raw = 0, raw_parity = 0, full_parity = 0, used = 0;   // a bit per stage: of the last copy into it
    bool ok = true;
    auto publish = [&] {
      const int at = round % ITEMS;
      if (!(ok = bar_wait(smem_u32(&sh.item_empty[at]), (round / ITEMS & 1) ^ 1, stop))) return;
      if (lane == 0) {
        sh.items[at] = w;
        bar_arrive(smem_u32(&sh.item_full[at]));
      }
      ++round;
    };
#pragma unroll 1
    for (int next = blockIdx.x; next >= 0;) {
      if (lane == 0) {
        bar_expect(smem_u32(&sh.next_full), 16);
        request_cta(smem_u32(&sh.next), smem_u32(&sh.next_full));
      }
      if (look_up(A, walk, whole, next, w)) publish();
      else w.lo = w.hi = 0;
      if (ok && w.hi > w.lo && lane == 0) {
        if ((ok = bar_wait_one(smem_u32(&sh.q_empty), q_phase, stop))) {
          q_phase ^= 1;
          bar_expect(smem_u32(&sh.q_full), w.paired ? TILE_BYTES : 2 * TILE_BYTES);
          for (int a = 0; a < (w.paired ? 1 : 2); ++a)
            for (int c = 0; c < 2; ++c)
              copy_box(q_at + a * TILE_BYTES + c * (TILE_BYTES / 2), &M.q, 64 * c, w.head0, w.at.q0 + w.i0 + a * half, smem_u32(&sh.q_full));
        }
#pragma unroll 1
        for (int i = w.lo; ok && i < w.hi; ++i) {
          const bool own = i >= w.before;
          const int token = own ? w.at.k0 + (i - w.before) * TILE : i * TILE;
#pragma unroll 1
          for (int side = 0; side < 2; ++side) {
            if (!(ok = bar_wait_one(smem_u32(&sh.kv_empty[stage]), kv_phase, stop))) break;
            const CUtensorMap* map = side ? (own ? &M.v : &M.pv) : (own ? &M.k : &M.pk);
            const bool raw_first = side && w.partly_seen(i);
            const uint32_t bar = smem_u32(raw_first ? &sh.v_raw[stage] : &sh.kv_full[stage]), bit = 1u << stage;
            if (used & bit) full_parity ^= bit;
            if (raw_first) raw_parity ^= bit;
            used |= bit;
            to_raw = raw_first ? to_raw | bit : to_raw & ~bit;
            bar_expect(bar, TILE_BYTES);
            for (int c = 0; c < 2; ++c) copy_box(kv_at + stage * TILE_BYTES + c * (TILE_BYTES / 2), map, 64 * c, w.kv, token, bar);
            if (++stage == KV_STAGES) stage = 0, kv_phase ^= 1;
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      // (an answer that does not come is waited for even where something else has gone wrong: it lands in this CTA's memory)
      if (!bar_wait(smem_u32(&sh.next_full), asked & 1, stop) || !ok) {
        bar_drain(smem_u32(&sh.next_full), asked & 1);
        ok = false;
        break;
      }
      ++asked;
      next = requested_cta(smem_u32(&sh.next));
      fence_generic_to_async();   // (read before the next answer is written)
      __syncwarp();
    }
    w.over = true;
    if (ok) publish();
    if (lane == 0) sh.copies = {q_phase, used, to_raw, raw_parity, full_parity};
  } else if (warp == 10) {
    // ---- V tiles that not every row sees
    unsigned parity = 0, fills = 0;   // a bit per stage; copies into stages before this item's
    bool ok = true;
#pragma unroll 1
    for (int round = 0; ok; ++round) {
      const Item* const item_at = item(round);
      if (!item_at) break;
      const Item& w = *item_at;
#pragma unroll 1
      for (int i = max(w.lo, w.before + w.seen_first / TILE); i < w.hi; ++i) {
        const int stage = (fills + 2 * (i - w.lo) + 1) % KV_STAGES, first = (i - w.before) * TILE;
        if (!w.partly_seen(i)) continue;
        if (!(ok = bar_wait(smem_u32(&sh.v_raw[stage]), parity >> stage & 1, stop))) break;
        parity ^= 1u << stage;
        // x * 0 added up is 0 as long as x is finite.  (Looked at one by one, the values of a tile took 7000 cycles.)
        uint4* const v = reinterpret_cast<uint4*>(tiles + (2 + stage) * TILE_BYTES);   // (which piece of a row comes where does not matter)
        const int from = max(w.seen_first - first, 0) * 8 + lane;                       // eight pieces of 16 bytes per row of 64 channels
        uint32_t zero = 0;
#pragma unroll 1
        for (int half_at = 0; half_at < TILE_BYTES / 16; half_at += TILE_BYTES / 32)
#pragma unroll 8
          for (int k = from; k < TILE_BYTES / 32; k += 32) {
            const uint4 x = v[half_at + k];
            zero = add_zeros<BF16>(zero, x.x), zero = add_zeros<BF16>(zero, x.y), zero = add_zeros<BF16>(zero, x.z), zero = add_zeros<BF16>(zero, x.w);
          }
        if (__any_sync(0xffffffffu, odd_pair<BF16>(zero))) {
          constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
          uint32_t* const word = reinterpret_cast<uint32_t*>(v);
          bool odd = false;
          for (int k = lane; k < TILE_BYTES / 4; k += 32) {
            const int j = first + (k >> 5 & (TILE - 1));
            if (j < w.seen_first || !odd_pair<BF16>(word[k])) continue;
            odd |= j < w.seen_last;
            if ((word[k] & e) == e) word[k] &= 0xFFFF0000u;
            if ((word[k] >> 16 & e) == e) word[k] &= 0x0000FFFFu;
          }
          if (odd) *const_cast<volatile int*>(&sh.odd[round % ITEMS]) = round;
        }
        fence_generic_to_async();
        __syncwarp();
        if (lane == 0) bar_arrive(smem_u32(&sh.kv_full[stage]));
      }
      fills += 2 * max(w.hi - w.lo, 0);
      fills %= KV_STAGES;
      done(round);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (*stop) {   // a wait has run out: what the roles have left in flight ends before the CTA does
    if ((warp == 8 || warp == 11) && elect_one()) {
      const uint32_t drained = smem_u32(&sh.drained[warp == 8 ? 0 : 1]);
      mma_commit(drained);
      bar_drain(drained, 0);
    }
    if (warp == 9 && lane == 0) {
      const LastCopies c = sh.copies;
      if (c.used || c.q_phase == 0) bar_drain(smem_u32(&sh.q_full), c.q_phase);
      for (int k = 0; k < KV_STAGES; ++k) {
        if (!(c.used >> k & 1)) continue;
        if (c.to_raw >> k & 1) bar_drain(smem_u32(&sh.v_raw[k]), (c.raw_parity >> k & 1) ^ 1);
        else bar_drain(smem_u32(&sh.kv_full[k]), c.full_parity >> k & 1);
      }
    }
    __syncthreads();
  }
  if (warp == 8) tmem_free(tmem, TMEM_COLUMNS);
  if (threadIdx.x == 0 && *stop) atomicAdd(&g_waits_expired, 1u);
}

// Joins the parts of a row: a warp per row.  What takes its time is one round trip to L2 after the other (starts, pairs, outputs).
template <bool BF16>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptArgs A) {
  using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), rows = static_cast<int64_t>(A.total_q) * A.nh_q;
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int token = static_cast<int>(row / A.nh_q), head = static_cast<int>(row % A.nh_q);
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int per = A.by_length ? __ldcg(A.share_size) : A.per_share;
  int parts = 0;   // of the token's rows; rows in no sequence have none
  for (int s0 = 0; s0 < A.n_seqs; s0 += 32) {
    const int s = s0 + lane;
    int q0 = 0, lq = 0, lk = 0;
    if (s < A.n_seqs) {
      q0 = start_of(A.q_starts, s, A.total_q), lq = max(start_of(A.q_starts, s + 1, A.total_q) - q0, 0);
      lk = max(start_of(A.k_starts, s + 1, A.total_k) - start_of(A.k_starts, s, A.total_k), 0);
    }
    const int i0 = (token - q0) >> A.block_shift << A.block_shift;
    if (token >= q0 && token < q0 + lq) parts = shares_of(A, is_longer(A, i0, lq) ? longer(per) : per, lq, lk);
  }
  parts = __reduce_max_sync(0xffffffffu, parts);
  if (parts < 2) return;   // (in no sequence, or written as a whole)
  // A lane has the pair of one part, up to 32 at a time; of their outputs eight are on the way at once.
  const float2* const ml = A.part_ml + row;
  const float* const po = A.part_o + row * 128 + 4 * lane;
  float m = -INFINITY, l = 0.f, ref = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int first = 0; first < parts; first += 32) {
    const int n = min(32, parts - first);
    const float2 part = lane < n ? __ldcg(ml + (first + lane) * rows) : make_float2(-INFINITY, 0.f);
    float top = part.x;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    top = fmaxf(m, top);
    ref = top == -INFINITY ? 0.f : top;
    const float before = exp2_approx(m - ref), f = part.y != 0.f ? exp2_approx(part.x - ref) : 0.f;   // (a part whose sum is 0 has no output)
    float sum = f * part.y;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    l = l * before + sum, m = top;
    o.x *= before, o.y *= before, o.z *= before, o.w *= before;
#pragma unroll 1
    for (int s = 0; s < n; s += 8) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __ldcg(reinterpret_cast<const float4*>(po + (first + min(s + k, n - 1)) * rows * 128));
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float by = __shfl_sync(0xffffffffu, f, s + k);   // (0 behind the last)
        if (by != 0.f) o.x += by * v[k].x, o.y += by * v[k].y, o.z += by * v[k].z, o.w += by * v[k].w;
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(static_cast<T*>(A.out) + row * 128 + 4 * lane) =
      make_uint2(narrow2<BF16>(o.x * inv, o.y * inv), narrow2<BF16>(o.z * inv, o.w * inv));
  if (lane == 0) A.lse[static_cast<int64_t>(head) * A.total_q + token] = l == 0.f ? -INFINITY : (ref + log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------------------------------------
// Importance
// ------------------------------------------------------------------------------------------------
// A tile of keys of one sequence and all heads, HB query heads of a kv head at a time: S^T = K Q^T with the keys as the matrix's rows,
// so that a thread holds all queries and heads of its key and the sum over the heads needs no other thread.  One CTA per SM goes
// from tile to tile; what it works on next is on its way meanwhile.
//   What bounds it: K from HBM, once (10.3 us for 32 k tokens of 8 heads at the copy bandwidth; 16 in a graph of such calls), as long as the
// first copies of all CTAs, which come together, and the launch are a good part of it.  Beside K every tile takes the queries of all
// heads from L2, 20 KB a kv head for 28 KB of K.  With a tile per CTA, two buffers and sums in shared memory it took 30 us.
//   warps 0-3, 4-7   exponentials and sums, a key per thread, every other eight columns (column = query * HB + head) each
//   warp 8           matrix products, into one of four places in tensor memory
//   warp 9           copies (K of a kv head and the last queries of the HB heads)
//   warp 10          the columns' denominators
constexpr int IMP_THREADS = 384, IMP_COLUMNS = 128, IMP_SLOTS = 4, IMP_STAGES = 4;   // columns: most per product; slots: products in flight
struct ImportanceShared {
  unsigned long long full[IMP_STAGES], empty[IMP_STAGES], s_full[IMP_SLOTS], s_empty[IMP_SLOTS], drained;
  uint32_t tmem;
  int stop;
  alignas(16) float log_sum[IMP_SLOTS][IMP_COLUMNS];
};
struct ImportanceShape {
  int rows, keys, columns, stages, tiles;   // keys per tile; columns: rows * HB in whole 16; tiles: as many as there can be
};
__host__ __device__ constexpr int imp_stage_bytes(const ImportanceShape& g) { return (g.keys + g.columns) * 256; }
static size_t imp_smem(const ImportanceShape& g) {   // (a product reads 128 rows of K, the last of them beyond a short tile)
  return g.stages * static_cast<size_t>(imp_stage_bytes(g)) + (TILE - g.keys) * 128 + sizeof(ImportanceShared);
}
struct KeyCount {
  int keys;
  static constexpr bool EVEN = true;
  __device__ __forceinline__ int blocks(int, int lk) const { return (lk + keys - 1) / keys; }
  __device__ __forceinline__ int each(int, int) const { return 1; }
};

template <bool BF16, int HB>
__global__ void __launch_bounds__(IMP_THREADS, 1) importance_kernel(const __grid_constant__ PromptArgs A, const __grid_constant__ PromptMaps M,
                                                                    const ImportanceShape G, const float* lse, __half* out) {
  extern __shared__ __align__(1024) unsigned char tiles[];
  const int stage_bytes = imp_stage_bytes(G), k_half = G.keys * 128;
  ImportanceShared& sh = *reinterpret_cast<ImportanceShared*>(tiles + G.stages * stage_bytes + (TILE - G.keys) * 128);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int per_kv = A.nh_q / A.nh_kv / HB, items = A.nh_kv * per_kv;   // products per tile
  volatile int* const stop = &sh.stop;
  if (warp == 8) tmem_alloc(smem_u32(&sh.tmem), IMP_SLOTS * IMP_COLUMNS);
  if (threadIdx.x == 0) {
    sh.stop = 0;
    bar_init(smem_u32(&sh.drained), 1);
    for (int i = 0; i < IMP_STAGES; ++i) {
      bar_init(smem_u32(&sh.full[i]), 1);
      bar_init(smem_u32(&sh.empty[i]), 1);
    }
    for (int i = 0; i < IMP_SLOTS; ++i) {
      bar_init(smem_u32(&sh.s_full[i]), 2);    // the product, the denominators
      bar_init(smem_u32(&sh.s_empty[i]), 8);
    }
    bar_init_fence();
  }
  if (warp == 9 && lane < 2) prefetch_map(lane ? &M.q : &M.k);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = uniform(sh.tmem);
  asm volatile("griddepcontrol.launch_dependents;");   // (with the tensor memory, as in the attention kernel: here two CTAs fit on an SM)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  Walk<KeyCount> walk(A, KeyCount{G.keys});
  Place w;
  auto next = [&](int tile) { return tile < G.tiles && walk.find(tile, w); };   // (never more than the starts allow when in order)
  int copy_stage = 0, used = 0;   // warp 9: where the next copy goes, stages in use
  unsigned copy_phase = 1;
  int slot = 0;
  unsigned slot_phase = 0;
  auto next_slot = [&] {
    if (++slot == IMP_SLOTS) slot = 0, slot_phase ^= 1;
  };
  if (warp < 8) {
    const int side = warp >> 2, key = threadIdx.x & 127;
    const float scale = A.scale_log2;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21) + 8 * side;
    constexpr int CHUNKS = IMP_COLUMNS / 16, EACH = 8 / HB;   // this side's eights of columns, and the queries in each
    bool ok = true;
#pragma unroll 1
    for (int tile = blockIdx.x; ok && next(tile); tile += gridDim.x) {
      const int t = min(G.rows, w.lq), j = w.block * G.keys + key;
      const int sees = A.causal ? j - (w.lk - t) : 0;   // the first of the t queries that sees this key
      float sum[CHUNKS * EACH];
#pragma unroll
      for (int i = 0; i < CHUNKS * EACH; ++i) sum[i] = 0.f;
      if (t > 0) {
#pragma unroll 1
        for (int item = 0; item < items; ++item) {
          if (!(ok = bar_wait(smem_u32(&sh.s_full[slot]), slot_phase, stop))) break;
          fence_after();
          const uint32_t at = lanes + slot * IMP_COLUMNS;
          const float* const log_sum = sh.log_sum[slot] + 8 * side;
          // (chunks of 32 of this side's columns, so that loads and exponentials of several are under way)
#pragma unroll
          for (int c4 = 0; c4 < CHUNKS; c4 += 4) {
            if (8 * side + 16 * c4 >= G.columns) break;
            uint32_t s[32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_load8(at + 16 * (c4 + c), s + 8 * c);   // (what lies behind the columns is not used)
            wait_loads(s);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (8 * side + 16 * (c4 + c) >= G.columns) break;
              const float4 d0 = *reinterpret_cast<const float4*>(log_sum + 16 * (c4 + c)), d1 = *reinterpret_cast<const float4*>(log_sum + 16 * (c4 + c) + 4);
              const float d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
#pragma unroll
              for (int k = 0; k < 8; ++k) sum[(c4 + c) * EACH + k / HB] += exp2_approx(fmaf(__uint_as_float(s[8 * c + k]), scale, -d[k]));
            }
          }
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(smem_u32(&sh.s_empty[slot]));
          next_slot();
        }
      }
      if (ok && key < G.keys && j < w.lk) {
        __half* const to = out + w.k0 + j;
#pragma unroll
        for (int i = 0; i < CHUNKS * EACH; ++i) {
          const int r = (16 * (i / EACH) + 8 * side) / HB + i % EACH;
          if (r < G.rows) to[static_cast<int64_t>(r) * A.total_k] = __float2half_rn(r < t && r >= sees ? sum[i] : 0.f);
        }
      }
    }
  } else if (warp == 8) {
    const uint32_t kind = mma_kind(BF16, TILE, G.columns, false);
    const uint64_t first = operand(smem_u32(tiles), 16);
    const int q_half = G.columns * 128;
    bool ok = true;
    int stage = 0;
    unsigned phase = 0;
#pragma unroll 1
    for (int tile = blockIdx.x; ok && next(tile); tile += gridDim.x) {
      const int n = uniform(w.lq > 0 ? items : 0);
#pragma unroll 1
      for (int item = 0; item < n; ++item) {
        if (!(ok = bar_wait(smem_u32(&sh.full[stage]), phase, stop) && bar_wait(smem_u32(&sh.s_empty[slot]), slot_phase ^ 1, stop))) break;
        fence_after();
        if (elect_one()) {
          const uint64_t k_at = first + (stage * stage_bytes >> 4), q_at = k_at + (G.keys * 256 >> 4);
#pragma unroll
          for (int c = 0; c < 8; ++c)
            mma_shared(tmem + slot * IMP_COLUMNS, k_at + (((c >> 2) * k_half + (c & 3) * 32) >> 4), q_at + (((c >> 2) * q_half + (c & 3) * 32) >> 4), kind, c > 0);
          mma_commit(smem_u32(&sh.s_full[slot]));
          mma_commit(smem_u32(&sh.empty[stage]));
        }
        if (++stage == G.stages) stage = 0, phase ^= 1;
        next_slot();
      }
    }
  } else if (warp == 9) {
    const uint32_t tiles_at = smem_u32(tiles);
    const unsigned bytes = 256u * (G.keys + G.rows * HB);
    bool ok = true;
#pragma unroll 1
    for (int tile = blockIdx.x; ok && next(tile); tile += gridDim.x) {
      const int n = w.lq > 0 ? items : 0, token = w.k0 + w.block * G.keys, query = w.q0 + w.lq - min(G.rows, w.lq);
      if (lane == 0)
#pragma unroll 1
        for (int item = 0; item < n; ++item) {
          if (!(ok = bar_wait_one(smem_u32(&sh.empty[copy_stage]), copy_phase, stop))) break;
          const uint32_t k_at = tiles_at + copy_stage * stage_bytes, q_at = k_at + G.keys * 256, bar = smem_u32(&sh.full[copy_stage]);
          bar_expect(bar, bytes);
          for (int c = 0; c < 2; ++c) {
            copy_box(k_at + c * k_half, &M.k, 64 * c, item / per_kv, token, bar);
            copy_box(q_at + c * G.columns * 128, &M.q, 64 * c, item * HB, query, bar);
          }
          if (used < G.stages) ++used;
          if (++copy_stage == G.stages) copy_stage = 0, copy_phase ^= 1;
        }
      ok = __all_sync(0xffffffffu, ok);
    }
  } else if (warp == 10) {
    bool ok = true;
#pragma unroll 1
    for (int tile = blockIdx.x; ok && next(tile); tile += gridDim.x) {
      const int t = min(G.rows, w.lq), n = w.lq > 0 ? items : 0;
      const float* const from = lse + w.q0 + w.lq - t;
      float v[4];
      auto load = [&](int item) {   // log2; 0 where a column is no query's
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int column = lane + 32 * k, r = column / HB, head = item * HB + column % HB;
          v[k] = item < n && r < t ? 1.4426950408889634f * __ldcg(from + static_cast<int64_t>(head) * A.total_q + r) : 0.f;
        }
      };
      load(0);
#pragma unroll 1
      for (int item = 0; item < n; ++item) {
        if (!(ok = bar_wait(smem_u32(&sh.s_empty[slot]), slot_phase ^ 1, stop))) break;
#pragma unroll
        for (int k = 0; k < 4; ++k) sh.log_sum[slot][lane + 32 * k] = v[k];
        load(item + 1);
        __syncwarp();
        if (lane == 0) bar_arrive(smem_u32(&sh.s_full[slot]));
        next_slot();
      }
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (*stop) {   // as in the attention kernel
    if (warp == 8 && elect_one()) {
      mma_commit(smem_u32(&sh.drained));
      bar_drain(smem_u32(&sh.drained), 0);
    }
    if (warp == 9 && lane == 0)
      for (int i = 1; i <= used; ++i) {   // the last `used` copies, in front of `copy_stage`
        const int at = (copy_stage - i + G.stages) % G.stages;
        bar_drain(smem_u32(&sh.full[at]), at < copy_stage ? copy_phase ^ 1 : copy_phase);
      }
    __syncthreads();
  }
  if (warp == 8) tmem_free(tmem, IMP_SLOTS * IMP_COLUMNS);
  if (threadIdx.x == 0 && *stop) atomicAdd(&g_waits_expired, 1u);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
// Query heads that share a row tile: those of one kv head, as many of them as a power of two takes (at most 32: four tokens).
static void set_groups(PromptArgs& A) {
  A.group = 1, A.row_shift = 7;
  while (A.group < 32 && A.nh_q / A.nh_kv % (2 * A.group) == 0) A.group *= 2, --A.row_shift;
  A.block_shift = A.row_shift + 1;
  A.groups = A.nh_q / A.group;
  A.groups_per_kv = A.groups / A.nh_kv;
}

static int prompt_args(const hqkv_prompt_t* p, bool values, PromptArgs& A) {
  HQKV_REQUIRE(p != nullptr, "prompt: null descriptor");
  HQKV_REQUIRE(p->dtype == HQKV_F16 || p->dtype == HQKV_BF16, "prompt: unknown type %d", p->dtype);
  HQKV_REQUIRE(p->D == 128, "prompt: head dim must be 128 (got %d)", p->D);
  HQKV_REQUIRE(p->nh_kv > 0 && p->nh_q > 0 && p->nh_q % p->nh_kv == 0, "prompt: nh_q (%d) must be a positive multiple of nh_kv (%d)",
               p->nh_q, p->nh_kv);
  HQKV_REQUIRE(p->nh_q <= 65535, "prompt: too many heads");
  HQKV_REQUIRE(p->n_seqs >= 0 && p->total_q >= 0 && p->total_k >= 0 && p->prefix_len >= 0, "prompt: negative size");
  HQKV_REQUIRE(p->total_q < (1ll << 30) && p->total_k < (1ll << 30) && p->prefix_len < (1ll << 30) && p->n_seqs < (1 << 24),
               "prompt: too many tokens or sequences");
  HQKV_REQUIRE(p->scale > 0.f && p->scale < 1e38f, "prompt: the scale must be positive, and below 1e38");
  const bool own = p->total_k > 0, before = p->prefix_len > 0;
  if (p->total_q > 0) {
    HQKV_REQUIRE(p->q && (!own || (p->k && (p->v || !values))) && (!before || (p->prefix_k && (p->prefix_v || !values))), "prompt: null pointer");
    HQKV_REQUIRE(p->n_seqs == 0 || (p->q_starts && p->k_starts && aligned(p->q_starts, 4) && aligned(p->k_starts, 4)),
                 "prompt: the starts are null or misaligned");
  }
  const void* const base[5] = {p->q, own ? p->k : nullptr, own && values ? p->v : nullptr, before ? p->prefix_k : nullptr,
                               before && values ? p->prefix_v : nullptr};
  const int64_t strides[5][2] = {{p->q_token, p->q_head}, {p->k_token, p->k_head}, {p->v_token, p->v_head},
                                 {p->prefix_k_token, p->prefix_k_head}, {p->prefix_v_token, p->prefix_v_head}};
  const int64_t entries[5][2] = {{p->total_q, p->nh_q}, {p->total_k, p->nh_kv}, {p->total_k, p->nh_kv}, {p->prefix_len, p->nh_kv}, {p->prefix_len, p->nh_kv}};
  for (int i = 0; i < 5; ++i) {
    if (!base[i]) continue;
    HQKV_REQUIRE(aligned(base[i], 16), "prompt: tensors must be 16-byte aligned");
    for (int d = 0; d < 2; ++d)
      HQKV_REQUIRE(entries[i][d] < 2 || (strides[i][d] > 0 && strides[i][d] % 8 == 0 && strides[i][d] < (1ll << 38)),
                   "prompt: strides must be multiples of 8 elements, and positive");
  }
  A = PromptArgs();
  A.q = p->q, A.k = p->k, A.v = p->v, A.pk = p->prefix_k, A.pv = p->prefix_v;
  A.q_token = p->q_token, A.q_head = p->q_head, A.k_token = p->k_token, A.k_head = p->k_head, A.v_token = p->v_token, A.v_head = p->v_head;
  A.pk_token = p->prefix_k_token, A.pk_head = p->prefix_k_head, A.pv_token = p->prefix_v_token, A.pv_head = p->prefix_v_head;
  A.q_starts = p->q_starts, A.k_starts = p->k_starts;
  A.n_seqs = p->n_seqs;
  A.total_q = static_cast<int>(p->total_q), A.total_k = static_cast<int>(p->total_k), A.prefix_len = static_cast<int>(p->prefix_len);
  A.nh_q = p->nh_q, A.nh_kv = p->nh_kv;
  A.causal = p->causal != 0;
  A.bf16 = p->dtype == HQKV_BF16;
  set_groups(A);
  A.scale_log2 = p->scale * 1.4426950408889634f;
  return HQKV_OK;
}

// Blocks of queries that all sequences together have at most (their lengths are on the device).
static int64_t most_blocks(const PromptArgs& A) {
  const int64_t tokens = int64_t{1} << A.block_shift, n = max(1, min(A.n_seqs, A.total_q));
  return (A.total_q + n * (tokens - 1)) >> A.block_shift;
}

// Blocks of one row tile, on which both halves of a CTA work, where there are at most two whole ones per SM and they see little but
// their own prompts.  us, 32 heads over 8, whole blocks / halves: 300 tokens 12.6 / 9.2, 1024 21.2 / 18.7, 2048 44.0 / 40.4, 2500 54 / 58,
// 4096 117 / 138; 3 x 500 21.7 / 18.1, 8 x 200 18.5 / 16.1, 8 x 300 23.3 / 23.4, 8 x 1000 85 / 96.  (Many keys before the queries are better shared
// out: two blocks of half the rows read them twice.)
static void choose_blocks(PromptArgs& A) {
  if (A.n_seqs > 0 && most_blocks(A) * A.groups <= 2 * PROMPT_CTAS && static_cast<int64_t>(A.prefix_len) + A.total_k - A.total_q <= A.total_q)
    A.block_shift = A.row_shift;
}

// Tiles of keys per share, and the shares that a block has at most.  Where the blocks do not fill the GPU, their keys are shared out:
// for one sequence so that it takes the least time in all - a microsecond a tile, and every share's parts are written and read - with at most
// an item for every CTA; for several the kernel chooses when it sees their lengths (share_size), or, where they are more than a warp
// counts at a time, into shares of which a CTA gets about three on average.
static int prompt_shares(PromptArgs& A) {
  choose_blocks(A);
  A.by_length = false;
  const int64_t blocks = most_blocks(A) * A.groups, n = max(1, A.n_seqs);
  const int64_t most = ceil_div(A.prefix_len, TILE) + ceil_div(A.total_k, TILE);
  int64_t per = max(int64_t{1}, most);
  if (blocks < PROMPT_CTAS && most > 1) {
    const int64_t average = ceil_div(A.prefix_len, TILE) + ceil_div(A.total_k, TILE * n);
    if (n == 1) {
      const double part = 1.6e-4 * A.total_q * A.nh_q;   // us: 1 KB a row, at HBM's rate
      double best = 0.;
      for (int64_t shares = 1; shares <= min(most, PROMPT_CTAS / blocks); ++shares) {
        const double us = static_cast<double>(ceil_div(most, shares)) + (shares > 1 ? part * shares : 0.);
        if (shares == 1 || us < best) best = us, per = ceil_div(most, shares);
      }
    }
    else per = max(int64_t{4}, ceil_div(blocks * average, 3 * PROMPT_CTAS));
    const int64_t room = max(int64_t{1}, 10 * PROMPT_CTAS / blocks);   // (the parts take memory)
    per = max(per, ceil_div(most, room));
    // (for few tiles the least share will do, and where the blocks are more than half as many as the CTAs one or two rounds are uneven)
    A.by_length = n > 1 && n <= 32 && room > 1 && most < (1 << 21) && 5 * blocks <= 3 * PROMPT_CTAS && blocks * average > SHARE_TILES * PROMPT_CTAS;
    if (A.by_length) {
      A.per_share = SHARE_TILES;
      return A.shares = static_cast<int>(min(room, ceil_div(most, SHARE_TILES)));
    }
  }
  A.per_share = static_cast<int>(per);
  A.shares = static_cast<int>(max(int64_t{1}, ceil_div(most, per)));
  // (as many sequences as a warp counts at a time, and items of like length: most of what they see lies before their queries, or all see all)
  A.split = A.shares == 1 && A.n_seqs >= 1 && A.n_seqs <= 32 && A.block_shift > A.row_shift &&
            (!A.causal || int64_t{n} * A.prefix_len + A.total_k - A.total_q >= A.total_q);
  return A.shares;
}

// Launched so that it may take its place while the kernel before it ends (see the waits in the kernels).
template <typename... Params, typename... Args>
static int launch_behind(void (*kernel)(Params...), int64_t grid, int block, size_t smem, cudaStream_t st, const Args&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  HQKV_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  return HQKV_OK;
}

static int tensor_map(CUtensorMap* map, const void* base, bool bf16, int64_t tokens, int heads, int64_t token_stride, int64_t head_stride,
                      int box_heads, int box_tokens) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;   // (whoever is first stores what every other thread would)
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    HQKV_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !f) return fail(HQKV_E_CUDA, "prompt: the driver has no cuTensorMapEncodeTiled");
    encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }
  const cuuint64_t size[3] = {128, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  // (a dimension of one entry may come with any stride)
  const cuuint64_t stride[2] = {static_cast<cuuint64_t>(heads > 1 ? 2 * head_stride : 256), static_cast<cuuint64_t>(tokens > 1 ? 2 * token_stride : 256)};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)}, step[3] = {1, 1, 1};
  const CUresult rc = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), size, stride,
                             box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return fail(HQKV_E_CUDA, "prompt: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(rc));
  return HQKV_OK;
}

static int launch_prompt(PromptArgs& A, int shares, cudaStream_t st) {
  PromptMaps M = {};
  if (int rc = tensor_map(&M.q, A.q, A.bf16, A.total_q, A.nh_q, A.q_token, A.q_head, A.group, TILE / A.group)) return rc;
  if (A.total_k > 0) {
    if (int rc = tensor_map(&M.k, A.k, A.bf16, A.total_k, A.nh_kv, A.k_token, A.k_head, 1, TILE)) return rc;
    if (int rc = tensor_map(&M.v, A.v, A.bf16, A.total_k, A.nh_kv, A.v_token, A.v_head, 1, TILE)) return rc;
  }
  if (A.prefix_len > 0) {
    if (int rc = tensor_map(&M.pk, A.pk, A.bf16, A.prefix_len, A.nh_kv, A.pk_token, A.pk_head, 1, TILE)) return rc;
    if (int rc = tensor_map(&M.pv, A.pv, A.bf16, A.prefix_len, A.nh_kv, A.pv_token, A.pv_head, 1, TILE)) return rc;
  }
  using Kernel = void (*)(PromptArgs, PromptMaps);
  static const Kernel kernels[4] = {prompt_kernel<false, false>, prompt_kernel<true, false>, prompt_kernel<false, true>, prompt_kernel<true, true>};
  static bool opted_in[64] = {};   // per device
  int dev = 0;
  HQKV_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !opted_in[dev]) {
    for (Kernel k : kernels) HQKV_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(PROMPT_SMEM)));
    if (dev >= 0 && dev < 64) opted_in[dev] = true;
  }
  int64_t items = most_blocks(A) * A.groups * shares + (A.split ? PROMPT_CTAS / 2 : 0);
  if (A.by_length) items = min(items, int64_t{2 * PROMPT_CTAS});
  HQKV_REQUIRE(items < (1ll << 30), "prompt: too many rows");
  return launch_behind(kernels[2 * A.by_length + A.bf16], items, PROMPT_THREADS, PROMPT_SMEM, st, A, M);
}

template <bool BF16, int HB>
static int launch_importance(const PromptArgs& A, const PromptMaps& M, const ImportanceShape& G, const float* lse, __half* out, cudaStream_t st) {
  static bool opted_in[64] = {};   // per device
  int dev = 0;
  HQKV_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !opted_in[dev]) {
    HQKV_CUDA(cudaFuncSetAttribute(importance_kernel<BF16, HB>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    if (dev >= 0 && dev < 64) opted_in[dev] = true;
  }
  return launch_behind(importance_kernel<BF16, HB>, min(G.tiles, PROMPT_CTAS), IMP_THREADS, imp_smem(G), st, A, M, G, lse, out);
}

static int launch_importance(const PromptArgs& A, const float* lse, int rows, __half* out, cudaStream_t st) {
  int hb = 1;   // query heads per product
  while (hb < 8 && A.nh_q / A.nh_kv % (2 * hb) == 0 && 2 * hb * rows <= IMP_COLUMNS) hb *= 2;
  ImportanceShape G;
  G.rows = rows;
  G.columns = (rows * hb + 15) / 16 * 16;
  // tiles of at most 128 keys, as many as make whole rounds of the CTAs (a sequence's last tile is half empty, on average)
  const int64_t n = max(1, min(A.n_seqs, A.total_k)), rounds = ceil_div(A.total_k + n * TILE / 2, PROMPT_CTAS * TILE);
  const int64_t keys = ceil_div(ceil_div(A.total_k, max(int64_t{1}, rounds * PROMPT_CTAS - n / 2)), 8) * 8;
  G.keys = static_cast<int>(max(int64_t{32}, min(int64_t{TILE}, keys)));
  const int64_t tiles = (A.total_k + n * (G.keys - 1)) / G.keys;
  G.tiles = static_cast<int>(tiles);   // (below 2^30 / 32 + 2^24)
  G.stages = IMP_STAGES;
  while (G.stages > 2 && imp_smem(G) > 227 * 1024) --G.stages;
  PromptMaps M = {};
  if (A.total_q > 0)
    if (int rc = tensor_map(&M.q, A.q, A.bf16, A.total_q, A.nh_q, A.q_token, A.q_head, hb, rows)) return rc;
  if (int rc = tensor_map(&M.k, A.k, A.bf16, A.total_k, A.nh_kv, A.k_token, A.k_head, 1, G.keys)) return rc;
  switch (hb) {
    case 1: return A.bf16 ? launch_importance<true, 1>(A, M, G, lse, out, st) : launch_importance<false, 1>(A, M, G, lse, out, st);
    case 2: return A.bf16 ? launch_importance<true, 2>(A, M, G, lse, out, st) : launch_importance<false, 2>(A, M, G, lse, out, st);
    case 4: return A.bf16 ? launch_importance<true, 4>(A, M, G, lse, out, st) : launch_importance<false, 4>(A, M, G, lse, out, st);
    default: return A.bf16 ? launch_importance<true, 8>(A, M, G, lse, out, st) : launch_importance<false, 8>(A, M, G, lse, out, st);
  }
}

int prefix_parts(const hqkv_prompt_t* p) {
  PromptArgs A;
  A.total_q = static_cast<int>(p->total_q), A.total_k = 0, A.n_seqs = 0, A.prefix_len = static_cast<int>(p->prefix_len);
  A.nh_q = p->nh_q, A.nh_kv = p->nh_kv;
  set_groups(A);
  return prompt_shares(A);
}

int prefix_partial(const hqkv_prompt_t* p, float* part_o, float2* part_ml, cudaStream_t st) {
  PromptArgs A;
  if (int rc = prompt_args(p, true, A)) return rc;
  A.part_o = part_o, A.part_ml = part_ml;
  A.partial = true;
  const int shares = prompt_shares(A);
  return launch_prompt(A, shares, st);
}

static size_t split_bytes(const PromptArgs& A, int shares, size_t* part_ml) {
  const size_t rows = static_cast<size_t>(A.total_q) * A.nh_q * shares;
  *part_ml = rows * 128 * sizeof(float);
  return shares > 1 ? *part_ml + rows * sizeof(float2) + sizeof(int) : 0;
}

}  // namespace hqkv

using namespace hqkv;

extern "C" size_t hqkv_prompt_workspace_bytes(const hqkv_prompt_t* prompt_host) {
  PromptArgs A;
  if (prompt_args(prompt_host, true, A) != HQKV_OK || A.total_q == 0 || A.n_seqs == 0) return 0;
  size_t ml;
  const int shares = prompt_shares(A);
  return split_bytes(A, shares, &ml);
}

extern "C" int hqkv_prompt_attention(const hqkv_prompt_t* prompt_host, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  PromptArgs A;
  if (int rc = prompt_args(prompt_host, true, A)) return rc;
  if (A.total_q == 0 || A.n_seqs == 0) return HQKV_OK;
  HQKV_REQUIRE(out && lse && aligned(out, 32) && aligned(lse, 4), "prompt: the outputs are null or misaligned");
  A.out = out, A.lse = lse;
  const int shares = prompt_shares(A);
  size_t ml;
  const size_t need = split_bytes(A, shares, &ml);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (shares == 1) return launch_prompt(A, 1, st);
  HQKV_REQUIRE(workspace && aligned(workspace, 256), "prompt: the workspace is null or not 256-byte aligned");
  if (workspace_bytes < need) return fail(HQKV_E_WORKSPACE, "prompt: the workspace holds %zu bytes, %zu needed", workspace_bytes, need);
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + ml);
  A.share_size = reinterpret_cast<int*>(A.part_ml + static_cast<int64_t>(A.total_q) * A.nh_q * shares);
  if (int rc = launch_prompt(A, shares, st)) return rc;
  return launch_behind(A.bf16 ? prompt_join_kernel<true> : prompt_join_kernel<false>, ceil_div(static_cast<int64_t>(A.total_q) * A.nh_q, 8), 256, 0, st, A);
}

extern "C" int hqkv_prompt_waits_expired(int reset, unsigned* count_host) {
  HQKV_REQUIRE(count_host != nullptr, "prompt_waits_expired: null pointer");
  const unsigned zero = 0;
  HQKV_CUDA(cudaDeviceSynchronize());   // (the copy alone does not wait for streams that do not wait for the default one)
  HQKV_CUDA(cudaMemcpyFromSymbol(count_host, hqkv::g_waits_expired, sizeof(unsigned)));
  if (reset) HQKV_CUDA(cudaMemcpyToSymbol(hqkv::g_waits_expired, &zero, sizeof(unsigned)));
  return HQKV_OK;
}

extern "C" int hqkv_prompt_limit_waits(int tries) {
#if HQKV_CHECKS_ENABLED
  const int n = tries > 0 ? min(tries, WAIT_TRIES) : WAIT_TRIES;
  HQKV_CUDA(cudaDeviceSynchronize());
  HQKV_CUDA(cudaMemcpyToSymbol(hqkv::g_wait_tries, &n, sizeof(int)));
  return HQKV_OK;
#else
  (void)tries;
  return fail(HQKV_E_UNSUPPORTED, "prompt_limit_waits: only the bounds-check build has a limit that can be set");
#endif
}

extern "C" int hqkv_prompt_importance(const hqkv_prompt_t* prompt_host, const float* lse, int rows, void* out_f16, void* stream) {
  PromptArgs A;
  if (int rc = prompt_args(prompt_host, false, A)) return rc;
  HQKV_REQUIRE(rows >= 1 && rows <= HQKV_IMPORTANCE_ROWS, "prompt_importance: rows must be 1 to %d (got %d)", HQKV_IMPORTANCE_ROWS, rows);
  if (A.total_k == 0 || A.n_seqs == 0) return HQKV_OK;
  HQKV_REQUIRE(out_f16 && aligned(out_f16, 2), "prompt_importance: the output is null or misaligned");
  HQKV_REQUIRE(A.total_q == 0 || (lse && aligned(lse, 4)), "prompt_importance: lse is null or misaligned");
  return launch_importance(A, lse, rows, static_cast<__half*>(out_f16), static_cast<cudaStream_t>(stream));
}
