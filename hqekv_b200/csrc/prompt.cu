// Attention over whole prompts and what a prompt leaves behind (sm_100a):
//   prompt_attention   softmax(scale q K^T) V over packed sequences, causal, query heads in groups; the keys of a sequence may
//                      reach further back than its queries, and every sequence may see a prefix that all of them share
//   prompt_importance  probabilities of each sequence's last queries, summed over the heads
//   prefix_partial     the same attention for single tokens that share a prefix, not yet normalised (decode.cu joins it with the
//                      sequences' own caches)
#include "prompt.cuh"

#include <cudaTypedefs.h>

#include <type_traits>

#include "tensor.cuh"

namespace hqkv {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ int start_of(const int* starts, int s, int total) { return min(max(starts[s], 0), total); }

// ------------------------------------------------------------------------------------------------
// Attention
// ------------------------------------------------------------------------------------------------
// A CTA takes 256 rows of queries - two tiles of 128 rows, a row being a (token, head of the group) - and walks the tiles of 128 keys that
// any of them sees: first the prefix, then the sequence's own.  One pass, with the running maximum and sum of the softmax.
//   warps 0-3, 4-7   softmax of the first and second row tile, a row per thread
//   warp 8           issues the matrix products (one thread)
//   warp 9           requests the tiles of Q, K and V (one thread)
//   warp 10          looks after V tiles that not every row sees (below)
// Tensor memory: S of both row tiles (128 columns each, overwritten by P in the type of V) and O of both.
constexpr int TILE = 128;                                // keys per tile, rows per row tile
constexpr int TILE_BYTES = TILE * 128 * 2;               // 64 channels of all its tokens, then the other 64
constexpr int KV_STAGES = 5;
constexpr int PROMPT_THREADS = 384;
constexpr unsigned TMEM_COLUMNS = 512;
constexpr float RESCALE_AT = 8.f;                        // powers of two that P may exceed 1 by

struct PromptWork {   // a block of a sequence, and where the sequence's queries and keys are
  int q0, lq, k0, lk, tile, found;
};
struct PromptShared {
  unsigned long long q_full, kv_full[KV_STAGES], kv_empty[KV_STAGES], v_raw[KV_STAGES];
  unsigned long long s_full[2], p_first[2], p_rest[2], o_full[2], drained;
  uint32_t tmem;
  int stop, odd_values;
  PromptWork work;
};
constexpr size_t PROMPT_SMEM = 1024 + (2 + KV_STAGES) * static_cast<size_t>(TILE_BYTES) + sizeof(PromptShared);
static_assert(PROMPT_SMEM <= 227 * 1024, "one CTA per SM");

static __device__ unsigned g_waits_expired;

// The t-th block of `tokens` queries or keys of all sequences (`starts` says whose), the last block of a sequence first: in a causal
// prompt it sees the most keys.  Lane `first` of the warp's result holds it; -1: there are not as many.
struct Block {
  int lane, seq, tile;
};
__device__ __forceinline__ Block find_block(const int* starts, int total, int n_seqs, int t, int tokens, int lane) {
  int before = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += 32) {
    const int s = s0 + lane;
    const int length = s < n_seqs ? max(start_of(starts, s + 1, total) - start_of(starts, s, total), 0) : 0;
    int sum = (length + tokens - 1) / tokens;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += up;
    }
    const unsigned past = __ballot_sync(0xffffffffu, t < before + sum);
    if (past) return {__ffs(past) - 1, s, before + sum - 1 - t};
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return {-1, 0, 0};
}
// What the CTA works on, into its shared memory.
__device__ __forceinline__ void find_work(const PromptArgs& A, const int* starts, int total, int t, int tokens, int lane, PromptWork& w) {
  if (lane == 0) w.found = 0;
  __syncwarp();
  if (A.n_seqs == 0) {   // a single sequence without keys of its own
    if (lane == 0) w.q0 = 0, w.lq = A.total_q, w.k0 = 0, w.lk = 0, w.tile = t, w.found = 1;
    return;
  }
  const Block b = find_block(starts, total, A.n_seqs, t, tokens, lane);
  if (lane != b.lane) return;
  w.q0 = start_of(A.q_starts, b.seq, A.total_q);
  w.lq = max(start_of(A.q_starts, b.seq + 1, A.total_q) - w.q0, 0);
  w.k0 = start_of(A.k_starts, b.seq, A.total_k);
  w.lk = max(start_of(A.k_starts, b.seq + 1, A.total_k) - w.k0, 0);
  w.tile = b.tile;
  w.found = 1;
}

// own keys that query i of its sequence sees
__device__ __forceinline__ int keys_seen(const PromptArgs& A, int i, int lq, int lk) {
  return A.causal ? min(max(i + 1 + lk - lq, 0), lk) : lk;
}

template <bool BF16>
__device__ __forceinline__ bool odd_pair(uint32_t v) {   // an infinity or NaN in either half
  constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
  return (v & e) == e || (v >> 16 & e) == e;
}

template <bool BF16>
__global__ void __launch_bounds__(PROMPT_THREADS, 1) prompt_kernel(const __grid_constant__ PromptArgs A, const __grid_constant__ PromptMaps M) {
  using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
  extern __shared__ unsigned char raw[];
  unsigned char* const tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  PromptShared& sh = *reinterpret_cast<PromptShared*>(tiles + (2 + KV_STAGES) * TILE_BYTES);
  const uint32_t q_at = smem_u32(tiles), kv_at = q_at + 2 * TILE_BYTES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = A.nh_q / A.group;                       // head groups of all kv heads
  const int t = blockIdx.x / groups, head0 = (blockIdx.x - t * groups) * A.group, kv = head0 / (A.nh_q / A.nh_kv);
  const int half = TILE / A.group, tokens = 2 * half;        // tokens per row tile and CTA
  if (warp == 0) find_work(A, A.q_starts, A.total_q, t, tokens, lane, sh.work);
  __syncthreads();
  if (!sh.work.found) return;
  const int q0 = sh.work.q0, lq = sh.work.lq, k0 = sh.work.k0, lk = sh.work.lk, i0 = sh.work.tile * tokens;   // i0: the CTA's first query in its sequence
  // tiles of keys: those of the prefix, then the own ones up to the last that a row tile sees; this CTA's are [lo, hi[a])
  const int before = (A.prefix_len + TILE - 1) / TILE;
  const int seen_first = keys_seen(A, i0, lq, lk), seen_last = keys_seen(A, min(i0 + tokens, lq) - 1, lq, lk);
  const int n1 = i0 + half < lq ? before + (seen_last + TILE - 1) / TILE : 0;
  const int n0 = before + (keys_seen(A, min(i0 + half, lq) - 1, lq, lk) + TILE - 1) / TILE;
  const int n = max(n0, n1);
  const int lo = static_cast<int>(static_cast<int64_t>(n) * blockIdx.y / gridDim.y), hi = static_cast<int>(static_cast<int64_t>(n) * (blockIdx.y + 1) / gridDim.y);
  const int hi0 = min(hi, n0), hi1 = min(hi, n1);
  volatile int* const stop = &sh.stop;
  if (warp == 8) tmem_alloc(smem_u32(&sh.tmem), TMEM_COLUMNS);
  if (threadIdx.x == 0) {
    sh.stop = 0, sh.odd_values = 0;
    bar_init(smem_u32(&sh.q_full), 1);
    bar_init(smem_u32(&sh.drained), 1);
    for (int i = 0; i < KV_STAGES; ++i) {
      bar_init(smem_u32(&sh.kv_full[i]), 1);
      bar_init(smem_u32(&sh.kv_empty[i]), 1);
      bar_init(smem_u32(&sh.v_raw[i]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      bar_init(smem_u32(&sh.s_full[a]), 1);
      bar_init(smem_u32(&sh.p_first[a]), 4);
      bar_init(smem_u32(&sh.p_rest[a]), 4);
      bar_init(smem_u32(&sh.o_full[a]), 1);
    }
    bar_init_fence();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  // Own V tiles that hold keys which some rows of the CTA do not see.  0 x NaN is NaN in a matrix product, so what lies behind
  // the last key that any row sees is set to 0; an infinity or NaN that only some rows see is set to 0 as well, and those rows
  // add it at the end.
  auto partly_seen = [&](int i) { return i >= before && (i - before + 1) * TILE > seen_first; };

  if (warp < 8) {
    // ---- softmax
    const int a = warp >> 2, row = threadIdx.x & 127, i = i0 + a * half + row / A.group, head = head0 + row % A.group;
    const int end = a ? hi1 : hi0, count = max(end - lo, 0);
    const bool live = i < lq;
    const int seen = live ? keys_seen(A, i, lq, lk) : lk;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);   // (32 lanes a warp, in bits 16 and up)
    const uint32_t s_at = lanes + a * TILE, o_at = lanes + 2 * TILE + a * 128;
    float ref = -INFINITY, sum = 0.f;
    const float scale = A.scale_log2;
    bool ok = true;
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      if (!(ok = __all_sync(0xffffffffu, bar_wait(smem_u32(&sh.s_full[a]), it & 1, stop)))) break;
      fence_after();
      uint32_t s[TILE];
#pragma unroll
      for (int c = 0; c < TILE; c += 32) tmem_load32(s_at + c, s + c);
      wait_loads();
      const int tile = lo + it, limit = tile < before ? A.prefix_len - tile * TILE : seen - (tile - before) * TILE;
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
      const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * scale;
      // O and the sum are scaled to the maximum only where it has grown enough to matter: P stays below 2^8
      const bool grown = top > ref + RESCALE_AT;
      if (__any_sync(0xffffffffu, grown)) {
        const float f = grown ? exp2_approx(ref - top) : 1.f;
        if (grown) ref = top;
        sum *= f;
        if (it > 0) {
          // (the product with the tile before, which was issued before this S, is complete)
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            uint32_t o[32];
            tmem_load32(o_at + c, o);
            wait_loads();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_store32(o_at + c, o);
          }
        }
      }
      const float shift = ref == -INFINITY ? 0.f : -ref;
      const uint64_t scale2 = pair(scale, scale), shift2 = pair(shift, shift);
      uint64_t sums[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < TILE; c += 32) {
        uint32_t p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x, y;
          unpair(pair_fma(pair(__uint_as_float(s[c + 2 * k]), __uint_as_float(s[c + 2 * k + 1])), scale2, shift2), x, y);
          x = exp2_approx(x), y = exp2_approx(y);
          sums[k & 1] = pair_add(sums[k & 1], pair(x, y));
          p[k] = narrow2<BF16>(x, y);
        }
        tmem_store16(s_at + c / 2, p);
        if (c >= TILE - 64) {
          wait_stores();
          fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(smem_u32(c == TILE - 64 ? &sh.p_first[a] : &sh.p_rest[a]));
        }
      }
      float x, y;
      unpair(pair_add(sums[0], sums[1]), x, y);
      sum += x + y;
    }
    // ---- output
    if (count > 0 && ok) ok = __all_sync(0xffffffffu, bar_wait(smem_u32(&sh.o_full[a]), 0, stop));
    if (ok) {
      fence_after();
      const int64_t at = (static_cast<int64_t>(q0 + i) * A.nh_q + head);
      const bool odd = *const_cast<volatile int*>(&sh.odd_values) != 0;
      const float by = A.part_o ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      if (live && A.part_o) A.part_ml[static_cast<int64_t>(blockIdx.y) * A.total_q * A.nh_q + at] = make_float2(ref, sum);
      else if (live) A.lse[static_cast<int64_t>(head) * A.total_q + q0 + i] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        uint32_t o[32];
        if (count > 0) {
          tmem_load32(o_at + c, o);
          wait_loads();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (!live) continue;
        if (odd) {
          const int to = min(seen, (end - before) * TILE);
          for (int j = max(seen_first, (lo - before) * TILE); j < to; ++j) {
            const T* v = static_cast<const T*>(A.v) + (k0 + j) * A.v_token + kv * A.v_head + c;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float x = to_float(v[k]);
              if (!isfinite(x)) o[k] = __float_as_uint(__uint_as_float(o[k]) + x);
            }
          }
        }
        if (A.part_o) {
          uint4* to = reinterpret_cast<uint4*>(A.part_o + (static_cast<int64_t>(blockIdx.y) * A.total_q * A.nh_q + at) * 128 + c);
#pragma unroll
          for (int k = 0; k < 8; ++k) to[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        } else {
          uint32_t h[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) h[k] = narrow2<BF16>(__uint_as_float(o[2 * k]) * by, __uint_as_float(o[2 * k + 1]) * by);
          uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(A.out) + at * 128 + c);
#pragma unroll
          for (int k = 0; k < 4; ++k) to[k] = make_uint4(h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
        }
      }
    }
  } else if (warp == 8) {
    // ---- matrix products
    if (lane == 0 && hi > lo) {
      constexpr uint32_t kind_s = mma_kind(BF16, TILE, TILE, false), kind_o = mma_kind(BF16, TILE, 128, true);
      int stage = 0;
      unsigned phase = 0;
      auto scores = [&](int a, uint32_t k_at) {   // S = Q K^T, 16 channels at a time
#pragma unroll
        for (int c = 0; c < 8; ++c)
          mma_shared(tmem + a * TILE, operand(q_at + a * TILE_BYTES + (c >> 2) * (TILE_BYTES / 2) + (c & 3) * 32, 16),
                     operand(k_at + (c >> 2) * (TILE_BYTES / 2) + (c & 3) * 32, 16), kind_s, c > 0);
        mma_commit(smem_u32(&sh.s_full[a]));
      };
      auto advance = [&] {
        if (++stage == KV_STAGES) stage = 0, phase ^= 1;
      };
      bool ok = bar_wait(smem_u32(&sh.q_full), 0, stop) && bar_wait(smem_u32(&sh.kv_full[0]), 0, stop);
      if (ok) {
        fence_after();
        if (lo < hi0) scores(0, kv_at);
        if (lo < hi1) scores(1, kv_at);
        mma_commit(smem_u32(&sh.kv_empty[0]));
        advance();
      }
#pragma unroll 1
      for (int i = lo; ok && i < hi; ++i) {
        const int v_stage = stage;
        if (!(ok = bar_wait(smem_u32(&sh.kv_full[stage]), phase, stop))) break;
        advance();
        const uint32_t v_at = kv_at + v_stage * TILE_BYTES, k_at = kv_at + stage * TILE_BYTES;
        bool have_k = false;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int end = a ? hi1 : hi0;
          if (i < end) {
            // O += P V, 16 keys at a time, the first three quarters as soon as they are there
            if (!(ok = bar_wait(smem_u32(&sh.p_first[a]), (i - lo) & 1, stop))) break;
            fence_after();
#pragma unroll
            for (int c = 0; c < 6; ++c)
              mma_tensor(tmem + 2 * TILE + a * 128, tmem + a * TILE + c * 8, operand(v_at + c * 2048, TILE_BYTES / 2), kind_o, c > 0 || i > lo);
            if (!(ok = bar_wait(smem_u32(&sh.p_rest[a]), (i - lo) & 1, stop))) break;
            fence_after();
#pragma unroll
            for (int c = 6; c < 8; ++c)
              mma_tensor(tmem + 2 * TILE + a * 128, tmem + a * TILE + c * 8, operand(v_at + c * 2048, TILE_BYTES / 2), kind_o, true);
            if (i + 1 == end) mma_commit(smem_u32(&sh.o_full[a]));
          }
          if (a == 1) mma_commit(smem_u32(&sh.kv_empty[v_stage]));
          if (i + 1 < end) {
            if (!have_k && !(ok = bar_wait(smem_u32(&sh.kv_full[stage]), phase, stop))) break;
            fence_after();
            have_k = true;
            scores(a, k_at);
          }
        }
        if (!ok) break;
        if (i + 1 < hi) {
          mma_commit(smem_u32(&sh.kv_empty[stage]));
          advance();
        }
      }
      if (!ok) {   // products in flight end before the CTA does
        mma_commit(smem_u32(&sh.drained));
        for (int k = 0; k < WAIT_TRIES && !bar_try(smem_u32(&sh.drained), 0); ++k) {
        }
      }
    }
  } else if (warp == 9) {
    // ---- copies: Q, then K and V of one tile after the other
    if (lane == 0 && hi > lo) {
      bar_expect(smem_u32(&sh.q_full), 2 * TILE_BYTES);
      for (int a = 0; a < 2; ++a)
        for (int c = 0; c < 2; ++c)
          copy_box(q_at + a * TILE_BYTES + c * (TILE_BYTES / 2), &M.q, 64 * c, head0, q0 + i0 + a * half, smem_u32(&sh.q_full));
      int stage = 0;
      unsigned phase = 1, to_raw = 0, raw_parity = 0, full_parity = 0, used = 0;   // a bit per stage: of the last copy into it
      bool ok = true;
#pragma unroll 1
      for (int i = lo; ok && i < hi; ++i) {
        const bool own = i >= before;
        const int token = own ? k0 + (i - before) * TILE : i * TILE;
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
          if (!(ok = bar_wait(smem_u32(&sh.kv_empty[stage]), phase, stop))) break;
          const CUtensorMap* map = side ? (own ? &M.v : &M.pv) : (own ? &M.k : &M.pk);
          const bool raw_first = side && partly_seen(i);
          const uint32_t bar = smem_u32(raw_first ? &sh.v_raw[stage] : &sh.kv_full[stage]), bit = 1u << stage;
          if (used & bit) full_parity ^= bit;
          if (raw_first) raw_parity ^= bit;
          used |= bit;
          to_raw = raw_first ? to_raw | bit : to_raw & ~bit;
          bar_expect(bar, TILE_BYTES);
          for (int c = 0; c < 2; ++c) copy_box(kv_at + stage * TILE_BYTES + c * (TILE_BYTES / 2), map, 64 * c, kv, token, bar);
          if (++stage == KV_STAGES) stage = 0, phase ^= 1;
        }
      }
      if (!ok) {   // copies in flight land before the CTA ends
        auto landed = [&](const unsigned long long& bar, unsigned parity) {
          for (int k = 0; k < WAIT_TRIES && !bar_try(smem_u32(&bar), parity); ++k) {
          }
        };
        landed(sh.q_full, 0);
        for (int k = 0; k < KV_STAGES; ++k) {
          if (!(used >> k & 1)) continue;
          if (to_raw >> k & 1) landed(sh.v_raw[k], (raw_parity >> k & 1) ^ 1);
          else landed(sh.kv_full[k], full_parity >> k & 1);
        }
      }
    }
  } else if (warp == 10) {
    // ---- V tiles that not every row sees
    unsigned parity = 0;   // a bit per stage
#pragma unroll 1
    for (int i = lo; i < hi; ++i) {
      if (!partly_seen(i)) continue;
      const int stage = (2 * (i - lo) + 1) % KV_STAGES, first = (i - before) * TILE;
      if (!bar_wait(smem_u32(&sh.v_raw[stage]), parity >> stage & 1, stop)) break;
      parity ^= 1u << stage;
      unsigned char* const v = tiles + (2 + stage) * TILE_BYTES;
      bool odd = false;
      // (which of a row's pieces of 16 bytes comes where does not matter here)
      for (int k = lane; k < TILE_BYTES / 16; k += 32) {
        const int token = first + (k >> 3 & (TILE - 1));
        if (token < seen_first) continue;
        uint4* const at = reinterpret_cast<uint4*>(v + k * 16);
        if (token >= seen_last) {
          *at = make_uint4(0u, 0u, 0u, 0u);
          continue;
        }
        uint4 x = *at;
        if (odd_pair<BF16>(x.x) || odd_pair<BF16>(x.y) || odd_pair<BF16>(x.z) || odd_pair<BF16>(x.w)) {
          odd = true;
          uint32_t* w = &x.x;
          constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
          for (int m = 0; m < 4; ++m) {
            if ((w[m] & e) == e) w[m] &= 0xFFFF0000u;
            if ((w[m] >> 16 & e) == e) w[m] &= 0x0000FFFFu;
          }
          *at = x;
        }
      }
      if (odd) *const_cast<volatile int*>(&sh.odd_values) = 1;
      fence_generic_to_async();
      __syncwarp();
      if (lane == 0) bar_arrive(smem_u32(&sh.kv_full[stage]));
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 8) tmem_free(tmem, TMEM_COLUMNS);
  if (threadIdx.x == 0 && *stop) atomicAdd(&g_waits_expired, 1u);
}

// Joins the parts of a row: a warp per row.
template <bool BF16>
__global__ void __launch_bounds__(256) prompt_join_kernel(const PromptArgs A, int splits) {
  using T = std::conditional_t<BF16, __nv_bfloat16, __half>;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), rows = static_cast<int64_t>(A.total_q) * A.nh_q;
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int token = static_cast<int>(row / A.nh_q), head = static_cast<int>(row % A.nh_q);
  bool in = false;
  for (int s = lane; s < A.n_seqs; s += 32)
    in |= token >= start_of(A.q_starts, s, A.total_q) && token < start_of(A.q_starts, s + 1, A.total_q);
  if (!__any_sync(0xffffffffu, in)) return;
  float m = -INFINITY, l = 0.f;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, A.part_ml[s * rows + row].x);
  const float ref = m == -INFINITY ? 0.f : m;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < splits; ++s) {
    const float2 part = A.part_ml[s * rows + row];
    if (part.y == 0.f) continue;   // it had no keys that this row sees
    const float f = exp2_approx(part.x - ref);
    const float4 v = *reinterpret_cast<const float4*>(A.part_o + (s * rows + row) * 128 + 4 * lane);
    l += f * part.y;
    o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(static_cast<T*>(A.out) + row * 128 + 4 * lane) =
      make_uint2(narrow2<BF16>(o.x * inv, o.y * inv), narrow2<BF16>(o.z * inv, o.w * inv));
  if (lane == 0) A.lse[static_cast<int64_t>(head) * A.total_q + token] = l == 0.f ? -INFINITY : (ref + log2f(l)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------------------------------------
// Importance
// ------------------------------------------------------------------------------------------------
// A CTA takes a tile of keys of one sequence and all heads, HB query heads of a kv head at a time: S^T = K Q^T with the keys as the
// matrix's rows, so that a thread holds all queries and heads of its key and the sum over the heads needs no other thread.
//   warps 0-3, 4-7   exponentials and sums, a key per thread, every other eight columns (column = query * HB + head) each
//   warp 8           matrix products;  warp 9  copies (K of a kv head and the last queries of the HB heads)
constexpr int IMP_THREADS = 320, IMP_COLUMNS = 128;   // columns: most per product
struct ImportanceShared {
  unsigned long long full[4], empty[4], s_full[2], s_empty[2], drained;
  uint32_t tmem;
  int stop;
  PromptWork work;
  alignas(16) float lse[2][IMP_COLUMNS];
};
struct ImportanceShape {
  int rows, keys, columns, stages;   // keys per tile; columns: rows * HB in whole 16
};
__host__ __device__ constexpr int imp_stage_bytes(const ImportanceShape& g) { return TILE_BYTES + g.columns * 256; }
static size_t imp_smem(const ImportanceShape& g) {
  return 1024 + g.stages * static_cast<size_t>(imp_stage_bytes(g)) + sizeof(float) * g.rows * TILE + sizeof(ImportanceShared);
}

template <bool BF16, int HB>
__global__ void __launch_bounds__(IMP_THREADS) importance_kernel(const __grid_constant__ PromptArgs A, const __grid_constant__ PromptMaps M,
                                                                 const ImportanceShape G, const float* lse, __half* out) {
  extern __shared__ unsigned char raw[];
  unsigned char* const tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int stage_bytes = imp_stage_bytes(G);
  float* const acc = reinterpret_cast<float*>(tiles + G.stages * stage_bytes);   // [rows][key]
  ImportanceShared& sh = *reinterpret_cast<ImportanceShared*>(acc + G.rows * TILE);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) find_work(A, A.k_starts, A.total_k, blockIdx.x, G.keys, lane, sh.work);
  __syncthreads();
  if (!sh.work.found) return;
  const int q0 = sh.work.q0, lq = sh.work.lq, k0 = sh.work.k0, lk = sh.work.lk, j0 = sh.work.tile * G.keys;
  const int t = min(G.rows, lq), first = q0 + lq - t;   // the queries
  const int per_kv = A.nh_q / A.nh_kv / HB, items = t > 0 ? A.nh_kv * per_kv : 0;
  volatile int* const stop = &sh.stop;
  if (warp == 8) tmem_alloc(smem_u32(&sh.tmem), 2 * IMP_COLUMNS);
  if (threadIdx.x == 0) {
    sh.stop = 0;
    bar_init(smem_u32(&sh.drained), 1);
    for (int i = 0; i < 4; ++i) {
      bar_init(smem_u32(&sh.full[i]), 1);
      bar_init(smem_u32(&sh.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(smem_u32(&sh.s_full[i]), 1);
      bar_init(smem_u32(&sh.s_empty[i]), 8);
    }
    bar_init_fence();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  if (warp < 8) {
    const int side = warp >> 2, key = threadIdx.x & 127, j = j0 + key;
    // the first of the t queries that sees this key
    const int sees = A.causal ? j - (lk - t) : 0;
    for (int r = side; r < G.rows; r += 2) acc[r * TILE + key] = 0.f;
    const float scale = A.scale_log2;
    const int column = threadIdx.x & 127, col_row = column / HB, col_head = column % HB;
    auto denominator = [&](int item) {   // of the column that this thread looks after: log2, 0 where there is none
      if (item >= items || col_row >= t) return 0.f;
      return 1.4426950408889634f * __ldg(lse + static_cast<int64_t>(item * HB + col_head) * A.total_q + first + col_row);
    };
    bool ok = true;
    float next = denominator(0);
#pragma unroll 1
    for (int item = 0; item < items; ++item) {
      float* const den = sh.lse[item & 1];
      if (side == 0) den[column] = next;
      asm volatile("bar.sync 1, 256;" ::: "memory");   // (a buffer is written again two items later: everyone has passed the barrier between)
      next = denominator(item + 1);
      ok = ok && __all_sync(0xffffffffu, bar_wait(smem_u32(&sh.s_full[item & 1]), item >> 1 & 1, stop));
      if (!ok) continue;   // (every warp comes to every barrier)
      fence_after();
      const uint32_t at = tmem + (static_cast<uint32_t>(warp & 3) << 21) + (item & 1) * IMP_COLUMNS;
#pragma unroll 1
      for (int c = 8 * side; c < G.columns; c += 16) {
        uint32_t s[8];
        tmem_load8(at + c, s);
        const float4 d0 = *reinterpret_cast<const float4*>(den + c), d1 = *reinterpret_cast<const float4*>(den + c + 4);
        const float d[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
        wait_loads();
#pragma unroll
        for (int k = 0; k < 8; k += HB) {
          float sum = 0.f;
#pragma unroll
          for (int h = 0; h < HB; ++h) sum += exp2_approx(fmaf(__uint_as_float(s[k + h]), scale, -d[k + h]));
          const int r = (c + k) / HB;
          if (r < t && r >= sees) acc[r * TILE + key] += sum;
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(smem_u32(&sh.s_empty[item & 1]));
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (ok && j < lk && key < G.keys)
      for (int r = side; r < G.rows; r += 2) out[static_cast<int64_t>(r) * A.total_k + k0 + j] = __float2half_rn(acc[r * TILE + key]);
  } else if (warp == 8) {
    if (lane == 0) {
      const uint32_t kind = mma_kind(BF16, TILE, G.columns, false), tiles_at = smem_u32(tiles), q_half = G.columns * 128;
      bool ok = true;
      int stage = 0;
      unsigned phase = 0;
#pragma unroll 1
      for (int item = 0; item < items; ++item) {
        if (!(ok = bar_wait(smem_u32(&sh.full[stage]), phase, stop) &&
                   bar_wait(smem_u32(&sh.s_empty[item & 1]), (item >> 1 & 1) ^ 1, stop))) break;
        fence_after();
        const uint32_t k_at = tiles_at + stage * stage_bytes, q_at = k_at + TILE_BYTES;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          mma_shared(tmem + (item & 1) * IMP_COLUMNS, operand(k_at + (c >> 2) * (TILE_BYTES / 2) + (c & 3) * 32, 16),
                     operand(q_at + (c >> 2) * q_half + (c & 3) * 32, 16), kind, c > 0);
        mma_commit(smem_u32(&sh.s_full[item & 1]));
        mma_commit(smem_u32(&sh.empty[stage]));
        if (++stage == G.stages) stage = 0, phase ^= 1;
      }
      if (!ok) {   // products in flight end before the CTA does
        mma_commit(smem_u32(&sh.drained));
        for (int k = 0; k < WAIT_TRIES && !bar_try(smem_u32(&sh.drained), 0); ++k) {
        }
      }
    }
  } else if (lane == 0) {
    const uint32_t tiles_at = smem_u32(tiles);
    const unsigned bytes = 256u * (G.keys + G.rows * HB);
    bool ok = true;
    int stage = 0, item = 0;
    unsigned phase = 1;
#pragma unroll 1
    for (; item < items; ++item) {
      if (!(ok = bar_wait(smem_u32(&sh.empty[stage]), phase, stop))) break;
      const uint32_t k_at = tiles_at + stage * stage_bytes, q_at = k_at + TILE_BYTES, bar = smem_u32(&sh.full[stage]);
      bar_expect(bar, bytes);
      for (int c = 0; c < 2; ++c) {
        copy_box(k_at + c * (TILE_BYTES / 2), &M.k, 64 * c, item / per_kv, k0 + j0, bar);
        copy_box(q_at + c * G.columns * 128, &M.q, 64 * c, item * HB, first, bar);
      }
      if (++stage == G.stages) stage = 0, phase ^= 1;
    }
    if (!ok)   // copies in flight land before the CTA ends
      for (int i = max(0, item - G.stages); i < item; ++i)
        for (int k = 0; k < WAIT_TRIES && !bar_try(smem_u32(&sh.full[i % G.stages]), i / G.stages & 1); ++k) {
        }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 8) tmem_free(tmem, 2 * IMP_COLUMNS);
  if (threadIdx.x == 0 && *stop) atomicAdd(&g_waits_expired, 1u);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
// Query heads that share a row tile: those of one kv head, as many of them as a power of two takes (at most 32: four tokens).
static int head_group(int nh_q, int nh_kv) {
  int g = 1;
  while (g < 32 && nh_q / nh_kv % (2 * g) == 0) g *= 2;
  return g;
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
  HQKV_REQUIRE(p->scale > 0.f && p->scale < INFINITY, "prompt: the scale must be positive and finite");
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
  A.group = head_group(p->nh_q, p->nh_kv);
  A.scale_log2 = p->scale * 1.4426950408889634f;
  return HQKV_OK;
}

// Blocks of queries that all sequences together have at most (their lengths are on the device).
static int64_t most_blocks(const PromptArgs& A) {
  const int64_t tokens = 2 * TILE / A.group, n = max(1, min(A.n_seqs, A.total_q));
  return (A.total_q + n * (tokens - 1)) / tokens;
}

// Where the CTAs do not fill the GPU, the tiles of keys are shared out as well.
static int prompt_splits(const PromptArgs& A) {
  const int64_t ctas = most_blocks(A) * (A.nh_q / A.group);
  const int64_t tiles = ceil_div(A.prefix_len, TILE) + ceil_div(A.total_k / max(1, A.n_seqs), TILE);
  return static_cast<int>(max(int64_t{1}, min(148 / max(int64_t{1}, ctas), tiles)));
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

static int launch_prompt(const PromptArgs& A, int splits, cudaStream_t st) {
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
  static bool opted_in[64] = {};   // per device
  int dev = 0;
  HQKV_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !opted_in[dev]) {
    HQKV_CUDA(cudaFuncSetAttribute(prompt_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(PROMPT_SMEM)));
    HQKV_CUDA(cudaFuncSetAttribute(prompt_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(PROMPT_SMEM)));
    if (dev >= 0 && dev < 64) opted_in[dev] = true;
  }
  const int64_t blocks = most_blocks(A) * (A.nh_q / A.group);
  HQKV_REQUIRE(blocks < (1ll << 31), "prompt: too many rows");
  const dim3 grid(static_cast<unsigned>(blocks), splits);
  (A.bf16 ? prompt_kernel<true> : prompt_kernel<false>)<<<grid, PROMPT_THREADS, PROMPT_SMEM, st>>>(A, M);
  HQKV_LAUNCH_CHECK("prompt");
  return HQKV_OK;
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
  const int64_t n = max(1, min(A.n_seqs, A.total_k)), blocks = (A.total_k + n * (G.keys - 1)) / G.keys;
  importance_kernel<BF16, HB><<<static_cast<unsigned>(blocks), IMP_THREADS, imp_smem(G), st>>>(A, M, G, lse, out);
  HQKV_LAUNCH_CHECK("importance");
  return HQKV_OK;
}

static int launch_importance(const PromptArgs& A, const float* lse, int rows, __half* out, cudaStream_t st) {
  int hb = 1;   // query heads per product
  while (hb < 8 && A.nh_q / A.nh_kv % (2 * hb) == 0 && 2 * hb * rows <= IMP_COLUMNS) hb *= 2;
  ImportanceShape G;
  G.rows = rows;
  G.columns = (rows * hb + 15) / 16 * 16;
  // as many tiles as two CTAs per SM take at once, of 64 to 128 keys
  const int64_t waves = ceil_div(A.total_k, 296 * TILE), keys = ceil_div(ceil_div(A.total_k, 296 * waves), 8) * 8;
  G.keys = static_cast<int>(max(int64_t{64}, min(int64_t{TILE}, keys)));
  G.stages = 4;
  while (G.stages > 2 && imp_smem(G) > 113 * 1024) --G.stages;
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

int prefix_splits(const hqkv_prompt_t* p) {
  PromptArgs A;
  A.total_q = static_cast<int>(p->total_q), A.total_k = 0, A.n_seqs = 0, A.prefix_len = static_cast<int>(p->prefix_len);
  A.nh_q = p->nh_q, A.nh_kv = p->nh_kv, A.group = head_group(p->nh_q, p->nh_kv);
  return prompt_splits(A);
}

int prefix_partial(const hqkv_prompt_t* p, float* part_o, float2* part_ml, int splits, cudaStream_t st) {
  PromptArgs A;
  if (int rc = prompt_args(p, true, A)) return rc;
  A.part_o = part_o, A.part_ml = part_ml;
  return launch_prompt(A, splits, st);
}

static size_t split_bytes(const PromptArgs& A, int splits, size_t* part_ml) {
  const size_t rows = static_cast<size_t>(A.total_q) * A.nh_q * splits;
  *part_ml = rows * 128 * sizeof(float);
  return splits > 1 ? *part_ml + rows * sizeof(float2) : 0;
}

}  // namespace hqkv

using namespace hqkv;

extern "C" size_t hqkv_prompt_workspace_bytes(const hqkv_prompt_t* prompt_host) {
  PromptArgs A;
  if (prompt_args(prompt_host, true, A) != HQKV_OK || A.total_q == 0 || A.n_seqs == 0) return 0;
  size_t ml;
  return split_bytes(A, prompt_splits(A), &ml);
}

extern "C" int hqkv_prompt_attention(const hqkv_prompt_t* prompt_host, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  PromptArgs A;
  if (int rc = prompt_args(prompt_host, true, A)) return rc;
  if (A.total_q == 0 || A.n_seqs == 0) return HQKV_OK;
  HQKV_REQUIRE(out && lse && aligned(out, 16) && aligned(lse, 4), "prompt: the outputs are null or misaligned");
  A.out = out, A.lse = lse;
  const int splits = prompt_splits(A);
  size_t ml;
  const size_t need = split_bytes(A, splits, &ml);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (splits == 1) return launch_prompt(A, 1, st);
  HQKV_REQUIRE(workspace && aligned(workspace, 256), "prompt: the workspace is null or not 256-byte aligned");
  if (workspace_bytes < need) return fail(HQKV_E_WORKSPACE, "prompt: the workspace holds %zu bytes, %zu needed", workspace_bytes, need);
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + ml);
  if (int rc = launch_prompt(A, splits, st)) return rc;
  const unsigned grid = static_cast<unsigned>(ceil_div(static_cast<int64_t>(A.total_q) * A.nh_q, 8));
  (A.bf16 ? prompt_join_kernel<true> : prompt_join_kernel<false>)<<<grid, 256, 0, st>>>(A, splits);
  HQKV_LAUNCH_CHECK("prompt_join");
  return HQKV_OK;
}

extern "C" int hqkv_prompt_waits_expired(int reset, unsigned* count_host) {
  HQKV_REQUIRE(count_host != nullptr, "prompt_waits_expired: null pointer");
  const unsigned zero = 0;
  HQKV_CUDA(cudaMemcpyFromSymbol(count_host, hqkv::g_waits_expired, sizeof(unsigned)));
  if (reset) HQKV_CUDA(cudaMemcpyToSymbol(hqkv::g_waits_expired, &zero, sizeof(unsigned)));
  return HQKV_OK;
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
