// Attention over whole prompts and what a prompt leaves behind (sm_100a):
//   prompt_attention   softmax(scale q K^T) V over packed sequences, causal, query heads in groups; the keys of a sequence may
//                      reach further back than its queries, and every sequence may see a prefix that all of them share
//   prompt_importance  probabilities of each sequence's last queries, summed over the heads
//   prefix_partial     the same attention for single tokens that share a prefix, not yet normalised (decode.cu joins it with the
//                      sequences' own caches)
#include "prompt.cuh"

namespace hqkv {

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ int start_of(const int* starts, int s, int total) { return min(max(starts[s], 0), total); }

// A warp per query row, four channels per lane, one pass over the keys with the running maximum and sum of the softmax.
template <typename T>
__global__ void __launch_bounds__(256) prompt_rows_kernel(const PromptArgs A) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= static_cast<int64_t>(A.total_q) * A.nh_q) return;
  const int token = static_cast<int>(row / A.nh_q), head = static_cast<int>(row % A.nh_q), kv = head / (A.nh_q / A.nh_kv);
  int first = 0, own = 0;
  if (A.n_seqs > 0) {
    int s = 0;
    while (s < A.n_seqs && start_of(A.q_starts, s + 1, A.total_q) <= token) ++s;
    if (s == A.n_seqs || start_of(A.q_starts, s, A.total_q) > token) return;   // in no sequence
    first = start_of(A.k_starts, s, A.total_k);
    own = max(start_of(A.k_starts, s + 1, A.total_k) - first, 0);
    if (A.causal) own = min(max(token + 1 + own - start_of(A.q_starts, s + 1, A.total_q), 0), own);
  }
  auto load = [&](const void* base, int64_t at, float (&v)[4]) {
    const T* p = static_cast<const T*>(base) + at + 4 * lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_float(p[i]);
  };
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  load(A.q, token * A.q_token + head * A.q_head, q);
  const int n = A.prefix_len + own;
  for (int j = 0; j < n; ++j) {
    float k[4], v[4];
    if (j < A.prefix_len) {
      load(A.pk, j * A.pk_token + kv * A.pk_head, k);
      load(A.pv, j * A.pv_token + kv * A.pv_head, v);
    } else {
      const int64_t t = first + (j - A.prefix_len);
      load(A.k, t * A.k_token + kv * A.k_head, k);
      load(A.v, t * A.v_token + kv * A.v_head, v);
    }
    float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
    for (int b = 16; b; b >>= 1) s += __shfl_xor_sync(0xffffffffu, s, b);
    s *= A.scale_log2;
    const float mx = fmaxf(m, s), ref = mx == -INFINITY ? 0.f : mx;
    const float f = exp2f(m - ref), p = exp2f(s - ref);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + p * v[i];
    m = mx;
  }
  if (A.part_o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) A.part_o[row * 128 + 4 * lane + i] = o[i];
    if (lane == 0) A.part_ml[row] = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) static_cast<T*>(A.out)[row * 128 + 4 * lane + i] = from_float<T>(o[i] * inv);
  if (lane == 0) A.lse[static_cast<int64_t>(head) * A.total_q + token] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// A thread per key, the sums over the heads in shared memory.
constexpr int IMP_KEYS = 64;
template <typename T>
__global__ void __launch_bounds__(IMP_KEYS) prompt_importance_kernel(const PromptArgs A, const float* lse, int rows, __half* out) {
  extern __shared__ float acc[];   // [rows][IMP_KEYS]
  const int64_t key = static_cast<int64_t>(blockIdx.x) * IMP_KEYS + threadIdx.x;
  if (key >= A.total_k) return;
  for (int r = 0; r < rows; ++r) acc[r * IMP_KEYS + threadIdx.x] = 0.f;
  int s = 0;
  while (s < A.n_seqs && start_of(A.k_starts, s + 1, A.total_k) <= key) ++s;
  const bool in = s < A.n_seqs && start_of(A.k_starts, s, A.total_k) <= key;
  if (!in) return;
  const int k0 = start_of(A.k_starts, s, A.total_k), k1 = start_of(A.k_starts, s + 1, A.total_k);
  const int q0 = start_of(A.q_starts, s, A.total_q), q1 = start_of(A.q_starts, s + 1, A.total_q);
  const int t = min(rows, max(q1 - q0, 0)), rep = A.nh_q / A.nh_kv;
  for (int kv = 0; kv < A.nh_kv; ++kv) {
    const T* k = static_cast<const T*>(A.k) + key * A.k_token + kv * A.k_head;
    for (int h = kv * rep; h < (kv + 1) * rep; ++h)
      for (int r = 0; r < t; ++r) {
        const int i = q1 - t + r;
        if (A.causal && key - k0 > i + (k1 - k0) - q1) continue;
        const T* q = static_cast<const T*>(A.q) + i * A.q_token + h * A.q_head;
        float x = 0.f;
        for (int d = 0; d < 128; ++d) x = fmaf(to_float(q[d]), to_float(k[d]), x);
        acc[r * IMP_KEYS + threadIdx.x] += exp2f(x * A.scale_log2 - lse[static_cast<int64_t>(h) * A.total_q + i] * 1.4426950408889634f);
      }
  }
  for (int r = 0; r < rows; ++r) out[r * A.total_k + key] = __float2half_rn(acc[r * IMP_KEYS + threadIdx.x]);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
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
  for (int i = 0; i < 5; ++i) {
    if (!base[i]) continue;
    HQKV_REQUIRE(aligned(base[i], 16), "prompt: tensors must be 16-byte aligned");
    for (int64_t s : strides[i])
      HQKV_REQUIRE(s >= 0 && s % 8 == 0 && s < (1ll << 38), "prompt: strides must be multiples of 8 elements, and not negative");
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
  A.scale_log2 = p->scale * 1.4426950408889634f;
  return HQKV_OK;
}

static int launch_rows(const PromptArgs& A, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(A.total_q) * A.nh_q;
  const unsigned grid = static_cast<unsigned>(ceil_div(rows, 8));
  if (A.bf16) prompt_rows_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(A);
  else prompt_rows_kernel<__half><<<grid, 256, 0, st>>>(A);
  HQKV_LAUNCH_CHECK("prompt_rows");
  return HQKV_OK;
}

int prefix_splits(const hqkv_prompt_t*) { return 1; }

int prefix_partial(const hqkv_prompt_t* p, float* part_o, float2* part_ml, int, cudaStream_t st) {
  PromptArgs A;
  if (int rc = prompt_args(p, true, A)) return rc;
  A.part_o = part_o, A.part_ml = part_ml;
  return launch_rows(A, st);
}

}  // namespace hqkv

using namespace hqkv;

extern "C" size_t hqkv_prompt_workspace_bytes(const hqkv_prompt_t*) { return 0; }

extern "C" int hqkv_prompt_attention(const hqkv_prompt_t* prompt_host, void* out, float* lse, void*, size_t, void* stream) {
  PromptArgs A;
  if (int rc = prompt_args(prompt_host, true, A)) return rc;
  if (A.total_q == 0 || A.n_seqs == 0) return HQKV_OK;
  HQKV_REQUIRE(out && lse && aligned(out, 16) && aligned(lse, 4), "prompt: the outputs are null or misaligned");
  A.out = out, A.lse = lse;
  return launch_rows(A, static_cast<cudaStream_t>(stream));
}

extern "C" int hqkv_prompt_importance(const hqkv_prompt_t* prompt_host, const float* lse, int rows, void* out_f16, void* stream) {
  PromptArgs A;
  if (int rc = prompt_args(prompt_host, false, A)) return rc;
  HQKV_REQUIRE(rows >= 1 && rows <= HQKV_IMPORTANCE_ROWS, "prompt_importance: rows must be 1 to %d (got %d)", HQKV_IMPORTANCE_ROWS, rows);
  if (A.total_k == 0 || A.n_seqs == 0) return HQKV_OK;
  HQKV_REQUIRE(out_f16 && aligned(out_f16, 2), "prompt_importance: the output is null or misaligned");
  HQKV_REQUIRE(A.total_q == 0 || (lse && aligned(lse, 4)), "prompt_importance: lse is null or misaligned");
  const unsigned grid = static_cast<unsigned>(ceil_div(A.total_k, IMP_KEYS));
  const size_t smem = sizeof(float) * rows * IMP_KEYS;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (A.bf16) prompt_importance_kernel<__nv_bfloat16><<<grid, IMP_KEYS, smem, st>>>(A, lse, rows, static_cast<__half*>(out_f16));
  else prompt_importance_kernel<__half><<<grid, IMP_KEYS, smem, st>>>(A, lse, rows, static_cast<__half*>(out_f16));
  HQKV_LAUNCH_CHECK("prompt_importance");
  return HQKV_OK;
}
