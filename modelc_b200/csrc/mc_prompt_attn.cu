// mc_prompt_attn.cu -- attention over whole packed prompts.
#include <math.h>

#include "mc_paged.cuh"

namespace mc {

struct PromptArgs {
  const void *q, *k, *v;  // [Tq][H][D], [Tk][Hk][D] with strides (elements)
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head;
  void* out;              // [Tq][H][D]
  const int *cu_q, *cu_k;
  int Tq, Tk, H, Hk, B, causal;
  float scale;
};

// One warp per (row, head): scores with a lane per key, then the values with
// a lane per dimension.
template <typename T, int D>
__global__ void __launch_bounds__(32) k_prompt_simple(const PromptArgs a) {
  constexpr int NB = D / 32;
  __shared__ float s_q[D];
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y;
  int z = -1;
  for (int i = 0; i < a.B; ++i)
    if (t >= a.cu_q[i] && t < a.cu_q[i + 1]) z = i;
  float o[NB] = {}, m = -INFINITY, l = 0.f;
  if (z >= 0) {
    const T* q = (const T*)a.q + t * a.q_tok + h * a.q_head;
    for (int i = lane; i < D; i += 32) s_q[i] = to_f(q[i]) * a.scale;
    __syncwarp();
    const int k0 = a.cu_k[z], L = min(a.cu_k[z + 1], a.Tk) - k0;
    const int n = a.causal ? min(L, a.cu_k[z + 1] - k0 - (a.cu_q[z + 1] - 1 - t)) : L;
    const int hk = h / (a.H / a.Hk);
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + lane;
      float x = -INFINITY;
      if (j < n) {
        const T* k = (const T*)a.k + (k0 + j) * a.k_tok + hk * a.k_head;
        x = 0.f;
        for (int i = 0; i < D; ++i) x += to_f(k[i]) * s_q[i];
      }
      float top = x;
      for (int f = 16; f; f >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, f));
      const float mn = fmaxf(m, top);
      const float c = m == -INFINITY ? 0.f : __expf(m - mn);
      const float e = x > -INFINITY ? __expf(x - mn) : (x != x ? x : 0.f);
      m = mn;
      l = l * c + e;
      for (int b = 0; b < NB; ++b) o[b] *= c;
      for (int i = 0; i < min(32, n - j0); ++i) {
        const float p = __shfl_sync(~0u, e, i);
        const T* v = (const T*)a.v + (k0 + j0 + i) * a.v_tok + hk * a.v_head;
        for (int b = 0; b < NB; ++b) o[b] += p * to_f(v[b * 32 + lane]);
      }
    }
    for (int f = 16; f; f >>= 1) l += __shfl_xor_sync(~0u, l, f);
  }
  T* out = (T*)a.out + ((size_t)t * a.H + h) * D;
  for (int b = 0; b < NB; ++b) out[b * 32 + lane] = from_f<T>(l != 0.f ? o[b] / l : 0.f);
}

}  // namespace mc

using namespace mc;

extern "C" mc_status mc_prompt_attention(const void* q, int64_t q_tok, int64_t q_head, const void* k,
                                         int64_t k_tok, int64_t k_head, const void* v, int64_t v_tok,
                                         int64_t v_head, int32_t dtype, int32_t n_q, int32_t n_k,
                                         int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                         const int32_t* cu_q, const int32_t* cu_k,
                                         int32_t n_sequences, float scale, int32_t causal, void* out,
                                         int32_t device, void* stream) {
  if (head_dim != 64 && head_dim != 128) return set_error(MC_E_SHAPE, "head dim must be 64 or 128");
  if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads)
    return set_error(MC_E_SHAPE, "heads must be a multiple of the key/value heads");
  if (dtype != MC_ACT_F16 && dtype != MC_ACT_BF16)
    return set_error(MC_E_DTYPE, "inputs must be f16 or bf16");
  if (n_q < 0 || n_k < 0 || n_sequences < 0) return set_error(MC_E_INVALID, "negative size");
  if (!isfinite(scale)) return set_error(MC_E_INVALID, "scale must be finite");
  if (n_q == 0) return MC_OK;
  if (!q || !out || !cu_q || !cu_k || (n_k && (!k || !v))) return set_error(MC_E_INVALID, "null pointer");
  MC_PCKS(paged_device(device));
  PromptArgs a{q, k, v, q_tok, q_head, k_tok, k_head, v_tok, v_head, out, cu_q, cu_k, n_q, n_k,
               n_heads, n_kv_heads, n_sequences, causal, scale};
  dim3 grid(n_q, n_heads);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == MC_ACT_F16) {
    if (head_dim == 128) k_prompt_simple<__half, 128><<<grid, 32, 0, s>>>(a);
    else k_prompt_simple<__half, 64><<<grid, 32, 0, s>>>(a);
  } else {
    if (head_dim == 128) k_prompt_simple<__nv_bfloat16, 128><<<grid, 32, 0, s>>>(a);
    else k_prompt_simple<__nv_bfloat16, 64><<<grid, 32, 0, s>>>(a);
  }
  MC_PCK(cudaGetLastError());
  return MC_OK;
}
