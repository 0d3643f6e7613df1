// mc_kv4_attn.cu -- attention of few query tokens over the 4-bit paged cache.
#include <math.h>

#include "mc_paged.cuh"

namespace mc {

struct Kv4Args {
  const void* q;  // [T][H][D] with strides
  long long q_tok, q_head;
  void* out;      // [T][H][D]
  const uint8_t* pool;
  const int *table, *kv_len, *cu_q;
  int T, H, Hk, B, width, n_pages;
  float scale;
};

// One warp per (query token, head): scores with a lane per key, then the
// values with a lane per dimension.
template <typename T, int D>
__global__ void __launch_bounds__(32) k_kv4_simple(const Kv4Args a) {
  constexpr int W = D / 8, NB = D / 32, PB = 32 / W;
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
    const int n = a.kv_len[z] - (a.cu_q[z + 1] - 1 - t);  // keys this row sees
    const int hk = h / (a.H / a.Hk);
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + lane, pi = j / kKv4Page;
      const int page = pi < a.width ? a.table[(size_t)z * a.width + pi] : -1;
      const bool on = j < n && page >= 0 && page < a.n_pages;
      const uint8_t* p = a.pool + ((size_t)max(page, 0) * a.Hk + hk) * kv4_page_bytes(D);
      const int s = j % kKv4Page;
      float x = 0.f;
      if (on) {
        const uint32_t* row = (const uint32_t*)(p + s * (D / 2));
        const __half* sc = (const __half*)(p + 64 * D);
        for (int i = 0; i < 8; ++i) {
          float acc = 0.f;
          for (int w = 0; w < W; ++w)
            acc += (float)((int)((row[kv4_word_at<D>(s, w)] >> (4 * kv4_nib(i))) & 15) - 8) * s_q[i * W + w];
          x += acc * __half2float(sc[kv4_scale_at(s, i / PB, NB)]);
        }
      }
      x = on ? x : -INFINITY;
      float top = x;
      for (int f = 16; f; f >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, f));
      const float mn = fmaxf(m, top);
      const float c = m == -INFINITY ? 0.f : __expf(m - mn);
      const float e = on && x > -INFINITY ? __expf(x - mn) : (x != x ? x : 0.f);
      m = mn;
      l = l * c + e;
      for (int b = 0; b < NB; ++b) o[b] *= c;
      const int cnt = min(32, n - j0);
      for (int i = 0; i < cnt; ++i) {
        const float e_i = __shfl_sync(~0u, e, i);
        const int page_i = __shfl_sync(~0u, on ? page : -1, i);
        if (page_i < 0) continue;
        const uint8_t* pv = a.pool + ((size_t)page_i * a.Hk + hk) * kv4_page_bytes(D);
        const int si = (j0 + i) % kKv4Page;
        const uint32_t* row = (const uint32_t*)(pv + 32 * D + si * (D / 2));
        const __half* sc = (const __half*)(pv + 68 * D);
        for (int b = 0; b < NB; ++b) {
          const int d = b * 32 + lane;
          o[b] += e_i * (float)((int)((row[kv4_word_at<D>(si, d % W)] >> (4 * kv4_nib(d / W))) & 15) - 8) *
                  __half2float(sc[kv4_scale_at(si, b, NB)]);
        }
      }
    }
    for (int f = 16; f; f >>= 1) l += __shfl_xor_sync(~0u, l, f);
  }
  T* out = (T*)a.out + ((size_t)t * a.H + h) * D;
  for (int b = 0; b < NB; ++b) out[b * 32 + lane] = from_f<T>(l != 0.f ? o[b] / l : 0.f);
}

}  // namespace mc

using namespace mc;

extern "C" mc_status mc_kv4_attention(const void* q, int64_t q_tok, int64_t q_head, int32_t dtype,
                                      int32_t n_tokens, int32_t n_heads, const void* pool,
                                      int64_t n_pages, int32_t n_kv_heads, int32_t head_dim,
                                      const int32_t* table, int32_t table_width,
                                      const int32_t* kv_len, const int32_t* cu_q,
                                      int32_t n_requests, float scale, void* out, int32_t device,
                                      void* stream) {
  if (head_dim != 64 && head_dim != 128) return set_error(MC_E_SHAPE, "head dim must be 64 or 128");
  if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads)
    return set_error(MC_E_SHAPE, "heads must be a multiple of the key/value heads");
  if (dtype != MC_ACT_F16 && dtype != MC_ACT_BF16)
    return set_error(MC_E_DTYPE, "queries must be f16 or bf16");
  if (n_tokens < 0 || n_requests < 0 || table_width < 0 || n_pages < 0)
    return set_error(MC_E_INVALID, "negative size");
  if (n_pages * kKv4Page > 0x7fffffffll) return set_error(MC_E_CAPACITY, "slots pass 31 bits");
  if (!isfinite(scale)) return set_error(MC_E_INVALID, "scale must be finite");
  if (n_tokens == 0) return MC_OK;
  if (!q || !out || !cu_q || (n_requests && (!kv_len || (table_width && !table))) || (n_pages && !pool))
    return set_error(MC_E_INVALID, "null pointer");
  if (n_pages && !aligned(pool, 16)) return set_error(MC_E_INVALID, "pool must be 16-byte aligned");
  MC_PCKS(paged_device(device));
  Kv4Args a{q, q_tok, q_head, out, (const uint8_t*)pool, table, kv_len, cu_q, n_tokens, n_heads,
            n_kv_heads, n_requests, table_width, (int)n_pages, scale};
  dim3 grid(n_tokens, n_heads);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == MC_ACT_F16) {
    if (head_dim == 128) k_kv4_simple<__half, 128><<<grid, 32, 0, s>>>(a);
    else k_kv4_simple<__half, 64><<<grid, 32, 0, s>>>(a);
  } else {
    if (head_dim == 128) k_kv4_simple<__nv_bfloat16, 128><<<grid, 32, 0, s>>>(a);
    else k_kv4_simple<__nv_bfloat16, 64><<<grid, 32, 0, s>>>(a);
  }
  MC_PCK(cudaGetLastError());
  return MC_OK;
}
