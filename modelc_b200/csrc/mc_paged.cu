// mc_paged.cu -- page bookkeeping, rotary positions and the 4-bit KV cache's
// append and read back (include/modelc_cuda.h, the paged serving section).
#include <algorithm>
#include <atomic>

#include "mc_paged.cuh"

namespace mc {

// ------------------------------------------------------------ device check
constexpr int kMaxDevices = 64;
static std::atomic<int> g_sms[kMaxDevices];  // SM count once checked, 0 before

mc_status paged_check(int device) {
  if (device < 0 || device >= kMaxDevices) return set_error(MC_E_INVALID, "bad device index");
  if (!g_sms[device].load(std::memory_order_acquire)) {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
      cudaGetLastError();
      return set_error(MC_E_CUDA, "no CUDA device");
    }
    if (device >= n) return set_error(MC_E_INVALID, "bad device index");
    int major = 0, minor = 0, sms = 0;
    MC_PCK(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
    MC_PCK(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device));
    MC_PCK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    if (major != 10 || minor != 0) return set_error(MC_E_CUDA, "not an sm_100 device");
    g_sms[device].store(sms, std::memory_order_release);
  }
  return MC_OK;
}

PagedDevice::PagedDevice(int device) : status(paged_check(device)) {
  if (status != MC_OK) return;
  int cur = -1;
  cudaError_t e = cudaGetDevice(&cur);
  if (e == cudaSuccess && cur != device) {
    e = cudaSetDevice(device);
    back_ = cur;
  }
  if (e != cudaSuccess) status = set_error(MC_E_CUDA, cudaGetErrorString(e));
}

int paged_sms(int device) { return g_sms[device].load(std::memory_order_acquire); }

// ---------------------------------------------- block tables and slot maps
struct SlotArgs {
  const int *kv_len, *q_len;
  int* table;
  const int *free_pages, *n_free;
  int *cu_q, *positions, *slots, *new_len, *n_free_out;
  int B, width, page, tokens, n_pages_free;
};

// Every block scans all requests, a chunk of one request per thread at a
// time, and places the tokens of its own stretch of the output that belong
// to the chunk: one launch, no exchange between blocks.  A fresh page is
// written into the table by the token that opens it (the one at a multiple
// of the page size), so tables cost no loop of their own.  The scan reads
// 8 B bytes from L2 in every block; what bounds the call is its latency.
// Lengths may be any int32: sums are taken in 64 bits, a position that passes
// 31 bits has no page, and what is written stops at kSlotMax.
constexpr int kSlotThreads = 1024;
constexpr int kSlotMax = 0x7fffffff;

__global__ void __launch_bounds__(kSlotThreads) k_paged_slots(const SlotArgs a) {
  __shared__ long long s_cu[kSlotThreads], s_start[kSlotThreads];
  __shared__ int s_kv[kSlotThreads];
  __shared__ long long w_tok[32], w_pg[32];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int per = (int)(((long long)a.tokens + gridDim.x - 1) / gridDim.x);
  const long long lo = (long long)blockIdx.x * per;
  const long long hi = min((long long)a.tokens, lo + per);
  const int n_free = max(*a.n_free, 0);
  long long base_tok = 0, base_pg = 0;
  if (blockIdx.x == 0 && tid == 0) a.cu_q[0] = 0;
  for (int z0 = 0; z0 < a.B; z0 += kSlotThreads) {
    const int z = z0 + tid;
    int kv = 0, q = 0;
    if (z < a.B) {
      kv = max(a.kv_len[z], 0);
      q = max(a.q_len[z], 0);
    }
    const int have = (int)min(((long long)kv + a.page - 1) / a.page, (long long)a.width);
    const int all = (int)min((long long)kv + q, (long long)kSlotMax);
    const int need = (int)min(((long long)all + a.page - 1) / a.page, (long long)a.width);
    long long tok = q, pg = need - have;  // inclusive sums over the chunk
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(~0u, tok, o), y = __shfl_up_sync(~0u, pg, o);
      if (lane >= o) tok += x, pg += y;
    }
    if (lane == 31) w_tok[wid] = tok, w_pg[wid] = pg;
    __syncthreads();
    if (wid == 0) {
      long long x = w_tok[lane], y = w_pg[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(~0u, x, o), v = __shfl_up_sync(~0u, y, o);
        if (lane >= o) x += u, y += v;
      }
      w_tok[lane] = x, w_pg[lane] = y;
    }
    __syncthreads();
    if (wid) tok += w_tok[wid - 1], pg += w_pg[wid - 1];
    const long long n_tok = w_tok[31], n_pg = w_pg[31];
    s_cu[tid] = tok - q;  // tokens of the chunk before this request
    s_start[tid] = pg - (need - have) - have;
    s_kv[tid] = kv;
    if (blockIdx.x == 0 && z < a.B) {
      a.cu_q[z + 1] = (int)min(base_tok + tok, (long long)kSlotMax);
      a.new_len[z] = all;
    }
    __syncthreads();
    // this chunk's tokens are [base_tok, base_tok + n_tok)
    const long long t0 = max(lo, base_tok), t1 = min(hi, base_tok + n_tok);
    const int nz = min(kSlotThreads, a.B - z0);
    for (long long t = t0 + tid; t < t1; t += kSlotThreads) {
      const long long i = t - base_tok;
      int l = 0, r = nz;  // the last request that starts at or before token i
      while (r - l > 1) {
        const int m = (l + r) >> 1;
        if (s_cu[m] <= i) l = m;
        else r = m;
      }
      const int kvl = s_kv[l], pos = (int)min(kvl + (i - s_cu[l]), (long long)kSlotMax), j = pos / a.page;
      int page = -1;
      if (j < a.width && pos < kSlotMax) {
        int* entry = a.table + (size_t)(z0 + l) * a.width + j;
        if ((long long)j * a.page >= kvl) {
          const long long nth = (long long)n_free - 1 - (base_pg + s_start[l] + j);
          if (nth >= 0 && nth < a.n_pages_free) page = a.free_pages[nth];
          if (pos % a.page == 0) *entry = page;
        } else {
          page = *entry;
        }
      }
      a.positions[t] = pos;
      const long long slot = (long long)page * a.page + pos % a.page;
      a.slots[t] = page < 0 || slot > 0x7fffffffll ? -1 : (int)slot;
    }
    // requests that the output cuts off: the pages that the tokens behind its
    // end open are taken all the same, so they have to be in the table
    if (base_tok + tok > a.tokens) {
      const long long placed = max(a.tokens - (base_tok + tok - q), 0ll);
      for (long long j = (kv + placed + a.page - 1) / a.page + blockIdx.x; j < need; j += gridDim.x) {
        const long long nth = (long long)n_free - 1 - (base_pg + s_start[tid] + j);
        a.table[(size_t)z * a.width + j] = nth >= 0 && nth < a.n_pages_free ? a.free_pages[nth] : -1;
      }
    }
    base_tok += n_tok;
    base_pg += n_pg;
    __syncthreads();
  }
  for (long long t = max(lo, base_tok) + tid; t < hi; t += kSlotThreads) {
    a.positions[t] = 0;
    a.slots[t] = -1;
  }
  if (blockIdx.x == 0 && tid == 0) *a.n_free_out = (int)max(*a.n_free - base_pg, -(long long)kSlotMax);
}

// -------------------------------------------------------- rotary positions
// cos and sin of position * frequency in 64 bits, rounded once: an angle of
// 1e5 radians held in 32 bits would be off by 4e-3.
__global__ void k_rope_table(const double* freq, int n, int positions, double factor, float* cs,
                             float* sn) {
  const long long total = (long long)positions * n;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    double s, c;
    sincos((double)(i / n) * freq[i % n], &s, &c);
    cs[i] = (float)(c * factor);
    sn[i] = (float)(s * factor);
  }
}

struct RopeArgs {
  const void *q, *k;
  void *qo, *ko;
  long long q_tok, q_head, k_tok, k_head;  // input strides, elements
  const int* positions;
  const float *cs, *sn;
  int T, H, Hk, D, rot, max_pos, HG;
};

template <typename T, int V>
struct __align__(sizeof(T) * V <= 16 ? sizeof(T) * V : 16) Pack {
  T x[V];
};

// A unit is 2V values of one head: V pairs, or 2V values behind the rotated
// part that are copied.  A thread keeps one (token, unit) for HPT heads, so
// its cos and sin are read once for all of them; consecutive threads take
// consecutive units, then heads.
template <typename TI, typename TO, int V, int HPT, bool HALF>
__global__ void __launch_bounds__(256) k_rope(const RopeArgs a) {
  const unsigned U = a.D / (2 * V);
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  const unsigned u = idx % U, rest = idx / U, hg = rest % a.HG, t = rest / a.HG;
  if (t >= (unsigned)a.T) return;
  const int half = a.rot / 2, RU = half / V;
  const bool turn = u < (unsigned)RU;
  // where the unit's two groups of V values start
  const int e0 = !turn ? a.rot + (u - RU) * 2 * V : HALF ? u * V : u * 2 * V;
  const int e1 = turn && HALF ? e0 + half : e0 + V;
  const int pos = a.positions[t];
  const bool known = pos >= 0 && pos < a.max_pos;
  Pack<TI, V> x0[HPT], x1[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = hg + i * a.HG;
    if (h < a.H + a.Hk) {
      const TI* p = h < a.H ? (const TI*)a.q + t * a.q_tok + h * a.q_head
                            : (const TI*)a.k + t * a.k_tok + (h - a.H) * a.k_head;
      x0[i] = *(const Pack<TI, V>*)(p + e0);
      x1[i] = *(const Pack<TI, V>*)(p + e1);
    }
  }
  Pack<float, V> c, s;
  if (turn && known) {
    c = *(const Pack<float, V>*)(a.cs + (size_t)pos * half + u * V);
    s = *(const Pack<float, V>*)(a.sn + (size_t)pos * half + u * V);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      c.x[j] = turn ? __int_as_float(0x7fffffff) : 1.f;  // no such position: NaN
      s.x[j] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = hg + i * a.HG;
    if (h >= a.H + a.Hk) break;
    Pack<TO, V> y0, y1;
    if (!turn) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y0.x[j] = from_f<TO>(to_f(x0[i].x[j]));
        y1.x[j] = from_f<TO>(to_f(x1[i].x[j]));
      }
    } else if (HALF) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float p = to_f(x0[i].x[j]), r = to_f(x1[i].x[j]);
        y0.x[j] = from_f<TO>(p * c.x[j] - r * s.x[j]);
        y1.x[j] = from_f<TO>(r * c.x[j] + p * s.x[j]);
      }
    } else {  // pair j of the unit: values 2j and 2j + 1 of its 2V
      float y[2 * V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float p = to_f(2 * j < V ? x0[i].x[(2 * j) % V] : x1[i].x[(2 * j) % V]);
        const float r = to_f(2 * j + 1 < V ? x0[i].x[(2 * j + 1) % V] : x1[i].x[(2 * j + 1) % V]);
        y[2 * j] = p * c.x[j] - r * s.x[j];
        y[2 * j + 1] = r * c.x[j] + p * s.x[j];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y0.x[j] = from_f<TO>(y[j]);
        y1.x[j] = from_f<TO>(y[V + j]);
      }
    }
    TO* o = h < a.H ? (TO*)a.qo + ((size_t)t * a.H + h) * a.D
                    : (TO*)a.ko + ((size_t)t * a.Hk + (h - a.H)) * a.D;
    *(Pack<TO, V>*)(o + e0) = y0;
    *(Pack<TO, V>*)(o + e1) = y1;
  }
}

template <typename TI, typename TO, int V, int HPT>
static cudaError_t run_rope(RopeArgs a, bool half, cudaStream_t s) {
  a.HG = (a.H + a.Hk + HPT - 1) / HPT;
  const long long n = (long long)a.T * a.HG * (a.D / (2 * V));
  const unsigned grid = (unsigned)((n + 255) / 256);
  if (half) k_rope<TI, TO, V, HPT, true><<<grid, 256, 0, s>>>(a);
  else k_rope<TI, TO, V, HPT, false><<<grid, 256, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename TI, typename TO>
static cudaError_t run_rope_types(const RopeArgs& a, bool half, int vec, bool wide, cudaStream_t s) {
  if (vec >= 4) {
    return wide ? run_rope<TI, TO, 4, 4>(a, half, s) : run_rope<TI, TO, 4, 1>(a, half, s);
  }
  return run_rope<TI, TO, 1, 1>(a, half, s);
}

// ------------------------------------------------ append to the 4-bit pages
struct AppendArgs {
  const void *k, *v;
  long long k_tok, k_head, v_tok, v_head;  // strides, elements
  const int* slots;
  uint8_t* pool;
  int T, Hk, n_slots;
};

// A row (a token's K or V of one head) is taken by D/8 lanes with 8
// consecutive values each, so loads are 16 or 32 bytes a lane.  Word w of a
// row holds the values w, w + W, ...: for each of the D/64 sets of 8 lanes
// (every lane of D = 64, lanes of one parity of D = 128) lane n's code j goes
// to word j of the set, nibble n.  That is a transposition of an 8 x 8 matrix
// of nibbles, three exchanges with the lane 4, 2 and 1 sets away.
template <int D>
__device__ __forceinline__ uint32_t nibble_transpose(uint32_t x) {
  constexpr int S = D / 64;  // lanes between neighbours of a set
  const int n = (threadIdx.x / S) % 8;
#pragma unroll
  for (int k = 4; k; k >>= 1) {
    const int sh = 4 * k;
    const uint32_t low = k == 4 ? 0x0000ffffu : k == 2 ? 0x00ff00ffu : 0x0f0f0f0fu;
    // lanes with bit k clear give their upper and get the other's lower parts
    const uint32_t got = __shfl_xor_sync(~0u, n & k ? x & low : (x >> sh) & low, k * S);
    x = n & k ? (x & low << sh) | got : (x & low) | got << sh;
  }
  return x;
}
// Even logical nibbles into the low, odd ones into the high half, and back.
__device__ __forceinline__ uint32_t nibbles_out(uint32_t x) {
  uint32_t e = x & 0x0f0f0f0fu, o = (x >> 4) & 0x0f0f0f0fu;
  e = (e | e >> 4) & 0x00ff00ffu, o = (o | o >> 4) & 0x00ff00ffu;
  e = (e | e >> 8) & 0xffffu, o = (o | o >> 8) & 0xffffu;
  return e | o << 16;
}
__device__ __forceinline__ uint32_t nibbles_in(uint32_t x) {
  uint32_t e = x & 0xffffu, o = x >> 16;
  e = (e | e << 8) & 0x00ff00ffu, o = (o | o << 8) & 0x00ff00ffu;
  e = (e | e << 4) & 0x0f0f0f0fu, o = (o | o << 4) & 0x0f0f0f0fu;
  return e | o << 4;
}
// Word that lane n of a set holds after the transposition.
template <int D>
__device__ __forceinline__ int lane_word(int c) {
  return D == 128 ? 8 * (c & 1) + (c >> 1) : c;
}

// The codes of 8 values x of one lane and their block's d.
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], float& d) {
  const int lane = threadIdx.x & 31;
  // the block's largest size over its 4 lanes (a NaN stays one), then the
  // first value that has it
  float top = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x[i])));
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float y = __shfl_xor_sync(~0u, top, o);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(y));
  }
  float mine = top;
  bool has = false;
#pragma unroll
  for (int i = 7; i >= 0; --i)
    if (fabsf(x[i]) == top) mine = x[i], has = true;
  const unsigned who = __ballot_sync(~0u, has) >> (lane & ~3) & 15u;
  top = __shfl_sync(~0u, mine, (lane & ~3) + (who ? __ffs(who) - 1 : 0));
  d = __fdiv_rn(top, -8.f);
  const float inv = d != 0.f ? __fdiv_rn(1.f, d) : 0.f;
  // codes without conversions: 2^23 + y, rounded down, has the code in its last
  // bits, and what stands before them is taken off the word at once
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // the product and the sum are rounded one by one, as the rule says
    const float y = __fadd_rn(__fmul_rn(x[i], inv), 8.5f);
    word += __float_as_uint(__fadd_rd(fminf(fmaxf(y, 0.f), 15.f), 8388608.f)) << (4 * i);
  }
  return word - 0x4B000000u * 0x11111111u;
}

// A thread takes K and V of PER (token, head) pairs, `step` apart, and has
// all their loads under way before it uses the first.
template <typename T, int D, bool VEC, int PER>
__global__ void __launch_bounds__(256) k_kv4_append(const AppendArgs a, uint32_t step) {
  constexpr int W = D / 8, NB = D / 32, V = VEC ? 16 / sizeof(T) : 1, N = 8 / V;
  const uint32_t first = (uint32_t)(((long long)blockIdx.x * 256 + threadIdx.x) / W), total = (uint32_t)(a.T * a.Hk);
  const int c = threadIdx.x % W;
  int slot[PER], h[PER];
  Pack<T, V> y[PER][2][N];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t th = first + i * step;
    const bool live = first < step && th < total;
    const uint32_t t = live ? th / (uint32_t)a.Hk : 0u;
    h[i] = live ? (int)(th - t * (uint32_t)a.Hk) : 0;
    slot[i] = live ? a.slots[t] : -1;
    const T* k = (const T*)a.k + t * a.k_tok + h[i] * a.k_head + 8 * c;
    const T* v = (const T*)a.v + t * a.v_tok + h[i] * a.v_head + 8 * c;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      y[i][0][n] = ((const Pack<T, V>*)k)[n];
      y[i][1][n] = ((const Pack<T, V>*)v)[n];
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float x[8], d;
#pragma unroll
      for (int n = 0; n < 8; ++n) x[n] = to_f(y[i][kv][n / V].x[n % V]);
      const uint32_t word = nibbles_out(nibble_transpose<D>(quantize8(x, d)));
      if (slot[i] < 0 || slot[i] >= a.n_slots) continue;
      const int s = slot[i] % kKv4Page;
      uint8_t* page = a.pool + ((size_t)(slot[i] / kKv4Page) * a.Hk + h[i]) * kv4_page_bytes(D);
      ((uint32_t*)(page + kv * 32 * D + s * (D / 2)))[kv4_word_at<D>(s, lane_word<D>(c))] = word;
      if (c % 4 == 0) ((__half*)(page + 64 * D + kv * 4 * D))[kv4_scale_at(s, c / 4, NB)] = __float2half_rn(d);
    }
}

struct ReadArgs {
  const uint8_t* pool;
  const int* slots;
  void *k, *v;  // [T][Hk][D]
  int T, Hk, n_slots;
};

template <typename T, int D, int PER>
__global__ void __launch_bounds__(256) k_kv4_read(const ReadArgs a, uint32_t step) {
  constexpr int W = D / 8, NB = D / 32, V = 16 / sizeof(T);
  const uint32_t first = (uint32_t)(((long long)blockIdx.x * 256 + threadIdx.x) / W), total = (uint32_t)(a.T * a.Hk);
  const int c = threadIdx.x % W;
  uint32_t word[PER][2] = {};
  float d[PER][2] = {};
  int slot[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t th = first + i * step;
    slot[i] = first < step && th < total ? a.slots[th / (uint32_t)a.Hk] : -1;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (slot[i] < 0 || slot[i] >= a.n_slots) continue;
    const int s = slot[i] % kKv4Page, h = (int)((first + i * step) % (uint32_t)a.Hk);
    const uint8_t* page = a.pool + ((size_t)(slot[i] / kKv4Page) * a.Hk + h) * kv4_page_bytes(D);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      word[i][kv] = ((const uint32_t*)(page + kv * 32 * D + s * (D / 2)))[kv4_word_at<D>(s, lane_word<D>(c))];
      d[i][kv] = __half2float(((const __half*)(page + 64 * D + kv * 4 * D))[kv4_scale_at(s, c / 4, NB)]);
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint32_t w = nibble_transpose<D>(nibbles_in(word[i][kv]));  // its own inverse
      const uint32_t th = first + i * step;
      if (first >= step || th >= total) continue;
      Pack<T, V>* o = (Pack<T, V>*)((T*)(kv ? a.v : a.k) + (size_t)th * D + 8 * c);
#pragma unroll
      for (int k = 0; k < 8 / V; ++k) {
        Pack<T, V> y;
#pragma unroll
        for (int n = 0; n < V; ++n)
          // 2^23 + code, less 2^23 + 8
          y.x[n] = from_f<T>((__uint_as_float(0x4B000000u | ((w >> (4 * (k * V + n))) & 15)) - 8388616.f) * d[i][kv]);
        o[k] = y;
      }
    }
}

template <template <typename, int> class F, int D, typename... A>
static cudaError_t by_type(int dtype, A&&... args) {
  if (dtype == MC_ACT_F32) return F<float, D>::run(args...);
  if (dtype == MC_ACT_F16) return F<__half, D>::run(args...);
  return F<__nv_bfloat16, D>::run(args...);
}
// (token, head) pairs that one thread takes: two once the single ones would
// fill the GPU more than once.
template <int D>
static int rows_per(int device, long long pairs) {
  return pairs * (D / 8) > 2048ll * paged_sms(device) ? 2 : 1;
}
static unsigned row_grid(uint32_t step, int W) { return (unsigned)(((long long)step * W + 255) / 256); }
template <typename T, int D>
struct Append {
  template <bool VEC>
  static cudaError_t run_vec(const AppendArgs& a, int device, cudaStream_t s) {
    const uint32_t n = (uint32_t)(a.T * a.Hk);
    if (rows_per<D>(device, n) == 2) {
      const uint32_t step = (n + 1) / 2;
      k_kv4_append<T, D, VEC, 2><<<row_grid(step, D / 8), 256, 0, s>>>(a, step);
    } else {
      k_kv4_append<T, D, VEC, 1><<<row_grid(n, D / 8), 256, 0, s>>>(a, n);
    }
    return cudaGetLastError();
  }
  static cudaError_t run(const AppendArgs& a, int device, cudaStream_t s) {
    // 16-byte loads where every row starts at a multiple of them
    const long long any = (a.k_tok | a.k_head | a.v_tok | a.v_head) * (long long)sizeof(T);
    return any % 16 == 0 && aligned(a.k, 16) && aligned(a.v, 16) ? run_vec<true>(a, device, s)
                                                                  : run_vec<false>(a, device, s);
  }
};
template <typename T, int D>
struct Read {
  static cudaError_t run(const ReadArgs& a, int device, cudaStream_t s) {
    const uint32_t n = (uint32_t)(a.T * a.Hk);
    if (rows_per<D>(device, n) == 2) {
      const uint32_t step = (n + 1) / 2;
      k_kv4_read<T, D, 2><<<row_grid(step, D / 8), 256, 0, s>>>(a, step);
    } else {
      k_kv4_read<T, D, 1><<<row_grid(n, D / 8), 256, 0, s>>>(a, n);
    }
    return cudaGetLastError();
  }
};

}  // namespace mc

using namespace mc;

// ------------------------------------------------------------------ C entries
extern "C" mc_status mc_paged_slots(const mc_slots_args* args, int32_t device, void* stream) {
  if (!args) return set_error(MC_E_INVALID, "null pointer");
  const int32_t *kv_len = args->kv_len, *q_len = args->q_len, *free_pages = args->free_pages,
                *n_free = args->n_free;
  int32_t *table = args->table, *cu_q = args->cu_q, *positions = args->positions, *slots = args->slots, *new_len = args->new_len, *n_free_out = args->n_free_out;
  const int32_t n_requests = args->n_requests, table_width = args->table_width,
                n_free_pages = args->n_free_pages, page_size = args->page_size, n_tokens = args->n_tokens;
  if (n_requests < 0 || n_tokens < 0 || table_width < 0 || n_free_pages < 0)
    return set_error(MC_E_INVALID, "negative size");
  if (page_size <= 0) return set_error(MC_E_SHAPE, "page size must be positive");
  if (!n_free || !cu_q || !n_free_out || (n_requests > 0 && (!kv_len || !q_len || !new_len)) ||
      (n_requests > 0 && table_width > 0 && !table) || (n_free_pages > 0 && !free_pages) ||
      (n_tokens > 0 && (!positions || !slots)))
    return set_error(MC_E_INVALID, "null pointer");
  MC_PAGED_DEVICE(device);
  SlotArgs a{kv_len, q_len, table, free_pages, n_free, cu_q, positions, slots, new_len, n_free_out,
             n_requests, table_width, page_size, n_tokens, n_free_pages};
  const int grid = std::max(1, std::min(paged_sms(device), n_tokens / kSlotThreads + 1));
  k_paged_slots<<<grid, kSlotThreads, 0, (cudaStream_t)stream>>>(a);
  MC_PCK(cudaGetLastError());
  return MC_OK;
}

extern "C" mc_status mc_rope_table(const double* freq, int32_t n_freq, int32_t positions,
                                   double factor, float* cos_out, float* sin_out, int32_t device,
                                   void* stream) {
  if (n_freq <= 0 || positions <= 0) return set_error(MC_E_SHAPE, "empty table");
  if (!freq || !cos_out || !sin_out) return set_error(MC_E_INVALID, "null pointer");
  MC_PAGED_DEVICE(device);
  const long long n = (long long)positions * n_freq;
  const int grid = (int)std::min<long long>((n + 255) / 256, 8ll * paged_sms(device));
  k_rope_table<<<grid, 256, 0, (cudaStream_t)stream>>>(freq, n_freq, positions, factor, cos_out, sin_out);
  MC_PCK(cudaGetLastError());
  return MC_OK;
}

static size_t act_size(int t) { return t == MC_ACT_F32 ? 4 : 2; }

extern "C" mc_status mc_rope(const mc_rope_args* args, int32_t device, void* stream) {
  if (!args) return set_error(MC_E_INVALID, "null pointer");
  const void *q = args->q, *k = args->k;
  const int32_t *positions = args->positions;
  const float *cos_table = args->cos_table, *sin_table = args->sin_table;
  void *q_out = args->q_out, *k_out = args->k_out;
  const int64_t q_tok = args->q_tok, q_head = args->q_head, k_tok = args->k_tok, k_head = args->k_head;
  const int32_t n_heads = args->n_heads, n_kv_heads = args->n_kv_heads, dtype = args->dtype,
                out_dtype = args->out_dtype, n_tokens = args->n_tokens, head_dim = args->head_dim,
                rot = args->rot, interleaved = args->interleaved, table_rows = args->table_rows;
  if (n_tokens < 0 || n_heads < 0 || n_kv_heads < 0) return set_error(MC_E_INVALID, "negative size");
  if (head_dim <= 0 || head_dim % 2 || rot <= 0 || rot % 2 || rot > head_dim)
    return set_error(MC_E_SHAPE, "rot must be even and positive, at most the (even) head dim");
  if (dtype < 0 || dtype > 2 || out_dtype < 0 || out_dtype > 2 ||
      (out_dtype != dtype && dtype != MC_ACT_F32))
    return set_error(MC_E_DTYPE, "output type: the input's, or any for f32 inputs");
  if (table_rows <= 0) return set_error(MC_E_SHAPE, "empty table");
  if (n_tokens == 0 || n_heads + n_kv_heads == 0) return MC_OK;
  if (!positions || !cos_table || !sin_table || (n_heads && (!q || !q_out)) ||
      (n_kv_heads && (!k || !k_out)))
    return set_error(MC_E_INVALID, "null pointer");
  if ((long long)n_tokens * (n_heads + n_kv_heads) * (head_dim / 2) >= (1ll << 31) * 4)
    return set_error(MC_E_CAPACITY, "too many values for one call");
  MC_PAGED_DEVICE(device);
  RopeArgs a{q, k, q_out, k_out, q_tok, q_head, k_tok, k_head, positions, cos_table, sin_table,
             n_tokens, n_heads, n_kv_heads, head_dim, rot, table_rows, 0};
  // Groups of four values where all sizes, strides and addresses allow the
  // aligned vector access they need, single values otherwise.
  const size_t vi = 4 * act_size(dtype), vo = 4 * act_size(out_dtype);
  const bool vec = (rot / 2) % 4 == 0 && head_dim % 8 == 0 && aligned(cos_table, 16) && aligned(sin_table, 16) &&
                   (!n_heads || (aligned(q, vi) && aligned(q_out, vo) && q_tok % 4 == 0 && q_head % 4 == 0)) &&
                   (!n_kv_heads || (aligned(k, vi) && aligned(k_out, vo) && k_tok % 4 == 0 && k_head % 4 == 0));
  if (!vec && (long long)n_tokens * (n_heads + n_kv_heads) * (head_dim / 2) >= (1ll << 31))
    return set_error(MC_E_CAPACITY, "too many values for one call");
  // Four heads a thread once that still fills the GPU.
  const bool wide = (long long)n_tokens * (n_heads + n_kv_heads) * head_dim >= (1ll << 22);
  cudaStream_t s = (cudaStream_t)stream;
  const int v = vec ? 4 : 1;
  const bool half = !interleaved;
  cudaError_t e;
  if (dtype == MC_ACT_F32)
    e = out_dtype == MC_ACT_F32   ? run_rope_types<float, float>(a, half, v, wide, s)
        : out_dtype == MC_ACT_F16 ? run_rope_types<float, __half>(a, half, v, wide, s)
                                  : run_rope_types<float, __nv_bfloat16>(a, half, v, wide, s);
  else if (dtype == MC_ACT_F16)
    e = run_rope_types<__half, __half>(a, half, v, wide, s);
  else
    e = run_rope_types<__nv_bfloat16, __nv_bfloat16>(a, half, v, wide, s);
  MC_PCK(e);
  return MC_OK;
}

static mc_status check_pool(const void* pool, int64_t n_pages, int32_t n_kv_heads, int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128) return set_error(MC_E_SHAPE, "head dim must be 64 or 128");
  if (n_kv_heads <= 0 || n_pages < 0) return set_error(MC_E_SHAPE, "bad pool shape");
  if (n_pages * kKv4Page > 0x7fffffffll) return set_error(MC_E_CAPACITY, "slots pass 31 bits");
  if (n_pages && (!pool || !aligned(pool, 16)))
    return set_error(MC_E_INVALID, "pool must be 16-byte aligned");
  return MC_OK;
}

extern "C" int64_t mc_kv4_page_bytes(int32_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? kv4_page_bytes(head_dim) : 0;
}

extern "C" mc_status mc_kv4_append(const mc_kv4_append_args* args, int32_t device, void* stream) {
  if (!args) return set_error(MC_E_INVALID, "null pointer");
  void *pool = args->pool;
  const void *k = args->k, *v = args->v;
  const int32_t *slots = args->slots;
  const int64_t n_pages = args->n_pages, k_tok = args->k_tok, k_head = args->k_head, v_tok = args->v_tok,
                v_head = args->v_head;
  const int32_t n_kv_heads = args->n_kv_heads, head_dim = args->head_dim, dtype = args->dtype,
                n_tokens = args->n_tokens;
  MC_PCKS(check_pool(pool, n_pages, n_kv_heads, head_dim));
  if (dtype < 0 || dtype > 2) return set_error(MC_E_DTYPE, "unknown type");
  if (n_tokens < 0) return set_error(MC_E_INVALID, "negative size");
  if (n_tokens == 0) return MC_OK;
  if (!k || !v || !slots) return set_error(MC_E_INVALID, "null pointer");
  if ((long long)n_tokens * n_kv_heads > 0x7fffffffll)
    return set_error(MC_E_CAPACITY, "too many rows for one call");
  MC_PAGED_DEVICE(device);
  AppendArgs a{k, v, k_tok, k_head, v_tok, v_head, slots, (uint8_t*)pool, n_tokens, n_kv_heads,
               (int)(n_pages * kKv4Page)};
  MC_PCK(head_dim == 128 ? (by_type<Append, 128>(dtype, a, device, (cudaStream_t)stream))
                         : (by_type<Append, 64>(dtype, a, device, (cudaStream_t)stream)));
  return MC_OK;
}

extern "C" mc_status mc_kv4_read(const mc_kv4_read_args* args, int32_t device, void* stream) {
  if (!args) return set_error(MC_E_INVALID, "null pointer");
  const void *pool = args->pool;
  const int32_t *slots = args->slots;
  void *k_out = args->k_out, *v_out = args->v_out;
  const int64_t n_pages = args->n_pages;
  const int32_t n_kv_heads = args->n_kv_heads, head_dim = args->head_dim, dtype = args->dtype,
                n_tokens = args->n_tokens;
  MC_PCKS(check_pool(pool, n_pages, n_kv_heads, head_dim));
  if (dtype < 0 || dtype > 2) return set_error(MC_E_DTYPE, "unknown type");
  if (n_tokens < 0) return set_error(MC_E_INVALID, "negative size");
  if (n_tokens == 0) return MC_OK;
  if (!k_out || !v_out || !slots) return set_error(MC_E_INVALID, "null pointer");
  if (!aligned(k_out, 16) || !aligned(v_out, 16))
    return set_error(MC_E_INVALID, "outputs must be 16-byte aligned");
  if ((long long)n_tokens * n_kv_heads > 0x7fffffffll)
    return set_error(MC_E_CAPACITY, "too many rows for one call");
  MC_PAGED_DEVICE(device);
  ReadArgs a{(const uint8_t*)pool, slots, k_out, v_out, n_tokens, n_kv_heads, (int)(n_pages * kKv4Page)};
  MC_PCK(head_dim == 128 ? (by_type<Read, 128>(dtype, a, device, (cudaStream_t)stream))
                         : (by_type<Read, 64>(dtype, a, device, (cudaStream_t)stream)));
  return MC_OK;
}
