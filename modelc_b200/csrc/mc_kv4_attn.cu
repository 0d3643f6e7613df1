// mc_kv4_attn.cu -- attention of few query tokens over the 4-bit paged cache.
//
// o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),
// k_j, v_j = (code - 8) d per block of 32 values.
//
// One pass over the pages.  All (request, key/value head, row block, page)
// units of a call form one line that is cut into equal stretches, one per
// warp of the GPU, so ragged lengths and few requests keep every SM's copies
// in flight; a warp that covers all pages of a row block writes its output,
// the others leave (max, sum, sum p v) for k_kv4_join.  A warp works alone:
// lane 0 streams whole pages (one contiguous bulk copy each) into the warp's
// own shared-memory ring, and no barrier between warps is needed.
//
// A code becomes its exact f16 value c - 8 in two instructions: (word & mask)
// | 0x6400 per half is 1024 + c (or 1024 + 16 c), and an exact f16 sum or
// fma takes the rest away.
//   scores:  S^T = K Q^T with mma.m16n8k16, 16 tokens as rows, 8 query rows as
//     columns; the block scale comes in in f32: S += (block's product) d.
//   values:  O^T = V^T P^T, 16 dimensions as rows; p takes the block's scale
//     with it, P' = f16(p d), and is transposed in registers.
// Feeding the bare codes as f16 subnormals (one AND) and taking -8 off by a
// second product was built first: the tensor cores align subnormal factors
// as if they were 2^-14, which left errors of 2^-13 of a block's scale.
// Accumulation, softmax statistics and merging are f32.  P' in f16 and the
// query in f16, scaled by a power of two per row (exact for bf16, and for f16
// but for values 2^-24 below the row's largest), are the only roundings besides
// the output's.  The weights are p = 2^(score - reference + K), with K such
// that p times the largest value scale so far stays below 2^14 (kv4_up): p d
// keeps f16's 11 bits down to 2^-28 of the largest and 2^-25 absolute below, so
// a row of small values, or one whose mass a single key takes, keeps its
// small weights too.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mc_paged.cuh"

namespace mc {

// Warps of a block (one block fills an SM) and the shared memory that their
// rings share: 12 warps of 2 pages of D = 128 (4 of D = 64) for 8 query rows,
// 8 warps of 3 (6) for 16 rows, whose accumulators take the registers.  (16
// warps of 128 registers, two to a ring and each on half of every page, were
// slower, 88 against 78 us for 273 MB.)  What bounds a call of 74 to 77 us over
// 273 MB, measured before the weights followed the value scales: copies of the
// kernel without the f16 arithmetic, without the logic, the tensor products, the
// scaling or the exponentials save 4 us at most each, one that only loads takes
// 61, and one that loads no page still takes 24: the start (a chain of loads of
// 1 us each to the first page, cold code) and the join of the parts.
template <int NP>
constexpr int kKv4Warps = NP == 1 ? 12 : 8;
constexpr int kKv4Rings = 24 * kv4_page_bytes(128);
// Headroom of the reference that takes the place of the running maximum, in
// log2 units: weights are 2^(score - reference) <= 1, and the accumulators
// are rescaled only when a score passes the reference.
constexpr float kKv4Headroom = 2.f;
// K for value scales below 2^(e - 14), e an f16 exponent field (0 for the
// subnormal ones, 30 for the largest).  In bf16 calls p itself is rounded to
// f16 before the product (short), and held below 2^14 where both factors then
// have 22 bits of range at least (kv4_short: the largest scale between 2^-7 and
// 2^6, values of 0.06 to 500).  Other calls round once, p d in f32 to f16: 770
// MB take 178 us so, and 158 the short way.  Following the largest scale costs
// 2 to 3 us of that.
template <bool SHORT>
__device__ __forceinline__ float kv4_up(int e) {
  return (float)(SHORT && e >= 8 ? min(14, 28 - e) : 28 - e);
}
__device__ __forceinline__ bool kv4_short(int e) { return e >= 8 && e <= 20; }

struct Kv4Args {
  const void* q;  // [T][H][D] with strides
  long long q_tok, q_head;
  void* out;      // [T][H][D]
  const uint8_t* pool;
  const int *table, *kv_len, *cu_q;
  int T, H, Hk, B, width, n_pages;
  float scale;
  // workspace
  long long* head;  // [0] units, [1] warps that have some, [2 + z] first unit of request z
  float* ml;        // [2 warps][rows][2] running maximum (log2 units) and sum
  float* part;      // [2 warps][rows][D] sum p v
};

struct Kv4Req {
  int c0, n, kv, pages, nb;  // first row of q, new tokens, tokens, pages, row blocks
};
template <int R>
__device__ __forceinline__ Kv4Req kv4_req(const Kv4Args& a, int z) {
  Kv4Req r;
  r.c0 = min(max(__ldg(a.cu_q + z), 0), a.T);
  r.n = max(min(__ldg(a.cu_q + z + 1), a.T) - r.c0, 0);
  r.kv = min(max(__ldg(a.kv_len + z), 0), 0x7fffff00);
  r.nb = (int)(((long long)r.n * (a.H / a.Hk) + R - 1) / R);
  // a request without tokens has one page that counts as absent
  r.pages = r.n ? max(1, min((r.kv + kKv4Page - 1) / kKv4Page, a.width)) : 0;
  return r;
}

// A place on the line of units, in shared memory: it is touched once a page,
// and the registers it would take are what bounds the warps of an SM.
struct Kv4Place {
  int z, hk, rb, page;  // request, key/value head, row block, page
  int pages, nb;        // of the request: pages, row blocks
};

// a / b, rounded down: an f32 estimate, put right by whole products (a 64-bit
// division takes a thousand cycles, and several stood between a warp and its
// first page).  The estimate is off by a 2^-22 of the quotient, and by one.
__device__ __forceinline__ long long line_div(long long a, long long b) {
  long long q = (long long)((float)a * __frcp_rn((float)b));
  while (q * b > a) --q;
  while ((q + 1) * b <= a) ++q;
  return q;
}
// First unit of warp w's stretch of a line of L units for N warps.
__device__ __forceinline__ long long line_at(int w, long long L, long long N) {
  const long long q = line_div(L, N);  // whole units for each, the rest spread
  return q * w + line_div((L - q * N) * w, N);
}

// m16n8k16, f16 operands, f32 accumulators: d = a b + c
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                      uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ float2 h2f(uint32_t x) {
  __half2 h;
  memcpy(&h, &x, 4);
  return __half22float2(h);
}
__device__ __forceinline__ uint32_t f2h(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  uint32_t x;
  memcpy(&x, &h, 4);
  return x;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8x8 matrix of f16 in a warp
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Two f16 without signs, as whole numbers: the larger ones (not NaN), and
// whether one is at least its bound.
__device__ __forceinline__ uint32_t max_pair(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("max.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
}
__device__ __forceinline__ bool reaches(uint32_t x, uint32_t bound) {
  uint32_t z;
  asm("set.ge.u32.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(bound));
  return z != 0;
}

// The f16 pair (c - 8) of the codes in the low (ODD = 0) or second nibbles of
// the halves of x.
template <int ODD>
__device__ __forceinline__ uint32_t codes(uint32_t x) {
  uint32_t y, z;  // (x & mask) | 0x6400 in one lop3
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "r"(ODD ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
  if (ODD)  // (1024 + 16 c) / 16 - 72
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(z) : "r"(y), "r"(0x2c002c00u), "r"(0xd480d480u));
  else  // 1024 + c - 1032
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(z) : "r"(y), "r"(0xe408e408u));
  return z;
}

template <typename T, int D, int NP>
__global__ void __launch_bounds__(32 * kKv4Warps<NP>, 1) k_kv4(const Kv4Args a) {
  constexpr int W = D / 8, NB = D / 32, R = 8 * NP;
  constexpr int kWarps = kKv4Warps<NP>, kThreads = 32 * kWarps;
  constexpr int PB = kv4_page_bytes(D), S = kKv4Rings / kWarps / PB, kRing = S * PB;
  constexpr int NV = D == 128 ? 8 : 4;  // 16-row tiles of V^T
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ long long s_pref[kThreads];  // units before thread i's share of the requests
  __shared__ long long s_warp[kWarps];
  __shared__ __align__(8) uint64_t s_full[kWarps][S];
  __shared__ int s_n[kWarps];
  __shared__ bool s_there[kWarps][S];
  __shared__ Kv4Place s_place[kWarps], s_src[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  // --- the line of units: thread i sums the requests [i per, (i + 1) per)
  const int per = (a.B + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int z = tid * per; z < min(a.B, (tid + 1) * per); ++z) {
    const Kv4Req r = kv4_req<R>(a, z);
    mine += (long long)a.Hk * r.nb * r.pages;
  }
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) s_warp[wid] = inc;
  if (lane < S) bar_init(&s_full[wid][lane], 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  long long L = 0, before = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < wid) before += s_warp[i];
    L += s_warp[i];
  }
  s_pref[tid] = before + inc - mine;
  const long long N = min((long long)gridDim.x * kWarps, L);
  if (blockIdx.x == 0) {
    long long at = before + inc - mine;
    for (int z = tid * per; z < min(a.B, (tid + 1) * per); ++z) {
      const Kv4Req r = kv4_req<R>(a, z);
      a.head[2 + z] = at;
      at += (long long)a.Hk * r.nb * r.pages;
    }
    if (tid == 0) a.head[0] = L, a.head[1] = N;
  }
  __syncthreads();
  const int me = wid * gridDim.x + blockIdx.x;  // neighbours of the line on different SMs
  if (me >= N) return;
  {
    // --- where the stretch starts
    const long long u0 = line_at(me, L, N), u1 = line_at(me + 1, L, N);
    int l = 0, r = kThreads;
    while (r - l > 1) {
      const int m = (l + r) >> 1;
      if (s_pref[m] <= u0) l = m;
      else r = m;
    }
    int z = l * per;
    long long at = s_pref[l];
    Kv4Req rq = kv4_req<R>(a, z);
    while (at + (long long)a.Hk * rq.nb * rq.pages <= u0) {
      at += (long long)a.Hk * rq.nb * rq.pages;
      rq = kv4_req<R>(a, ++z);
    }
    const int seg = (int)((u0 - at) / rq.pages);  // head * row blocks + row block
    const int page = (int)(u0 - at - (long long)seg * rq.pages);
    if (lane == 0) {
      s_place[wid] = s_src[wid] = Kv4Place{z, seg / rq.nb, seg % rq.nb, page, rq.pages, rq.nb};
      s_n[wid] = (int)(u1 - u0);
    }
    __syncwarp();
  }
  const int n = s_n[wid];

  // --- the producer, lane 0, with its own place on the line
  uint8_t* ring = ring_all + wid * kRing;
  Kv4Place& src = s_src[wid];
  auto page_id = [&]() -> int {
    return src.page < a.width ? __ldg(a.table + (size_t)src.z * a.width + src.page) : -1;
  };
  auto fetch = [&](int st, int id) {  // the page at the producer's place
    const bool there = id >= 0 && id < a.n_pages;
    s_there[wid][st] = there;
    if (there) {
      bar_expect(&s_full[wid][st], PB);
      copy_bulk(ring + st * PB, a.pool + ((size_t)id * a.Hk + src.hk) * PB, PB, &s_full[wid][st]);
    } else {
      bar_arrive(&s_full[wid][st]);
    }
  };
  auto forward = [&](Kv4Place& at) {
    if (++at.page < at.pages) return;
    at.page = 0;
    if (++at.rb < at.nb) return;
    at.rb = 0;
    if (++at.hk < a.Hk) return;
    at.hk = 0;
    do {
      if (++at.z >= a.B) return;
      const Kv4Req r = kv4_req<R>(a, at.z);
      at.pages = r.pages, at.nb = r.nb;
    } while (at.pages == 0 || at.nb == 0);
  };
  int nid = -1;  // the next page to fetch, read one page ahead
  if (lane == 0) {
    for (int i = 0; i < min(S, n); ++i) {
      fetch(i, page_id());
      if (i + 1 < n) forward(src);
    }
    if (S < n) nid = page_id();
  }

  const int G = a.H / a.Hk;
  // Row g of a score product is the first, row g + 8 the second token of the
  // pair (group of 8 g % 2, scale entry (g / 2) ^ 2 (g % 2)): one scale entry
  // holds both, and the rows that a quarter (K) or a half (V) of the warp
  // reads at once lie in different banks.
  int k_row[2], k_off[2], v_off[2][2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    k_row[e] = 8 * (g & 1) + kv4_token(2 * ((g >> 1) ^ ((g & 1) * 2)) + e);
    k_off[e] = k_row[e] * (D / 2) + (D == 128 ? (t * 16) ^ ((k_row[e] & 2) << 4) : t * 8);
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // rows 2t + j of the pairs' order
      const int r = 8 * j + kv4_token(2 * (t ^ (2 * j)) + e);
      v_off[j][e] = 32 * D + r * (D / 2) + (D == 128 ? (g * 8) ^ ((r & 2) << 4) : g * 4);
    }
  }
  // scale entries of the lane's pair, and of the pairs that lie in rows 2t and 2t + 1
  const int d_off = ((g & 1) * 4 + ((g >> 1) ^ ((g & 1) * 2))) * NB * 4;
  const int t_off[2] = {t * NB * 4, (4 + (t ^ 2)) * NB * 4};
  // For bf16 outputs p and its product with the scale are both rounded to f16:
  // twice 2^-11 against the output's 2^-8 (a fifth fewer instructions).  Pages
  // under a mask, and value scales that kv4_short excludes, have p d rounded once.
  constexpr bool FAST = std::is_same<T, __nv_bfloat16>::value;

  int st = 0, phase = 0;
  bool failed = false, lead = true;  // lead: the stretch's first row block
  for (int i = 0; i < n;) {
    int page = s_place[wid].page, end, first;
    // per column 2t, 2t + 1 of the products: query rows p * 8 + 2t + e
    float2 cs[NP], m[NP], l[NP], room[NP];
    int vis[NP][2];
    uint32_t bq[4 * (D / 64)][NP][2];
    {
    const Kv4Place at = s_place[wid];
    const Kv4Req rq = kv4_req<R>(a, at.z);
    const int hk = at.hk, rb = at.rb, rows = rq.n * G - rb * R;  // live rows of the block
    end = min(at.pages, page + (n - i));
    // every live row sees the whole page below this token
    first = rq.kv - rq.n + rb * R / G + 1;
    // --- the query rows, in f16 after scaling by a power of two
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      m[p] = make_float2(-INFINITY, -INFINITY);
      l[p] = make_float2(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = p * 8 + 2 * t + e;
        vis[p][e] = row < rows ? max(rq.kv - rq.n + (rb * R + row) / G + 1, 0) : 0;
      }
      const int row = p * 8 + g, idx = rb * R + row, j = idx / G;  // the row this lane reads
      const bool live = row < rows;
      const T* q = (const T*)a.q + (long long)(rq.c0 + (live ? j : 0)) * a.q_tok +
                   (long long)(hk * G + (live ? idx - j * G : 0)) * a.q_head;
      float x[8][W / 4];  // word t (W/4) + i of the row, logical nibble k
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int w = 0; w < W / 4; ++w) {
          x[k][w] = live ? to_f(q[k * W + t * (W / 4) + w]) : 0.f;
          top = fmaxf(top, fabsf(x[k][w]));
        }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      // 2^(13 - exponent of the largest value), so values lie below 2^14
      const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 100);
      const float up = __uint_as_float((uint32_t)(127 + 13 - ex) << 23);
      const float c = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - 13 + ex) << 23);
      cs[p] = make_float2(__shfl_sync(~0u, c, 8 * t), __shfl_sync(~0u, c, 8 * t + 4));
      // the headroom in the scores' units; none where they all have the same weight
      room[p].x = cs[p].x > 0.f ? fminf(kKv4Headroom / cs[p].x, 1e30f) : 0.f;
      room[p].y = cs[p].y > 0.f ? fminf(kKv4Headroom / cs[p].y, 1e30f) : 0.f;
      const float f = a.scale < 0.f ? -up : up;
#pragma unroll
      for (int k = 0; k < 4; ++k)  // values of the nibble pair (2k, 2k + 1)
#pragma unroll
        for (int w = 0; w < W / 4; ++w)
          bq[k * (D / 64) + w / 2][p][w & 1] = f2h(x[2 * k][w] * f, x[2 * k + 1][w] * f);
    }
    }
    int big = 0;  // exponent field of the largest value scale so far
    float up = kv4_up<FAST>(0);
    float o[NV][NP][4];
#pragma unroll
    for (int x = 0; x < NV; ++x)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[x][p][c] = 0.f;
    // 32 tokens, half a page, K codes at kp, K scales at sp; MASK: some row
    // does not see all of them
    auto step = [&](const uint8_t* kp, const uint8_t* sp, int base, auto mask) {
      constexpr bool MASK = decltype(mask)::value;
      // --- scores: [2e + column] of token pairs
      float s[2][NP][4];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t k0[W / 4], k1[W / 4], sc[NB];
        if constexpr (D == 128) {
          *(uint4*)k0 = *(const uint4*)(kp + c * 8 * D + k_off[0]);
          *(uint4*)k1 = *(const uint4*)(kp + c * 8 * D + k_off[1]);
          *(uint4*)sc = *(const uint4*)(sp + c * D + d_off);
        } else {
          *(uint2*)k0 = *(const uint2*)(kp + c * 8 * D + k_off[0]);
          *(uint2*)k1 = *(const uint2*)(kp + c * 8 * D + k_off[1]);
          *(uint2*)sc = *(const uint2*)(sp + c * D + d_off);
        }
        float acc[NP][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
          for (int j = 0; j < D / 64; ++j) {
            auto part = [&](uint32_t w) {
              w >>= 8 * (k / 2);
              return k & 1 ? codes<1>(w) : codes<0>(w);
            };
            const uint32_t a0 = part(k0[2 * j]), a1 = part(k1[2 * j]), a2 = part(k0[2 * j + 1]),
                           a3 = part(k1[2 * j + 1]);
            const bool open = j == 0 && (NB == 4 || (k & 1) == 0);  // a block's first product
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              float(&x)[4] = acc[p];
              const uint32_t* q = bq[k * (D / 64) + j][p];
              mma16(x, a0, a1, a2, a3, q[0], q[1], open ? 0.f : x[0], open ? 0.f : x[1], open ? 0.f : x[2],
                    open ? 0.f : x[3]);
            }
          }
          if (NB == 4 || (k & 1)) {
            const int b = k * NB / 4;
            const float2 d = h2f(sc[b]);
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float de = e < 2 ? d.x : d.y;
                s[c][p][e] = b == 0 ? acc[p][e] * de : fmaf(acc[p][e], de, s[c][p][e]);
              }
          }
        }
      }
      // --- the reference and the weights
      bool moved = false;
      float2 top[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        if (MASK) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (base + 16 * c + k_row[e / 2] >= vis[p][e & 1]) s[c][p][e] = -INFINITY;
        }
        top[p].x = fmaxf(fmaxf(s[0][p][0], s[0][p][2]), fmaxf(s[1][p][0], s[1][p][2]));
        top[p].y = fmaxf(fmaxf(s[0][p][1], s[0][p][3]), fmaxf(s[1][p][1], s[1][p][3]));
        moved |= top[p].x > m[p].x || top[p].y > m[p].y;
      }
      if (__any_sync(~0u, moved)) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          float2 f;
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) {
            top[p].x = fmaxf(top[p].x, __shfl_xor_sync(~0u, top[p].x, sh));
            top[p].y = fmaxf(top[p].y, __shfl_xor_sync(~0u, top[p].y, sh));
          }
          // a reference that is passed moves a headroom above the new maximum
          const float nx = top[p].x > m[p].x ? top[p].x + room[p].x : m[p].x;
          const float ny = top[p].y > m[p].y ? top[p].y + room[p].y : m[p].y;
          f.x = nx == m[p].x ? 1.f : m[p].x == -INFINITY ? 0.f : ex2((m[p].x - nx) * cs[p].x);
          f.y = ny == m[p].y ? 1.f : m[p].y == -INFINITY ? 0.f : ex2((m[p].y - ny) * cs[p].y);
          m[p] = make_float2(nx, ny);
          l[p].x *= f.x, l[p].y *= f.y;
#pragma unroll
          for (int v = 0; v < NV; ++v) o[v][p][0] *= f.x, o[v][p][1] *= f.y, o[v][p][2] *= f.x, o[v][p][3] *= f.y;
        }
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const float2 mc = make_float2(m[p].x == -INFINITY ? 0.f : fmaf(-m[p].x, cs[p].x, up),
                                      m[p].y == -INFINITY ? 0.f : fmaf(-m[p].y, cs[p].y, up));
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            float2 w = fma2(make_float2(s[c][p][e], s[c][p][e + 1]), cs[p], mc);
            w.x = ex2(w.x), w.y = ex2(w.y);
            if (MASK) {
              if (base + 16 * c + k_row[e / 2] >= vis[p][0]) w.x = 0.f;
              if (base + 16 * c + k_row[e / 2] >= vis[p][1]) w.y = 0.f;
            }
            s[c][p][e] = w.x, s[c][p][e + 1] = w.y;
            l[p] = add2(l[p], w);
          }
      }
      // --- values, 16 tokens at a time
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t bp[NB][NP][2];
        if constexpr (MASK || !FAST) {
          uint32_t sc[NB];
          if constexpr (NB == 4) *(uint4*)sc = *(const uint4*)(sp + 4 * D + c * D + d_off);
          else *(uint2*)sc = *(const uint2*)(sp + 4 * D + c * D + d_off);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const float2 d = h2f(sc[b]);
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float x = s[c][p][2 * e] * (e ? d.y : d.x), y = s[c][p][2 * e + 1] * (e ? d.y : d.x);
                if (MASK) {  // no scale of a hidden token reaches a sum
                  if (base + 16 * c + k_row[e] >= vis[p][0]) x = 0.f;
                  if (base + 16 * c + k_row[e] >= vis[p][1]) y = 0.f;
                }
                bp[b][p][e] = transpose8(f2h(x, y));
              }
          }
        } else {
          uint32_t x[NB], y[NB], w[NP][2];
          if constexpr (NB == 4) {
            *(uint4*)x = *(const uint4*)(sp + 4 * D + c * D + t_off[0]);
            *(uint4*)y = *(const uint4*)(sp + 4 * D + c * D + t_off[1]);
          } else {
            *(uint2*)x = *(const uint2*)(sp + 4 * D + c * D + t_off[0]);
            *(uint2*)y = *(const uint2*)(sp + 4 * D + c * D + t_off[1]);
          }
#pragma unroll
          for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int e = 0; e < 2; ++e) w[p][e] = transpose8(f2h(s[c][p][2 * e], s[c][p][2 * e + 1]));
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t d = __byte_perm(x[b], y[b], e ? 0x7632 : 0x5410);
#pragma unroll
              for (int p = 0; p < NP; ++p)
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(bp[b][p][e]) : "r"(w[p][e]), "r"(d));
            }
        }
        auto product = [&](int v, int b, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, auto odd) {
          constexpr int O = decltype(odd)::value;
          const uint32_t a0 = codes<O>(r0), a1 = codes<O>(r1), a2 = codes<O>(r2), a3 = codes<O>(r3);
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            float(&x)[4] = o[v][p];
            mma16(x, a0, a1, a2, a3, bp[b][p][0], bp[b][p][1], x[0], x[1], x[2], x[3]);
          }
        };
        using Even = std::integral_constant<int, 0>;
        using Odd = std::integral_constant<int, 1>;
        if constexpr (D == 128) {
          uint2 w[2][2];  // [token of the pair][pair] words 2g (x) and 2g + 1 (y)
#pragma unroll
          for (int h = 0; h < 4; ++h) w[h / 2][h & 1] = *(const uint2*)(kp + c * 8 * D + v_off[h & 1][h / 2]);
#pragma unroll
          for (int by = 0; by < 2; ++by) {  // bytes 2 by, 2 by + 1 of both tokens: nibbles 4 by ..
            const uint32_t sel = by ? 0x7632 : 0x5410;
            const uint32_t r0 = __byte_perm(w[0][0].x, w[0][1].x, sel), r1 = __byte_perm(w[0][0].y, w[0][1].y, sel);
            const uint32_t r2 = __byte_perm(w[1][0].x, w[1][1].x, sel), r3 = __byte_perm(w[1][0].y, w[1][1].y, sel);
            product(4 * by, 0, r0, r1, r2, r3, Even());
            product(4 * by + 1, 1, r0, r1, r2, r3, Odd());
            product(4 * by + 2, NB - 2, r0 >> 8, r1 >> 8, r2 >> 8, r3 >> 8, Even());
            product(4 * by + 3, NB - 1, r0 >> 8, r1 >> 8, r2 >> 8, r3 >> 8, Odd());
          }
        } else {
          uint32_t w[2][2];
#pragma unroll
          for (int h = 0; h < 4; ++h) w[h / 2][h & 1] = *(const uint32_t*)(kp + c * 8 * D + v_off[h & 1][h / 2]);
          // bytes 0, 1: the even nibble of a pair (rows g); bytes 2, 3: the odd one (rows g + 8)
          const uint32_t r0 = __byte_perm(w[0][0], w[0][1], 0x5410), r1 = __byte_perm(w[0][0], w[0][1], 0x7632);
          const uint32_t r2 = __byte_perm(w[1][0], w[1][1], 0x5410), r3 = __byte_perm(w[1][0], w[1][1], 0x7632);
          product(0, 0, r0, r1, r2, r3, Even());
          product(1, 0, r0, r1, r2, r3, Odd());
          product(2, 1, r0 >> 8, r1 >> 8, r2 >> 8, r3 >> 8, Even());
          product(3, 1, r0 >> 8, r1 >> 8, r2 >> 8, r3 >> 8, Odd());
        }
      }
    };

    for (; page < end; ++page) {
      if (!failed && !warp_wait(&s_full[wid][st], phase)) failed = true;
      if (!failed && s_there[wid][st]) {
        const uint8_t* pg = ring + st * PB;
        const int base = page * kKv4Page;
        // --- the page's value scales, one group and scale entry a lane: should
        // one pass the largest so far, the weights come down
        uint32_t vd[NB];
        if constexpr (NB == 4) *(uint4*)vd = *(const uint4*)(pg + 68 * D + lane * 16);
        else *(uint2*)vd = *(const uint2*)(pg + 68 * D + lane * 8);
        uint32_t vt = vd[0] & 0x7fff7fffu;
#pragma unroll
        for (int b = 1; b < NB; ++b) vt = max_pair(vt, vd[b] & 0x7fff7fffu);
        if (__any_sync(~0u, reaches(vt, (uint32_t)(big + 1) * 0x04000400u))) {
          int e = 0;
          const int kv = __ldg(a.kv_len + s_place[wid].z);
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // scales that are not finite reach their sums as they are, and
              // those behind the last token none
              const int x = vd[b] >> (16 * h) & 0x7fff;
              if (x < 0x7c00 && base + 8 * (lane >> 2) + kv4_token(2 * t + h) < kv) e = max(e, x >> 10);
            }
          e = __reduce_max_sync(~0u, e);
          if (e > big) {
            const float to = kv4_up<FAST>(e), f = ex2(to - up);
            big = e, up = to;
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              l[p].x *= f, l[p].y *= f;
#pragma unroll
              for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[v][p][c] *= f;
            }
          }
        }
        // Half pages, in a loop that stays one: with the whole page written out
        // the code is longer, and it is fetched cold (one request of 1100
        // tokens: 14.1 against 14.3 us; 770 MB of pages: 161.6 against 160.9).
        // Pages that every row sees whole have a copy without masks all the
        // same (188 us without it against 174, on a slower GPU).
        if (base + 64 <= first && (!FAST || kv4_short(big))) {
#pragma unroll 1
          for (int h = 0; h < 2; ++h) step(pg + h * 16 * D, pg + 64 * D + h * 2 * D, base + 32 * h, std::false_type());
        } else {
#pragma unroll 1
          for (int h = 0; h < 2; ++h) step(pg + h * 16 * D, pg + 64 * D + h * 2 * D, base + 32 * h, std::true_type());
        }
      }
      __syncwarp();
      if (lane == 0 && i + S < n && !failed) {
        fetch(st, nid);
        if (i + S + 1 < n) {
          forward(src);
          nid = page_id();
        }
      }
      ++i;
      if (++st == S) st = 0, phase ^= 1;
    }

    // --- the row block's sums
    const Kv4Place at = s_place[wid];
    const Kv4Req rq = kv4_req<R>(a, at.z);
    const int hk = at.hk, rb = at.rb, rows = rq.n * G - rb * R;
    const bool all = at.page == 0 && end == at.pages;
    const int slot = 2 * me + (lead ? 0 : 1);
    lead = false;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int sh = 4; sh < 32; sh <<= 1) {
        l[p].x += __shfl_xor_sync(~0u, l[p].x, sh);
        l[p].y += __shfl_xor_sync(~0u, l[p].y, sh);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = p * 8 + 2 * t + e, idx = rb * R + row, j = idx / G;
        const float top = e ? m[p].y : m[p].x;
        const float sum = failed ? __int_as_float(0x7fffffff) : e ? l[p].y : l[p].x;
        if (!all && g == 0) {
          float* ml = a.ml + ((size_t)slot * R + row) * 2;
          ml[0] = top == -INFINITY ? -INFINITY : fmaf(top, e ? cs[p].y : cs[p].x, -up);
          ml[1] = sum;
        }
        const float f = all ? (sum != 0.f ? 1.f / sum : 0.f) : 1.f;
        if (row >= rows) continue;
        T* out = (T*)a.out + ((size_t)(rq.c0 + j) * a.H + hk * G + (idx - j * G)) * D;
        float* part = a.part + ((size_t)slot * R + row) * D;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float y0 = o[v][p][e] * f, y1 = o[v][p][2 + e] * f;
          // dimensions of rows g and g + 8 of the tile
          const int d0 = D == 128 ? (v < 4 ? 2 * v : 2 * v - 7) * 16 + 2 * g : 16 * v + g;
          const int d1 = D == 128 ? d0 + 1 : d0 + 8;
          if (all) {
            out[d0] = from_f<T>(y0);
            out[d1] = from_f<T>(y1);
          } else {
            part[d0] = y0;
            part[d1] = y1;
          }
        }
      }
    }
    // --- the next row block
    __syncwarp();
    if (lane == 0 && i < n) {
      s_place[wid].page = at.pages - 1;
      forward(s_place[wid]);
    }
    __syncwarp();
  }
  if (failed)  // leave no copy in flight behind
    for (int i = 0; i < S; ++i) bar_wait(&s_full[wid][(st + i) % S], (st + i) % S < st ? phase ^ 1 : phase);
}

// Joins the parts of the rows that several warps worked on, in the line's
// order whatever the order in which they came; zeroes rows of no request.
// One block for a token's rows of one key/value head, kJoinWarps / group warps
// to a row: the request in one round of loads, the parts in a second.
constexpr int kJoinWarps = 16;
template <typename T, int D, int NP>
__global__ void __launch_bounds__(32 * kJoinWarps) k_kv4_join(const Kv4Args a) {
  constexpr int R = 8 * NP, V = D / 32;
  __shared__ float s_o[kJoinWarps][D], s_l[kJoinWarps], s_m[kJoinWarps];
  __shared__ Kv4Req s_rq;
  __shared__ long long s_first;
  __shared__ int s_z;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int t = blockIdx.x / a.Hk, hk = blockIdx.x - t * a.Hk, G = a.H / a.Hk;
  if (tid == 0) s_rq.n = 0, s_z = a.B;
  __syncthreads();
  grid_wait();
  const long long L = __ldcg(a.head), N = __ldcg(a.head + 1);
  for (int z0 = 0; z0 < a.B; z0 += 32 * kJoinWarps) {
    const int z = z0 + tid;
    const Kv4Req rq = z < a.B ? kv4_req<R>(a, z) : Kv4Req{0, 0, 0, 0, 0};
    const long long first = z < a.B ? __ldcg(a.head + 2 + z) : 0;
    const bool mine = rq.c0 <= t && t < rq.c0 + rq.n;
    if (mine) atomicMin(&s_z, z);  // should several claim the row, the first has it
    __syncthreads();
    if (mine && s_z == z) s_rq = rq, s_first = first;
  }
  __syncthreads();
  const Kv4Req rq = s_rq;
  T* out = (T*)a.out + ((size_t)t * a.H + (size_t)hk * G) * D;
  if (!rq.n) {
    for (int d = tid; d < G * D; d += 32 * kJoinWarps) out[d] = from_f<T>(0.f);
    return;
  }
  const int per = max(1, kJoinWarps / G), at_once = kJoinWarps / per;  // warps to a row, rows at once
  const int sub = wid % per;
  for (int r0 = 0; r0 < G; r0 += at_once) {
    const int r = r0 + wid / per;
    int n = 0;
    float o[V] = {}, l = 0.f, m = -INFINITY;
    if (wid / per < at_once && r < G) {
      const int idx = (t - rq.c0) * G + r, rb = idx / R, row = idx - rb * R;
      const long long s0 = s_first + ((long long)hk * rq.nb + rb) * rq.pages;
      // the warps whose stretches hold the row block's first and last unit
      const int w0 = (int)line_div((s0 + 1) * N - 1, L);
      n = (int)line_div((s0 + rq.pages) * N - 1, L) - w0 + 1;
      // only the first part can be its warp's second row block
      const int second = (long long)w0 * L >= s0 * N ? 0 : 1;
      auto at = [&](int i) { return (size_t)(2 * (w0 + i) + (i ? 0 : second)) * R + row; };
      if (n > 1) {  // one part was written by its warp
        constexpr int kBatch = 4;  // parts whose loads are under way at once
#pragma unroll 1
        for (int i0 = sub; i0 < n; i0 += kBatch * per) {
          float2 ml[kBatch];
          float x[kBatch][V];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const int i = i0 + k * per;
            ml[k] = make_float2(-INFINITY, 0.f);
            if (i < n) {
              const size_t slot = at(i);
              ml[k] = __ldcg((const float2*)(a.ml + slot * 2));
              if constexpr (V == 4) *(float4*)x[k] = __ldcg((const float4*)(a.part + slot * D) + lane);
              else *(float2*)x[k] = __ldcg((const float2*)(a.part + slot * D) + lane);
            }
          }
          float top = m;
#pragma unroll
          for (int k = 0; k < kBatch; ++k) top = fmaxf(top, ml[k].x);
          const float f0 = m == -INFINITY ? 0.f : ex2(m - top);
          m = top;
          l *= f0;
#pragma unroll
          for (int v = 0; v < V; ++v) o[v] *= f0;
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            // a part without keys has no sum, unless its copies failed
            const float f = ml[k].x == -INFINITY ? 0.f : ex2(ml[k].x - top);
            l += ml[k].y != ml[k].y ? ml[k].y : f * ml[k].y;
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] += f == 0.f ? 0.f : f * x[k][v];
          }
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) s_o[wid][lane * V + v] = o[v];
    if (lane == 0) s_l[wid] = l, s_m[wid] = m;
    __syncthreads();
    if (n > 1 && sub == 0) {
      float all = 0.f, y[V] = {}, top = -INFINITY;
#pragma unroll 1
      for (int w = 0; w < per; ++w) top = fmaxf(top, s_m[wid + w]);
#pragma unroll 1
      for (int w = 0; w < per; ++w) {
        const float f = s_m[wid + w] == -INFINITY ? 0.f : ex2(s_m[wid + w] - top), lw = s_l[wid + w];
        all += lw != lw ? lw : f * lw;
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] += f == 0.f ? 0.f : f * s_o[wid + w][lane * V + v];
      }
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = all != 0.f ? y[v] / all : 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) out[r * D + lane * V + v] = from_f<T>(y[v]);
    }
    __syncthreads();
  }
}

struct Kv4Space {
  size_t head, ml, part, total;
};
static Kv4Space kv4_space(int sms, int B, int rows, int D) {
  const size_t slots = (size_t)2 * sms * (rows == 8 ? kKv4Warps<1> : kKv4Warps<2>);
  Kv4Space s;
  s.head = 0;
  s.ml = ((size_t)(B + 2) * 8 + 127) / 128 * 128;
  s.part = s.ml + slots * rows * 8;
  s.total = s.part + slots * rows * D * 4;
  return s;
}
// Query rows of a block: 16 where a request has more rows (tokens times
// grouped heads) than that on average, else 8, with the twelve warps that its
// registers allow.  Blocks of 8, which dequantize a page once for each 8 rows,
// against 16, at D = 128: 105 and 119 us for 24 requests of 12 rows on
// average, 229 and 203 us for 36 rows.  Blocks of 24 lost to both.
static int kv4_rows(int T, int B, int H, int Hk) {
  return (long long)T * (H / Hk) <= 16ll * std::max(B, 1) ? 8 : 16;
}

template <typename T, int D, int NP>
static cudaError_t run_kv4(const Kv4Args& a, int sms, cudaStream_t s) {
  constexpr size_t smem = kKv4Rings;
  static std::atomic<unsigned long long> ready{0};  // devices whose attribute is set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    e = cudaFuncSetAttribute(k_kv4<T, D, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(1ull << dev, std::memory_order_acq_rel);
  }
  k_kv4<T, D, NP><<<sms, 32 * kKv4Warps<NP>, smem, s>>>(a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)(a.T * a.Hk));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_kv4_join<T, D, NP>, a);
}
template <typename T, int D>
static cudaError_t run_kv4_rows(const Kv4Args& a, int rows, int sms, cudaStream_t s) {
  return rows == 8 ? run_kv4<T, D, 1>(a, sms, s) : run_kv4<T, D, 2>(a, sms, s);
}

}  // namespace mc

using namespace mc;

extern "C" int64_t mc_kv4_attention_workspace(int32_t n_requests, int32_t head_dim, int32_t device) {
  if (n_requests < 0 || (head_dim != 64 && head_dim != 128)) return 0;
  if (paged_check(device) != MC_OK) return 0;
  const int sms = paged_sms(device);
  return (int64_t)std::max(kv4_space(sms, n_requests, 8, head_dim).total,
                           kv4_space(sms, n_requests, 16, head_dim).total);
}

extern "C" mc_status mc_kv4_attention(const mc_kv4_attention_args* args, int32_t device, void* stream) {
  if (!args) return set_error(MC_E_INVALID, "null pointer");
  const void *q = args->q, *pool = args->pool;
  const int32_t *table = args->table, *kv_len = args->kv_len, *cu_q = args->cu_q;
  void *out = args->out, *workspace = args->workspace;
  const int64_t q_tok = args->q_tok, q_head = args->q_head, n_pages = args->n_pages,
                workspace_bytes = args->workspace_bytes;
  const int32_t dtype = args->dtype, n_tokens = args->n_tokens, n_heads = args->n_heads,
                n_kv_heads = args->n_kv_heads, head_dim = args->head_dim, table_width = args->table_width,
                n_requests = args->n_requests;
  const float scale = args->scale;
  if (head_dim != 64 && head_dim != 128) return set_error(MC_E_SHAPE, "head dim must be 64 or 128");
  if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads)
    return set_error(MC_E_SHAPE, "heads must be a multiple of the key/value heads");
  if (dtype != MC_ACT_F16 && dtype != MC_ACT_BF16)
    return set_error(MC_E_DTYPE, "queries must be f16 or bf16");
  if (n_tokens < 0 || n_requests < 0 || table_width < 0 || n_pages < 0)
    return set_error(MC_E_INVALID, "negative size");
  if (n_pages * kKv4Page > 0x7fffffffll || (long long)n_tokens * n_heads > 0x7fffffffll)
    return set_error(MC_E_CAPACITY, "slots or rows pass 31 bits");
  if (!isfinite(scale)) return set_error(MC_E_INVALID, "scale must be finite");
  if (n_tokens == 0) return MC_OK;
  if (!q || !out || !cu_q || !workspace || (n_requests && (!kv_len || (table_width && !table))) ||
      (n_pages && !pool))
    return set_error(MC_E_INVALID, "null pointer");
  if ((n_pages && !aligned(pool, 16)) || !aligned(workspace, 16))
    return set_error(MC_E_INVALID, "pool and workspace must be 16-byte aligned");
  MC_PAGED_DEVICE(device);
  const int sms = paged_sms(device), rows = kv4_rows(n_tokens, n_requests, n_heads, n_kv_heads);
  const Kv4Space sp = kv4_space(sms, n_requests, rows, head_dim);
  if (workspace_bytes < (int64_t)sp.total) return set_error(MC_E_CAPACITY, "workspace too small");
  uint8_t* ws = (uint8_t*)workspace;
  Kv4Args a{q, q_tok, q_head, out, (const uint8_t*)pool, table, kv_len, cu_q, n_tokens, n_heads,
            n_kv_heads, n_requests, table_width, (int)n_pages, scale, (long long*)(ws + sp.head),
            (float*)(ws + sp.ml), (float*)(ws + sp.part)};
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (dtype == MC_ACT_F16)
    e = head_dim == 128 ? run_kv4_rows<__half, 128>(a, rows, sms, s) : run_kv4_rows<__half, 64>(a, rows, sms, s);
  else
    e = head_dim == 128 ? run_kv4_rows<__nv_bfloat16, 128>(a, rows, sms, s)
                        : run_kv4_rows<__nv_bfloat16, 64>(a, rows, sms, s);
  MC_PCK(e);
  return MC_OK;
}
