// mc_prompt_attn.cu -- attention over whole packed prompts.
//
// O = softmax(scale Q K^T) V per sequence and head, one pass over the keys.
// A block takes two tiles of 128 query rows and walks their keys in tiles of
// 128.  The tiles are the same rows of two heads of one key/value head where
// the groups have an even number of heads, so that both have the same keys,
// and 256 rows of one head otherwise (adjacent rows for all: the second tile's
// additional keys under a causal mask leave the first idle, and short
// sequences the second).
//   - one thread loads Q once and K, V tiles through a shared-memory ring
//     (cp.async.bulk.tensor, 128-byte swizzle);
//   - one thread issues tcgen05.mma: S = Q K^T of a tile into tensor memory,
//     and O += P V with P read from tensor memory, where it took the place of
//     S;
//   - two groups of four warps, one per tile, turn S into P: a thread owns a
//     row, so maxima and sums need no exchange.
// While one tile's rows are in the softmax the tensor cores work on the
// other tile.  Scores, statistics and O are f32; P is rounded to the inputs'
// type (11 bits from f16, 8 from bf16).  The reference of the exponentials follows the running maximum only
// when that has grown by more than 2^8: O is then rescaled in tensor memory.
#include <cuda.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mc_paged.cuh"

namespace mc {

constexpr int kPromptRows = 128;  // rows of a query tile, keys of a key tile
constexpr int kPromptThreads = 384;
// Barriers of the rounds of products: round 0 is the first scores, round j + 1
// the values j and the scores j + 1.  The loads run at most Slots / 2 rounds
// ahead of the round that they wait for, so with more barriers than that no
// barrier is two phases ahead of a waiting load.
constexpr int kPromptRounds = 8;
constexpr float kPromptGrow = 8.f;  // log2 growth of the maximum that is let pass
// Weights of f16 inputs are 2^7 larger, so that they reach 2^15 at most and keep
// their 11 bits down to 2^-21 of the first reference: without it the small ones
// of a row whose mass one key takes were subnormal.
template <typename T>
constexpr float kPromptUp = std::is_same<T, __half>::value ? 7.f : 0.f;

struct PromptArgs {
  const void *q, *k, *v;  // [Tq][H][D], [Tk][Hk][D] with strides (elements)
  long long q_tok, q_head, k_tok, k_head, v_tok, v_head;
  void* out;              // [Tq][H][D]
  const int *cu_q, *cu_k;
  int Tq, Tk, H, Hk, B, causal;
  int pair, rows, units;  // tiles of two heads; rows of a block; blocks over the same rows
  float scale;
};

template <int D>
struct PromptCfg {
  static constexpr int Tile = kPromptRows * D * 2;         // bytes of a Q, K or V tile
  static constexpr int Half = kPromptRows * 128;           // of 64 of its columns
  static constexpr int Slots = D == 128 ? 5 : 10;          // K and V tiles in the ring
  static constexpr int Smem = (2 + Slots) * Tile + 1024;   // + alignment to the swizzle atoms
  static constexpr uint32_t O = 256;                       // tensor memory columns: S 0, S 1, O 0, O 1
};

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t pred;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(pred));
  return pred;
}
// 64 columns x 128 rows at (column x, head h, token t)
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* m, int x, int h, int t, uint64_t* b) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(sm_ptr(dst)),
      "l"(m), "r"(x), "r"(h), "r"(t), "r"(sm_ptr(b))
      : "memory");
}
// Shared-memory descriptors: the low word has the start address and the
// leading byte offset, the high word the stride (8 rows of 128 bytes), the
// version 1 and the 128-byte swizzle; offsets count 16 bytes.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
  return ((addr >> 4) & 0x3FFF) | ((lbo >> 4) << 16);
}
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
// The products are issued by the lane whose `one` is set.  All lanes run the
// code around them, so that its values stay in uniform registers: with one
// lane inside a branch each product waited for its operands to be moved there.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 a, {%1, %6};\n\tmov.b64 b, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(one), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 b, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(one), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* b, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(sm_ptr(b)),
      "r"(one)
      : "memory");
}
#define MC_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define MC_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of the warp's 32 lanes
__device__ __forceinline__ void tm_load(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : MC_R8(r, 0), MC_R8(r, 8), MC_R8(r, 16), MC_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tm_store(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::MC_I8(r, 0),
      MC_I8(r, 8), MC_I8(r, 16), MC_I8(r, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  uint32_t x;
  memcpy(&x, &h, 4);
  return x;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  uint32_t x;
  memcpy(&x, &h, 4);
  return x;
}

// One copy of the polling loop for the waits of the loading and the issuing
// thread, so that the code between them is short.
__device__ __noinline__ bool bar_poll(uint32_t b, uint32_t parity) { return bar_loop(b, parity); }
__device__ __forceinline__ bool bar_wait_far(uint64_t* b, uint32_t parity) {
  return bar_try(b, parity) || bar_poll(sm_ptr(b), parity);
}

struct PromptWork {
  int q0, n_q;     // first query row of the block and how many the sequence has from there
  int k0, L;       // first key, keys
  int shift;       // row i of the block sees the keys below i + shift (causal)
  int ok;          // there is work
};

// The block's rows: tiles are counted over the sequences, the last ones
// first, since under a causal mask they have the most keys.  One warp.
__device__ __forceinline__ void prompt_work(const PromptArgs& a, int index, PromptWork* w) {
  const int lane = threadIdx.x & 31;
  // the sequences from the last one down, 32 at a time; all four bounds are
  // read at once, since this load's latency is most of a short block's start
  int seen = 0;
  if (lane == 0) w->ok = 0;
  __syncwarp();
  for (int z1 = a.B; z1 > 0 && seen <= index; z1 -= 32) {
    const int z = z1 - 1 - lane;
    int c0 = 0, n = 0, k0 = 0, k1 = 0;
    if (z >= 0) c0 = a.cu_q[z], n = a.cu_q[z + 1], k0 = a.cu_k[z], k1 = a.cu_k[z + 1];
    const int keys = k1 - k0;
    c0 = min(max(c0, 0), a.Tq);
    n = max(min(n, a.Tq) - c0, 0);
    k0 = min(max(k0, 0), a.Tk);
    k1 = max(min(k1, a.Tk), k0);
    const int mine = (n + a.rows - 1) / a.rows;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, inc, o);
      if (lane >= o) inc += x;
    }
    const int last = seen + inc - 1;  // the sequence's tiles are last - mine + 1 .. last, its last tile first
    if (index <= last && index > last - mine) {
      const int r = (last - index) * a.rows;
      w->q0 = c0 + r;
      w->n_q = n - r;
      w->k0 = k0;
      w->L = k1 - k0;
      w->shift = a.causal ? keys - n + r + 1 : 1 << 30;
      w->ok = 1;
    }
    seen += __shfl_sync(~0u, inc, 31);
  }
  __syncwarp();
}

// The last key in [from, to) of the sequence at k0 whose V row holds a NaN or an
// infinity, or -1.  A row whose result is not finite has it from the keys that
// it sees, and then it is right, or from one of these behind them: the product
// of a hidden key's weight 0 with its NaN or infinity is not 0.
template <typename T, int D>
__device__ __noinline__ int prompt_last_bad(const PromptArgs& a, int h, int k0, int from, int to) {
  constexpr uint32_t kTop = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;  // exponents of those
  const int lane = threadIdx.x & 31, x = lane % (D / 8);
  const T* vp = (const T*)a.v + h / (a.H / a.Hk) * a.v_head + x * 8;
  int last = -1;
#pragma unroll 4
  for (int j = from + lane / (D / 8); j < to; j += 256 / D) {
    const uint4 y = *(const uint4*)(vp + (long long)(k0 + j) * a.v_tok);
    const uint32_t w[4] = {y.x, y.y, y.z, y.w};
    for (int i = 0; i < 4; ++i)
      if ((w[i] & kTop) == kTop || (w[i] >> 16 & kTop) == kTop) last = j;
  }
  return __reduce_max_sync(~0u, last);
}

// One row again, with a lane per key and then per column, over its own keys
// alone: for rows that a hidden key spoiled.
template <typename T, int D>
__device__ __noinline__ void prompt_row(const PromptArgs& a, int t, int h, int k0, int n) {
  constexpr int NB = D / 32;
  const int lane = threadIdx.x & 31;
  const T* q = (const T*)a.q + t * a.q_tok + h * a.q_head;
  const int hk = h / (a.H / a.Hk);
  const T* kp = (const T*)a.k + hk * a.k_head;
  const T* vp = (const T*)a.v + hk * a.v_head;
  float o[NB] = {}, m = -INFINITY, l = 0.f;
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    float x = -INFINITY;
    if (j < n) {
      const T* k = kp + (long long)(k0 + j) * a.k_tok;
      x = 0.f;
#pragma unroll 4
      for (int i = 0; i < D; i += 8) {
        const uint4 kk = *(const uint4*)(k + i), qq = *(const uint4*)(q + i);
        const T *ke = (const T*)&kk, *qe = (const T*)&qq;
#pragma unroll
        for (int e = 0; e < 8; ++e) x += to_f(ke[e]) * to_f(qe[e]);
      }
      x *= a.scale;
    }
    float top = x;
    for (int f = 16; f; f >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, f));
    const float mn = fmaxf(m, top);
    const float c = m == -INFINITY ? 0.f : __expf(m - mn);
    const float e = x > -INFINITY ? __expf(x - mn) : (x != x ? x : 0.f);
    m = mn;
    l = l * c + e;
    for (int b = 0; b < NB; ++b) o[b] *= c;
#pragma unroll 4
    for (int i = 0; i < min(32, n - j0); ++i) {
      const float p = __shfl_sync(~0u, e, i);
      const T* v = vp + (long long)(k0 + j0 + i) * a.v_tok;
      for (int b = 0; b < NB; ++b) o[b] += p * to_f(v[b * 32 + lane]);
    }
    // nothing that follows changes a row that is NaN in every column
    bool settled = true;
    for (int b = 0; b < NB; ++b) settled = settled && o[b] != o[b];
    if (__all_sync(~0u, settled)) break;
  }
  for (int f = 16; f; f >>= 1) l += __shfl_xor_sync(~0u, l, f);
  T* out = (T*)a.out + ((size_t)t * a.H + h) * D;
  for (int b = 0; b < NB; ++b) out[b * 32 + lane] = from_f<T>(l != 0.f ? o[b] / l : 0.f);
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
    k_prompt(const PromptArgs a, const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
             const __grid_constant__ CUtensorMap mv) {
  using C = PromptCfg<D>;
  constexpr int NH = D / 64;  // 64-column halves of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (sm_ptr(smem_raw) & 1023u)) & 1023u);
  uint8_t *sq = smem, *ring = smem + 2 * C::Tile;
  __shared__ __align__(8) uint64_t b_q[2], b_full[C::Slots], b_round[kPromptRounds], b_s[2], b_p[2][2], b_pv[2],
      b_tail, b_fix;
  __shared__ uint32_t s_tmem;
  __shared__ int s_fail;
  __shared__ PromptWork s_work;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int index = blockIdx.x / a.units, unit = blockIdx.x % a.units;
  // tile t has the rows from t * row_1 of head + t * pair
  const int head = a.pair ? 2 * unit : unit, row_1 = a.pair ? 0 : kPromptRows;

  // the start, spread over warps: the work, the barriers, tensor memory (this
  // block is alone on its SM), and clearing the rows of no sequence
  if (warp == 0) {
    prompt_work(a, index, &s_work);
  } else if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_ptr(&s_tmem)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tid == 32) {
    for (int i = 0; i < C::Slots; ++i) bar_init(&b_full[i], 1);
    for (int i = 0; i < kPromptRounds; ++i) bar_init(&b_round[i], 1);
    for (int i = 0; i < 2; ++i) {
      bar_init(&b_q[i], 1), bar_init(&b_s[i], 1), bar_init(&b_pv[i], 1);
      bar_init(&b_p[i][0], 4), bar_init(&b_p[i][1], 4);
    }
    bar_init(&b_tail, 1), bar_init(&b_fix, 1);
    s_fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  } else if (tid == 288) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  } else if (warp >= 10) {
    const int start = min(max(a.cu_q[0], 0), a.Tq), end = min(max(a.cu_q[a.B], start), a.Tq);
    const long long row = (long long)a.H * (D / 8), front = start * row, n = front + (a.Tq - end) * row;
    uint4* z = (uint4*)a.out;
    for (long long i = (long long)blockIdx.x * 64 + tid - 320; i < n; i += (long long)gridDim.x * 64)
      z[i < front ? i : i - front + end * row] = make_uint4(0, 0, 0, 0);
  }
  tm_before();
  __syncthreads();
  tm_after();
  if (!s_work.ok) {
    if (warp == 8)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(512u) : "memory");
    return;
  }
  const uint32_t tmem = s_tmem;
  const PromptWork w = s_work;
  const int hk = head / (a.H / a.Hk);
  // keys that the last row of a tile sees, and its key tiles
  int lim[2], n_t[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int rows = min(max(w.n_q - t * row_1, 0), kPromptRows);
    lim[t] = rows ? min(max(t * row_1 + rows - 1 + w.shift, 0), w.L) : 0;
    n_t[t] = (lim[t] + kPromptRows - 1) / kPromptRows;
  }
  const int n_max = max(n_t[0], n_t[1]);
  // keys of the last key tile, where the sequence or the mask ends inside it
  const int tail = max(lim[0], lim[1]) - (n_max - 1) * kPromptRows;
  const bool fix = n_max > 0 && tail % 16 != 0;

  // Of the block's 384 x 168 registers the softmax's two groups of warps take
  // 216 a thread and the third group keeps 72: 256 x 216 + 128 x 72 is the same.
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 9) {
    // ----------------------------------------------------------- loads
    if (n_max > 0 && elect_one()) {
      auto load_k = [&](int i) {  // K 0, V 0, K 1, V 1, ...
        const int slot = i % C::Slots;
        bar_expect(&b_full[slot], C::Tile);
        for (int h = 0; h < NH; ++h)
          load_tile(ring + slot * C::Tile + h * C::Half, i & 1 ? &mv : &mk, h * 64, hk, w.k0 + (i >> 1) * kPromptRows,
                    &b_full[slot]);
      };
      for (int t = 0; t < 2; ++t) {
        if (n_t[t]) {
          bar_expect(&b_q[t], C::Tile);
          for (int h = 0; h < NH; ++h)
            load_tile(sq + t * C::Tile + h * C::Half, &mq, h * 64, head + t * a.pair,
                      w.q0 + t * row_1, &b_q[t]);
        }
        if (t == 0) load_k(0);
      }
      for (int i = 1; i < 2 * n_max; ++i) {
        // the slot's last tile was number i - Slots: K j is read in round j, V j in round j + 1
        const int last = i - C::Slots, round = (last + 1) >> 1;
        if (last >= 0 && !bar_wait_far(&b_round[round % kPromptRounds], (round / kPromptRounds) & 1)) {
          s_fail = 1;
          break;
        }
        load_k(i);
      }
    }
  } else if (warp == 10) {
    // The last V tile's rows behind the last key, as far as a product's 16
    // keys reach, become 0: what lies there is not this sequence's.
    if (fix) {
      const int i = 2 * n_max - 1, slot = i % C::Slots;
      // b_tail first: only then is the slot's last use the one whose parity is waited for
      if (warp_wait(&b_tail, 0) && warp_wait(&b_full[slot], (i / C::Slots) & 1)) {
        for (int r = tail; r < (tail + 15) / 16 * 16; ++r)
          for (int x = lane; x < NH * 8; x += 32)
            *(uint4*)(ring + slot * C::Tile + (x / 8) * C::Half + r * 128 + (x % 8) * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) bar_arrive(&b_fix);
      } else {
        s_fail = 1;
      }
    }
  } else if (warp == 8) {
    // -------------------------------------------------------- products
    if (n_max > 0) {
      // f32 accumulator; type of A and B; B of P V has its columns contiguous; N; M
      constexpr uint32_t F = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      const uint32_t id_s = (1u << 4) | (F << 7) | (F << 10) | ((a.scale < 0.f ? 1u : 0u) << 13) |
                            ((uint32_t)(kPromptRows >> 3) << 17) | ((uint32_t)(kPromptRows >> 4) << 24);
      const uint32_t id_o = (1u << 4) | (F << 7) | (F << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
                            ((uint32_t)(kPromptRows >> 4) << 24);
      const uint32_t one = elect_one();
      const uint32_t d_q = desc_lo(sm_ptr(sq), 16), d_k = desc_lo(sm_ptr(ring), 16), d_v = desc_lo(sm_ptr(ring), C::Half);
      auto scores = [&](int t, int slot) {
        const uint32_t da = d_q + t * (C::Tile >> 4), db = d_k + slot * (C::Tile >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k % 4) * 2 + (k / 4) * (C::Half >> 4);
          mma_ss(tmem + t * 128, da + off, db + off, id_s, k > 0, one);
        }
        mma_commit(&b_s[t], one);
      };
      bool ok = bar_wait(&b_full[0], 0);
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (n_t[t]) {
          ok &= bar_wait(&b_q[t], 0);
          tm_after();
          scores(t, 0);
        }
      mma_commit(&b_round[0], one);
      int vs = 1, ks = 2, vp = 0, kp = 0;  // slots of V j and K j + 1, their parities
#pragma unroll 1
      for (int j = 0; j < n_max && ok; ++j) {
        const bool more = j + 1 < n_max;
        ok = bar_wait(&b_full[vs], vp);
        if (more) ok &= bar_wait(&b_full[ks], kp);
        if (!more && fix) {
          if (one) bar_arrive(&b_tail);
          __syncwarp();
          ok &= bar_wait(&b_fix, 0);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j >= n_t[t]) continue;
          const int steps = min(8, (lim[t] - j * kPromptRows + 15) / 16);
          const uint32_t db = d_v + vs * (C::Tile >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // the halves of P
            ok &= bar_wait(&b_p[t][h], j & 1);
            tm_after();
#pragma unroll
            for (int k = 4 * h; k < 4 * h + 4; ++k)
              mma_ts(tmem + C::O + t * D, tmem + t * 128 + k * 8, db + k * (2048 >> 4), id_o, j > 0 || k > 0,
                     k < steps ? one : 0);
          }
          // the scores' commit stands for the values before them too
          if (j + 1 < n_t[t]) scores(t, ks);
          else mma_commit(&b_pv[t], one);
        }
        if (more) mma_commit(&b_round[(j + 1) % kPromptRounds], one);
        if ((vs += 2) >= C::Slots) vs -= C::Slots, vp ^= 1;
        if ((ks += 2) >= C::Slots) ks -= C::Slots, kp ^= 1;
        ok = __all_sync(~0u, ok);
      }
      if (!ok && one) s_fail = 1;
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // --------------------------------------------------------- softmax
    const int t = warp >> 2, first = t * row_1 + (warp & 3) * 32, row = first + lane, head_t = head + t * a.pair;
    const uint32_t base = tmem + ((uint32_t)(warp & 3) << 21);  // the warp's 32 lanes
    const uint32_t ts = base + t * 128, to = base + C::O + t * D;
    const int n = n_t[t];
    // keys of this row; rows past the sequence go with its last one
    const int see = min(max(min(row, w.n_q - 1) + w.shift, 0), w.L);
    const float c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = ok && warp_wait(&b_s[t], j & 1);
      if (!ok) break;
      tm_after();
      uint32_t s[128];
#pragma unroll
      for (int i = 0; i < 4; ++i) tm_load(ts + i * 32, s + i * 32);
      tm_wait_ld();
      const int left = see - j * kPromptRows;  // visible columns
      if (!__all_sync(~0u, left >= kPromptRows)) {
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = i < left ? s[i] : 0xff800000u;
      }
      float top4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) top4[i] = __uint_as_float(s[i]);
#pragma unroll
      for (int i = 4; i < 128; ++i) top4[i & 3] = fmaxf(top4[i & 3], __uint_as_float(s[i]));
      const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
      const bool grown = (top - m) * c > kPromptGrow;  // also from -inf
      if (__any_sync(~0u, grown)) {
        const float mn = grown ? top : m;
        if (j > 0) {  // rescale O: the products before these scores are in it
          const float f = mn == m ? 1.f : m == -INFINITY ? 0.f : ex2((m - mn) * c);
          l *= f;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t o[32];
            tm_load(to + i * 32, o);
            tm_wait_ld();
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
            tm_store(to + i * 32, o);
          }
        }
        m = mn;
      }
      const float mc = m == -INFINITY ? 0.f : fmaf(m, c, -kPromptUp<T>);
      float2 sum[2] = {};
      // (a cubic on the f32 pipes for a part of the exponentials was measured
      // slower, 936 against 977 TFLOP/s: the special function unit is not
      // what a tile waits for)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t p[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          float2 e = fma2(make_float2(__uint_as_float(s[i * 64 + 2 * x]), __uint_as_float(s[i * 64 + 2 * x + 1])),
                          make_float2(c, c), make_float2(-mc, -mc));
          e.x = ex2(e.x), e.y = ex2(e.y);
          sum[x & 1] = add2(sum[x & 1], e);
          p[x] = pack2<T>(e.x, e.y);
        }
        tm_store(ts + i * 32, p);
        tm_wait_st();
        tm_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&b_p[t][i]);
      }
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    }
    // ------------------------------------------------------- the result
    if (n > 0) ok = ok && warp_wait(&b_pv[t], 0);
    if (!ok) s_fail = 1;
    tm_after();
    const float f = l != 0.f ? 1.f / l : 0.f;
    const bool live = row < w.n_q;
    bool bad = false;
    if (n > 0 && ok) {
      // the warp's rows go through its part of the tile's queries, which the
      // products no longer read, so that whole rows are written at once
      uint8_t* stage = sq + t * C::Tile + (warp & 3) * 32 * D * 2;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        uint32_t o[32], y[16];
        tm_load(to + i * 32, o);
        tm_wait_ld();
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float y0 = __uint_as_float(o[2 * x]) * f, y1 = __uint_as_float(o[2 * x + 1]) * f;
          bad |= !(fabsf(y0) <= 3e38f) || !(fabsf(y1) <= 3e38f);
          y[x] = pack2<T>(y0, y1);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
          *(uint4*)(stage + lane * D * 2 + (((i * 4 + x) ^ lane) % (D / 8)) * 16) =
              make_uint4(y[4 * x], y[4 * x + 1], y[4 * x + 2], y[4 * x + 3]);
      }
      __syncwarp();
#pragma unroll 4
      for (int i = lane; i < 32 * (D / 8); i += 32) {
        const int r = i / (D / 8), x = i % (D / 8);
        if (first + r < w.n_q)
          *(uint4*)((T*)a.out + ((size_t)(w.q0 + first + r) * a.H + head_t) * D + x * 8) =
              *(const uint4*)(stage + r * D * 2 + ((x ^ r) % (D / 8)) * 16);
      }
    } else if (live) {  // no keys; or a wait ran out
      T* out = (T*)a.out + ((size_t)(w.q0 + row) * a.H + head_t) * D;
      const uint32_t y = ok ? 0u : 0x7fff7fffu;
      for (int x = 0; x < D / 8; ++x) *(uint4*)(out + x * 8) = make_uint4(y, y, y, y);
    }
    __syncwarp();
    unsigned again = __ballot_sync(~0u, bad && live);
    if (again) {
      // the products reached whole groups of 16 keys; `see` grows along the rows
      const int last = prompt_last_bad<T, D>(a, head_t, w.k0, __shfl_sync(~0u, see, __ffs(again) - 1),
                                             min((lim[t] + 15) / 16 * 16, w.L));
      again &= __ballot_sync(~0u, last >= see);
    }
    for (; again; again &= again - 1) {
      const int r = __ffs(again) - 1;
      prompt_row<T, D>(a, w.q0 + first + r, head_t, w.k0, __shfl_sync(~0u, see, r));
    }
    tm_before();
  }
  __syncthreads();
  if (s_fail && warp == 9) {  // leave no copy in flight
    for (int t = 0; t < 2; ++t)
      if (n_t[t]) warp_wait(&b_q[t], 0);
    for (int i = max(0, 2 * n_max - C::Slots); i < 2 * n_max; ++i) warp_wait(&b_full[i % C::Slots], (i / C::Slots) & 1);
  }
  if (warp == 8) {
    tm_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------- host side
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
  static std::atomic<EncodeTiled> fn{nullptr};
  EncodeTiled f = fn.load(std::memory_order_acquire);
  if (!f) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess &&
        r == cudaDriverEntryPointSuccess)
      fn.store(f = (EncodeTiled)p, std::memory_order_release);
  }
  return f;
}
// boxes of 64 columns x 1 head x 128 tokens of [n][heads][D]
static bool head_map(CUtensorMap* m, bool bf16, const void* p, int D, int heads, int n, long long tok, long long head) {
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)n};
  const cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)tok * 2};
  const cuuint32_t box[3] = {64, 1, kPromptRows}, step[3] = {1, 1, 1};
  EncodeTiled f = encode_tiled();
  return f && f(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void*)p, dims,
                strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <typename T, int D>
static cudaError_t run_prompt(const PromptArgs& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                              unsigned grid, cudaStream_t s) {
  static std::atomic<unsigned long long> ready{0};  // devices whose attribute is set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    e = cudaFuncSetAttribute(k_prompt<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptCfg<D>::Smem);
    if (e != cudaSuccess) return e;
    ready.fetch_or(1ull << dev, std::memory_order_acq_rel);
  }
  k_prompt<T, D><<<grid, kPromptThreads, PromptCfg<D>::Smem, s>>>(a, q, k, v);
  return cudaGetLastError();
}

}  // namespace mc

using namespace mc;

extern "C" mc_status mc_prompt_attention(const mc_prompt_args* args, int32_t device, void* stream) {
  if (!args) return set_error(MC_E_INVALID, "null pointer");
  const void *q = args->q, *k = args->k, *v = args->v;
  const int32_t *cu_q = args->cu_q, *cu_k = args->cu_k;
  void *out = args->out;
  const int64_t q_tok = args->q_tok, q_head = args->q_head, k_tok = args->k_tok, k_head = args->k_head,
                v_tok = args->v_tok, v_head = args->v_head;
  const int32_t dtype = args->dtype, n_q = args->n_q, n_k = args->n_k, n_heads = args->n_heads,
                n_kv_heads = args->n_kv_heads, head_dim = args->head_dim, n_sequences = args->n_sequences,
                causal = args->causal;
  const float scale = args->scale;
  if (head_dim != 64 && head_dim != 128) return set_error(MC_E_SHAPE, "head dim must be 64 or 128");
  if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads)
    return set_error(MC_E_SHAPE, "heads must be a multiple of the key/value heads");
  if (dtype != MC_ACT_F16 && dtype != MC_ACT_BF16)
    return set_error(MC_E_DTYPE, "inputs must be f16 or bf16");
  if (n_q < 0 || n_k < 0 || n_sequences < 0) return set_error(MC_E_INVALID, "negative size");
  if (!isfinite(scale)) return set_error(MC_E_INVALID, "scale must be finite");
  if (n_q == 0) return MC_OK;
  if (!q || !out || !cu_q || !cu_k || (n_k && (!k || !v))) return set_error(MC_E_INVALID, "null pointer");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) ||
      (q_tok | q_head | k_tok | k_head | v_tok | v_head) % 8)
    return set_error(MC_E_INVALID, "rows must be 16-byte aligned");
  if (q_tok < 0 || q_head < 0 || k_tok < 0 || k_head < 0 || v_tok < 0 || v_head < 0)
    return set_error(MC_E_INVALID, "negative stride");
  const int pair = n_heads / n_kv_heads % 2 == 0, rows = pair ? kPromptRows : 2 * kPromptRows;
  const int units = pair ? n_heads / 2 : n_heads;
  const long long blocks = (((long long)n_q + rows - 1) / rows + n_sequences) * units;
  if (blocks > 0x7fffffffll || n_q > 0x7fffff00 || n_k > 0x7fffff00)
    return set_error(MC_E_CAPACITY, "too many rows for one call");
  MC_PAGED_DEVICE(device);
  cudaStream_t s = (cudaStream_t)stream;
  if (n_k == 0 || n_sequences == 0) {  // no row sees a key
    MC_PCK(cudaMemsetAsync(out, 0, (size_t)n_q * n_heads * head_dim * 2, s));
    return MC_OK;
  }
  PromptArgs a{q, k, v, q_tok, q_head, k_tok, k_head, v_tok, v_head, out, cu_q, cu_k, n_q, n_k,
               n_heads, n_kv_heads, n_sequences, causal, pair, rows, units, scale};
  CUtensorMap mq, mk, mv;
  const bool bf = dtype == MC_ACT_BF16;
  if (!head_map(&mq, bf, q, head_dim, n_heads, n_q, q_tok, q_head) ||
      !head_map(&mk, bf, k, head_dim, n_kv_heads, n_k, k_tok, k_head) ||
      !head_map(&mv, bf, v, head_dim, n_kv_heads, n_k, v_tok, v_head))
    return set_error(MC_E_CUDA, "the driver refused a tensor map of these strides");
  cudaError_t e;
  if (bf)
    e = head_dim == 128 ? run_prompt<__nv_bfloat16, 128>(a, mq, mk, mv, (unsigned)blocks, s)
                        : run_prompt<__nv_bfloat16, 64>(a, mq, mk, mv, (unsigned)blocks, s);
  else
    e = head_dim == 128 ? run_prompt<__half, 128>(a, mq, mk, mv, (unsigned)blocks, s)
                        : run_prompt<__half, 64>(a, mq, mk, mv, (unsigned)blocks, s);
  MC_PCK(e);
  return MC_OK;
}
