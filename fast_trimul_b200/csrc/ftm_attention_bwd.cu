// Attention backward (sm_100a). With p the forward's weights, recomputed tile by tile from the
// row maximum and sum it kept, g the output's gradient and d = rowsum(g * o):
//
//   dv = p^T g,   dp = g v^T,   ds = p (dp - d),   dq = scale ds k,   dk = scale ds^T q,
//   dbias = sum over the rows that share it of ds.
//
// Three kernels on the same scheme -- two products into TMEM, the elementwise part in
// registers, a 16-bit operand back into TMEM for the accumulating products:
//   dq     one query tile, loop over its key tiles:    S, dP -> dS;   dQ += dS K
//   dkv    one key tile, loop over its query tiles:    S^T, dP^T -> P^T, dS^T;
//          dV += P^T dO, dK += dS^T Q; with grouped heads the loop covers the whole group
//   dbias  one tile of the bias, loop over the rows that share it, sums in registers (a bias of
//          one row alone: dq writes dS along)
// Each result has one owner, so there are no atomics and a call gives the same bits every
// time, at the price of forming S and dP twice (7 products instead of 5). fp32 everywhere
// but the 16-bit operands P and dS, rounded once like the inputs of any product here.
//
// Roles: warps 0-15 elementwise (four per TMEM lane quarter, 32 of the columns each), warp 16
// TMA (and, in dkv, the per-query constants), warp 17 MMA. The elementwise part is the long
// one, and bound by latency: with 8 warps it took 3450 clocks of a dkv tile's 3800 at dim 128
// (the products take 2048); with 16 a tile takes 3700, in dq 3150 (of 1536). What is left is
// the way round: product, elementwise part, product, each handing over through a barrier.
// Issuing the products of a step together, with everything waited for before, took 2 % off dkv
// and put as much on dq and the small sizes, so they stand one by one. All 512 TMEM columns, one
// block per SM: dq holds S twice (the next tile's scores are formed under this one's
// elementwise part), dkv holds S^T, dP^T, dV, dK.
//
// A sequence of 8192 tokens, causal, 16 heads on 4, dim 128, bf16: dq 440 us, dkv 694 us
// (935 and 790 TFLOP/s over the products they form; one large product reaches 1700). 20 us of
// dkv's are the barriers that vote on expired waits; two buffers for the next item's Q and g, or
// K and V, and finding that item under the last product gave 3 us of 331 at N = 250 and cost as
// much at dim 128, so they are not there.
#include <climits>

#include "ftm_attention.cuh"

namespace ftm {
namespace {

enum : int { KERNEL_DQ = 5, KERNEL_DKV = 6, KERNEL_DBIAS = 7 };
constexpr int kBwdThreads = 576;
constexpr int kTmaWarp = 16, kMmaWarp = 17, kElemWarps = 16;

// fp16 has 11 bits from 2^-14 to 65504 and loses them below. dS is about |g| / keys, and the weights
// of many keys are as small, so in fp16 both are formed times a power of two that the stores take
// out again; it enters exponents and constants that are there anyway. Weights are at most 1 (1.02
// where a bias puts the scores far from 0): P^T of dkv times 2^14. |dp - d| <= |g| (|v| + |o|), and o
// is a mean of rows of V: times 2^lift(|g|, largest |v|), |.| the norm of a row, dS stays below
// 2^15.1. dq takes each row's own |g|; dkv, whose sums run over queries, the largest of the call,
// which leaves dS of evenly spread weights 13 binades above 2^-14 at 4096 keys: queries whose
// gradients are more than 2^13 below the largest, or beside one outlier of V, give up bits of dk
// again. 4096 keys, dim 64: dq was off by 2.8 times the rounding of the result at gradients of 1e-2
// and by 8 at 1e-3, now by 1.42 and 1.05 (there the result itself is subnormal). bf16 has the
// exponents of fp32 and needs none of this. It costs fp16 3 to 4 % of a step (ragged batch of 8192
// rows, 12 heads on 6 of 64: 289 -> 300 us; one sequence of 8192, 16 on 4 of 128: 1550 -> 1586).
constexpr int kLiftP = 14;
template <typename T>
constexpr bool kLift = !IsBf16<T>::v;
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ int lift(float g, float v) {
  const float x = g * v;      // 2^k <= x < 2^(k + 1), so 2.02 x < 2^(k + 2.1)
  const int k = (__float_as_int(x) >> 23) - 127;
  return x > 0.f && x < 1e38f ? min(13 - k, 60) : 0;      // (rows that are not finite: nothing to keep)
}
// the largest row norms of g and v, from the delta kernel's parts; all threads of the block, red: two
// words of shared memory that are 0
__device__ __forceinline__ float2 largest_norms(const AttnArgs& a, int* red) {
  float g = 0.f, v = 0.f;
  for (int i = threadIdx.x; i < a.norm_parts; i += blockDim.x) {
    g = fmaxf(g, a.norms[i].x);
    v = fmaxf(v, a.norms[i].y);
  }
  const uint32_t wg = __reduce_max_sync(0xffffffffu, __float_as_uint(g));   // not negative: ordered like
  const uint32_t wv = __reduce_max_sync(0xffffffffu, __float_as_uint(v));   // their bits
  if ((threadIdx.x & 31) == 0) {
    atomicMax(red, static_cast<int>(wg));
    atomicMax(red + 1, static_cast<int>(wv));
  }
  __syncthreads();
  return make_float2(__int_as_float(red[0]), __int_as_float(red[1]));
}

// first and behind-last row that belong to a sequence
__device__ __forceinline__ void rows_inside(const AttnArgs& a, const int* cu, int rows, int& lo, int& hi) {
  lo = cu ? min(max(cu[0], 0), rows) : 0;
  hi = cu ? min(max(cu[a.seqs], lo), rows) : rows;
}

// bstats[head][row], so that a tile's are read in whole lines: without a bias
// x = m c + log2(l) with c = scale log2(e), so that p = 2^(c s - x); with one x = m, y = log2(l), p = 2^((t - x) log2(e) - y), which stays
// exact for scores near the type's lowest value. z = rowsum(g * o). A row without keys has
// log2(l) = inf, hence p = 0. In fp16 w = |g| of the row, and the block's largest norms of g and v
// go to `norms`; masked keys and rows of no sequence, which may hold anything, do not count.
template <typename T>
__global__ void __launch_bounds__(256)
attn_delta_kernel(const __grid_constant__ AttnArgs a, int lanes, int bias) {
  grid_dep_wait();
  const long long n = static_cast<long long>(a.q_rows) * a.heads;
  const int per = blockDim.x / lanes, l = threadIdx.x % lanes;
  const float c = log2_scale(a.scale);
  float top_g = 0.f, top_v = 0.f;
  int lo = 0, hi = 0;
  if (kLift<T>) rows_inside(a, a.cu_q, a.q_rows, lo, hi);
  // the bound is the same for all threads of a warp: the sums below exchange lanes
  for (long long i0 = static_cast<long long>(blockIdx.x) * per; i0 < n; i0 += static_cast<long long>(gridDim.x) * per) {
    const long long i = i0 + threadIdx.x / lanes;
    float s = 0.f, gg = 0.f;
    if (i < n && l * 8 < a.dim) {
      const long long row = i / a.heads;
      const int head = static_cast<int>(i - row * a.heads);
      float x[8], y[8], z[8] = {};
      if (a.out_low)
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.out_low) + i * a.dim + l * 8), IsBf16<T>::v, z);
      unpack8(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.o) + i * a.dim + l * 8), IsBf16<T>::v, x);
      unpack8(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.g) + row * a.g_row + head * a.g_head + l * 8),
              IsBf16<T>::v, y);
#pragma unroll
      for (int k = 0; k < 8; ++k) s = fmaf(x[k] + z[k], y[k], s);
      if (kLift<T>)
#pragma unroll
        for (int k = 0; k < 8; ++k) gg = fmaf(y[k], y[k], gg);
    }
    for (int o = lanes / 2; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      if (kLift<T>) gg += __shfl_xor_sync(0xffffffffu, gg, o);
    }
    if (i < n && l == 0) {
      const float2 st = a.stats[i];
      const float w = kLift<T> ? sqrtf(gg) : 0.f;
      if (kLift<T> && w < 1e38f && i / a.heads >= lo && i / a.heads < hi) top_g = fmaxf(top_g, w);
      a.bstats[static_cast<size_t>(i % a.heads) * a.q_rows + i / a.heads] = bias ? make_float4(st.x, st.y, s, w) : make_float4(fmaf(st.x, c, st.y), 0.f, s, w);
    }
  }
  if (kLift<T>) {
    const long long nv = static_cast<long long>(a.kv_rows) * a.kv_heads;
    rows_inside(a, a.cu_k, a.kv_rows, lo, hi);
    for (long long i0 = static_cast<long long>(blockIdx.x) * per; i0 < nv; i0 += static_cast<long long>(gridDim.x) * per) {
      const long long i = i0 + threadIdx.x / lanes, row = i / a.kv_heads;
      float vv = 0.f;
      if (i < nv && l * 8 < a.dim && row >= lo && row < hi && !(a.key_mask && a.key_mask[row] == 0)) {
        float y[8];
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + row * a.v_row + (i - row * a.kv_heads) * a.v_head + l * 8),
                IsBf16<T>::v, y);
#pragma unroll
        for (int k = 0; k < 8; ++k) vv = fmaf(y[k], y[k], vv);
      }
      for (int o = lanes / 2; o > 0; o >>= 1) vv += __shfl_xor_sync(0xffffffffu, vv, o);
      if (vv < 1e38f) top_v = fmaxf(top_v, sqrtf(vv));
    }
    __shared__ int red[2];
    if (threadIdx.x < 2) red[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t wg = __reduce_max_sync(0xffffffffu, __float_as_uint(top_g));
    const uint32_t wv = __reduce_max_sync(0xffffffffu, __float_as_uint(top_v));
    if ((threadIdx.x & 31) == 0) {
      atomicMax(red, static_cast<int>(wg));
      atomicMax(red + 1, static_cast<int>(wv));
    }
    __syncthreads();
    if (threadIdx.x == 0) a.norms[blockIdx.x] = make_float2(__int_as_float(red[0]), __int_as_float(red[1]));
  }
  grid_dep_release();
}

// rows of no sequence, in front of the first and behind the last, set to zero
template <typename T>
__device__ __forceinline__ void zero_outside(const int* cu, int seqs, int rows, long long per, T* out, int t,
                                             int threads) {
  const int lo = min(max(cu[0], 0), rows), hi = min(max(cu[seqs], lo), rows);
  const long long gone = (static_cast<long long>(lo) + rows - hi) * per;
  for (long long i = static_cast<long long>(blockIdx.x) * threads + t; i < gone;
       i += static_cast<long long>(gridDim.x) * threads)
    reinterpret_cast<uint4*>(out)[i < lo * per ? i : hi * per + (i - lo * per)] = make_uint4(0, 0, 0, 0);
}

// COLS columns of an accumulator row, times f, as 16-bit values to out[0 .. dim)
template <int COLS, typename T>
__device__ __forceinline__ void store_acc(uint32_t taddr, int col0, int dim, float f, bool live, bool any, T* out) {
#pragma unroll
  for (int q = 0; q < COLS / 16; ++q) {
    uint32_t o[16];
    __syncwarp();
    if (any) {
      tmem_ld16_nowait(taddr + col0 + q * 16, o);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = 0;
    }
    if (!live) continue;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = col0 + q * 16 + e * 8;
      if (c >= dim) break;
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(o[e * 8 + k]) * f;
      *reinterpret_cast<uint4*>(out + c) =
          make_uint4(pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7]));
    }
  }
}

// the same unrounded, to a row of a partial sum
template <int COLS>
__device__ __forceinline__ void store_part(uint32_t taddr, int col0, int dim, float f, bool live, bool any, float* out) {
#pragma unroll
  for (int q = 0; q < COLS / 16; ++q) {
    uint32_t o[16];
    __syncwarp();
    if (any) {
      tmem_ld16_nowait(taddr + col0 + q * 16, o);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = 0;
    }
    if (!live) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = col0 + q * 16 + e * 4;
      if (c >= dim) break;
      *reinterpret_cast<float4*>(out + c) =
          make_float4(__uint_as_float(o[e * 4]) * f, __uint_as_float(o[e * 4 + 1]) * f,
                      __uint_as_float(o[e * 4 + 2]) * f, __uint_as_float(o[e * 4 + 3]) * f);
    }
  }
}

// the bits of key_bits() for this warp's 32 columns of tile kt
__device__ __forceinline__ uint32_t key_word(const AttnArgs& a, const Item& it, int kt, int part, int lane) {
  const int c = kt * kTileRows + part * 32 + lane;
  bool on = c < it.klen;
  if (on && a.key_mask) on = a.key_mask[static_cast<size_t>(it.k0) + c] != 0;
  return __ballot_sync(0xffffffffu, on);
}

// --------------------------------------------------------------------------------- dq
// K of a tile is held from its scores to dQ += dS K, two tiles of the loop: with two buffers the
// next scores waited for their K to be loaded, 1800 clocks of a tile's 4400 at dim 128.
// A bias that one row alone has (a single representation's attention) has dS itself for its
// gradient, which the dq kernel then writes along: 2 x 1001 positions, 16 heads of 24, training
// 180 us (dq 63) against 237 (dq 38, dbias 85) with the dbias kernel, which forms S and dP once
// more. At DP = 128 shared memory has no room for the transposed tiles.
template <int DP>
constexpr bool kDirectBias = DP == 64;

template <int DP, bool BIAS>
struct DqCfg {
  static constexpr int kTile = DP / 64 * kBlk;
  static constexpr int kK = 3, kV = (DP == 128 && BIAS) ? 1 : 2;
  static constexpr int kOffG = kTile;
  static constexpr int kOffK = 2 * kTile;
  static constexpr int kOffV = kOffK + kK * kTile;
  static constexpr int kOffB = kOffV + kV * kTile;
  static constexpr int kOffBar = kOffB + (BIAS ? 2 * kBlk : 0);
  static constexpr int kOffT = kOffBar + 256;      // a warp's 32 x 32 of dS, rows of 16 + 1 words
  static constexpr int kSmem = kOffT + (kDirectBias<DP> && BIAS ? kElemWarps * 32 * 17 * 4 : 0) + 1024;
  static_assert(kSmem <= 232448, "dq exceeds 227 KB of shared memory");
};

template <int DP, bool BIAS, typename T>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dq_kernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnArgs a) {
  using C = DqCfg<DP, BIAS>;
  constexpr bool E = !(BIAS && DP == 128);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sG = smem + C::kOffG;
  uint8_t* sK = smem + C::kOffK;
  uint8_t* sV = smem + C::kOffV;
  uint8_t* sB = smem + C::kOffB;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_full + 2;     // 3
  uint64_t* k_empty = q_full + 5;    // 3
  uint64_t* v_full = q_full + 8;     // 2
  uint64_t* v_empty = q_full + 10;   // 2
  uint64_t* b_full = q_full + 12;
  uint64_t* b_empty = q_full + 13;
  uint64_t* s_full = q_full + 14;    // 2
  uint64_t* dp_full = q_full + 16;
  uint64_t* ds_ready = q_full + 17;
  uint64_t* acc_full = q_full + 18;
  uint64_t* drain = q_full + 19;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 20);
  int* red = reinterpret_cast<int*>(tmem_slot + 1);   // 2

  const int warp = uniform<E>(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 20; ++i) mbar_init(q_full + i, i == 13 || i == 17 ? kElemWarps : 1);
    fence_mbar_init();
    red[0] = red[1] = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform<E>(*tmem_slot);
  grid_dep_wait();
  grid_dep_release();
  const float top_v = kLift<T> ? largest_norms(a, red).y : 0.f;
  // columns: S of even tiles 0, dP 128, dQ 256, S of odd tiles 384
  int n = blockIdx.x;
  Item it;

  if (warp == kTmaWarp) {
    const uint32_t q_bytes = 2u * (DP / 64 * 128u * (a.group * a.tq));
    int qn = 0, kn = 0, kf = 0;
    bool ok = true;
    for (; ok && walk_item<false>(a, n, it); n += gridDim.x) {
      if (it.kt1 <= it.kt0) continue;
      if (lane == 0) {
        ok = mbar_wait(q_empty, (qn & 1) ^ 1, a.err, err_code(KERNEL_DQ, ROLE_PRODUCER, 1));
        if (ok) {
          mbar_arrive_expect_tx(q_full, q_bytes);
          load_tile4<DP>(&maps.q, q_full, sQ, 0, it.head, it.q0);
          load_tile4<DP>(&maps.g, q_full, sG, 0, it.head, it.q0);
          ++qn;
        }
        for (int t = it.kt0; ok && t < it.kt1; ++t) {
          const int s = kn % C::kK, sv = kn % C::kV;
          ok = mbar_wait(&k_empty[s], ((kn / C::kK) & 1) ^ 1, a.err, err_code(KERNEL_DQ, ROLE_PRODUCER, 2)) &&
               !(a.test_stall == STALL_DQ && blockIdx.x == 0 && kn == 0);
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[s], C::kTile);
          load_tile4<DP>(&maps.k, &k_full[s], sK + s * C::kTile, it.head, it.k0 + t * kTileRows, it.kb);
          ++kf;
          ok = mbar_wait(&v_empty[sv], ((kn / C::kV) & 1) ^ 1, a.err, err_code(KERNEL_DQ, ROLE_PRODUCER, 3)) &&
               (!BIAS || mbar_wait(b_empty, (kn & 1) ^ 1, a.err, err_code(KERNEL_DQ, ROLE_PRODUCER, 4)));
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[sv], C::kTile);
          load_tile4<DP>(&maps.v, &v_full[sv], sV + sv * C::kTile, it.head, it.k0 + t * kTileRows, it.kb);
          if (BIAS) {
            mbar_arrive_expect_tx(b_full, 2 * kBlk);
            for (int h = 0; h < 2; ++h)
              tma_load_4d(&maps.bias, b_full, sB + h * kBlk, t * kTileRows + h * 64, it.pos0, it.head,
                          it.seq / a.bias_seqs);
          }
          ++kn;
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
    }
    if (lane == 0) {
      if (qn) mbar_wait_drain(q_full, (qn - 1) & 1);
      for (int i = kf > C::kK ? kf - C::kK : 0; i < kf; ++i) mbar_wait_drain(&k_full[i % C::kK], (i / C::kK) & 1);
      for (int i = kn > C::kV ? kn - C::kV : 0; i < kn; ++i) mbar_wait_drain(&v_full[i % C::kV], (i / C::kV) & 1);
      if (BIAS && kn) mbar_wait_drain(b_full, (kn - 1) & 1);
    }
  } else if (warp == kMmaWarp) {
    constexpr uint32_t id_s = idesc_f16(IsBf16<T>::v, 128, 128, 0, 0);
    constexpr uint32_t id_o = idesc_f16(IsBf16<T>::v, 128, DP, 0, 1);
    const uint32_t q_addr = uniform<E>(smem_u32(sQ)), g_addr = uniform<E>(smem_u32(sG));
    int qn = 0, kn = 0;
    bool ok = true;
    // scores of key tile number i (of all this block meets); rows of K that are not keys of
    // this sequence are cleared first, since 0 * K enters dQ
    auto scores = [&](int i, int kt) -> bool {
      const int s = i % C::kK;
      uint32_t keep[4];
      if (a.key_mask) key_bits(a, it, kt, lane, keep);
      if (!mbar_wait_warp(&k_full[s], (i / C::kK) & 1, a.err, err_code(KERNEL_DQ, ROLE_MMA, 2))) return false;
      const int valid = it.klen - kt * kTileRows;
      if (a.key_mask) {
        if ((keep[0] & keep[1] & keep[2] & keep[3]) != 0xffffffffu) {
          zero_rows_masked<DP>(sK + s * C::kTile, keep, lane);
          fence_proxy_async_smem();
          __syncwarp();
        }
      } else if (valid < kTileRows) {
        zero_rows_from<DP>(sK + s * C::kTile, valid, lane);
        fence_proxy_async_smem();
        __syncwarp();
      }
      tc_fence_after();
      const uint32_t odd = uniform<E>(i & 1), k_addr = uniform<E>(smem_u32(sK + s * C::kTile));
      if (issuer<E>(lane)) {
        mma_rows<E>(tmem + odd * 384, q_addr, k_addr, id_s, a.ksteps);
        umma_commit(&s_full[odd]);
      }
      __syncwarp();
      return true;
    };
    auto weights_grad = [&](int i) -> bool {
      const int s = i % C::kV;
      if (!mbar_wait_warp(&v_full[s], (i / C::kV) & 1, a.err, err_code(KERNEL_DQ, ROLE_MMA, 3))) return false;
      tc_fence_after();
      const uint32_t su = uniform<E>(s), v_addr = uniform<E>(smem_u32(sV + s * C::kTile));
      if (issuer<E>(lane)) {
        mma_rows<E>(tmem + 128, g_addr, v_addr, id_s, a.ksteps);
        umma_commit(dp_full);
        umma_commit(&v_empty[su]);
      }
      __syncwarp();
      return true;
    };
    for (; ok && walk_item<false>(a, n, it); n += gridDim.x) {
      const int tiles = it.kt1 - it.kt0;
      if (tiles <= 0) continue;
      ok = mbar_wait_warp(q_full, qn & 1, a.err, err_code(KERNEL_DQ, ROLE_MMA, 1));
      ok = ok && scores(kn, it.kt0) && weights_grad(kn);
      for (int j = 0; ok && j < tiles; ++j, ++kn) {
        if (j + 1 < tiles) ok = scores(kn + 1, it.kt0 + j + 1);
        ok = ok && mbar_wait_warp(ds_ready, kn & 1, a.err, err_code(KERNEL_DQ, ROLE_MMA, 4));
        if (ok && j + 1 < tiles) ok = weights_grad(kn + 1);
        if (!ok) break;
        tc_fence_after();
        const uint32_t s = uniform<E>(kn % C::kK), odd = uniform<E>(kn & 1), more = uniform<E>(j > 0);
        const uint32_t k_addr = uniform<E>(smem_u32(sK + s * C::kTile)), last = uniform<E>(j + 1 == tiles);
        if (issuer<E>(lane)) {
          mma_cols<E>(tmem + 256, tmem + odd * 384, k_addr, id_o, more);
          umma_commit(&k_empty[s]);
          if (last) {
            umma_commit(acc_full);
            umma_commit(q_empty);
          }
        }
        __syncwarp();
      }
      ++qn;
    }
    if (!ok) report_failure(a, KERNEL_DQ);
    if (issuer<E>(lane)) {
      umma_commit(drain);
      mbar_wait_drain(drain, 0);
    }
  } else {
    const int quad = warp & 3, part = warp >> 2;   // columns 32 part and on
    const int row = quad * 32 + lane;
    const int tok = row / a.group, gi = row - tok * a.group;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c = log2_scale(a.scale);
    T* dq = static_cast<T*>(a.dq);
    if (a.walk == WALK_LIST)
      zero_outside(a.cu_q, a.seqs, a.q_rows, static_cast<long long>(a.heads) * a.dim / 8, dq, threadIdx.x, kElemWarps * 32);
    int kn = 0, qn = 0;
    bool ok = true;
    // A failed wait is carried to the next barrier, where the quarter's warps leave together.
    for (; walk_item<false>(a, n, it); n += gridDim.x) {
      const bool live = tok < it.nq && row < a.group * a.tq;
      const size_t orow = (static_cast<size_t>(it.q0) + tok) * a.heads + it.head * a.group + gi;
      const int seen = a.causal ? min(it.klen, it.pos0 + tok + it.off + 1) : it.klen;
      const float4 st = live ? a.bstats[static_cast<size_t>(it.head * a.group + gi) * a.q_rows + it.q0 + tok]
                             : make_float4(0.f, INFINITY, 0.f, 0.f);
      const int up = kLift<T> ? lift(st.w, top_v) : 0;
      const float ref = BIAS ? st.x : live ? st.x - up : INFINITY, ylift = st.y - up;
      for (int kt = it.kt0; kt < it.kt1; ++kt, ++kn) {
        const int b = kn & 1;
        const uint32_t on = (a.key_mask ? key_word(a, it, kt, part, lane) : 0xffffffffu) &
                            bits_below(seen - kt * kTileRows, part);
        const bool cut = __any_sync(0xffffffffu, on != 0xffffffffu);
        ok = ok && mbar_wait_warp(&s_full[b], (kn >> 1) & 1, a.err, err_code(KERNEL_DQ, ROLE_EPILOGUE, 1));
        if (BIAS) ok = ok && mbar_wait_warp(b_full, kn & 1, a.err, err_code(KERNEL_DQ, ROLE_EPILOGUE, 2));
        tc_fence_after();
        const uint32_t scol = lanes + (b ? 384 : 0);
        uint32_t r[32];
        FTM_TMEM_LD32_NOWAIT(scol + part * 32, r);
        tmem_wait_ld();
        if (BIAS) {
          add_bias<T>(r, sB + (part >> 1) * kBlk, row, (part & 1) * 4, a.scale);
          __syncwarp();
          if (lane == 0) mbar_arrive(b_empty);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = __uint_as_float(r[e]);
          r[e] = __float_as_uint(ex2(BIAS ? fmaf(x - ref, kLog2e, -ylift) : fmaf(x, c, -ref)));
        }
        if (cut) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(on & (1u << e))) r[e] = 0u;
        }
        ok = ok && mbar_wait_warp(dp_full, kn & 1, a.err, err_code(KERNEL_DQ, ROLE_EPILOGUE, 3));
        tc_fence_after();
        uint32_t pk[16], d[32];
        FTM_TMEM_LD32_NOWAIT(lanes + 128 + part * 32, d);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float x0 = __uint_as_float(r[e]) * (__uint_as_float(d[e]) - st.z);
          float x1 = __uint_as_float(r[e + 1]) * (__uint_as_float(d[e + 1]) - st.z);
          if (cut) {   // a key that is not seen gives nothing, whatever its V holds
            x0 = r[e] ? x0 : 0.f;
            x1 = r[e + 1] ? x1 : 0.f;
          }
          pk[e / 2] = pack16<T>(x0, x1);
        }
        ok = named_barrier_all(1 + quad, 128, ok);   // the whole row of S has been read: dS goes over it
        if (!ok) break;
        tmem_st16(scol + part * 16, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
        if (kDirectBias<DP> && BIAS && a.dbias_direct) {
          // transposed in shared memory, so that a warp writes neighbours of one row at a time
          uint32_t* tile = reinterpret_cast<uint32_t*>(smem + C::kOffT) + warp * 32 * 17;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (kLift<T>) {   // exact, or a subnormal
              const float2 f = unpack2<T>(pk[e]);
              pk[e] = pack16<T>(f.x * pow2(-up), f.y * pow2(-up));
            }
            tile[lane * 17 + e] = pk[e];
          }
          __syncwarp();
          const int col = kt * kTileRows + part * 32 + lane, row0 = it.pos0 + quad * 32;
          if (col < a.k_len) {
            uint16_t* to = static_cast<uint16_t*>(a.dbias) +
                           ((static_cast<size_t>(it.seq) * a.heads + it.head) * a.q_len + row0) * a.k_len + col;
            const int rows = min(32, a.q_len - row0);
#pragma unroll 4
            for (int y = 0; y < rows; ++y)
              to[static_cast<size_t>(y) * a.k_len] =
                  static_cast<uint16_t>(tile[y * 17 + (lane >> 1)] >> ((lane & 1) * 16));
          }
          __syncwarp();
        }
      }
      const bool any = it.kt1 > it.kt0;
      if (any) {
        if (!ok) break;
        ok = mbar_wait_warp(acc_full, qn & 1, a.err, err_code(KERNEL_DQ, ROLE_EPILOGUE, 4));
        ++qn;
        tc_fence_after();
      }
      store_acc<DP / 4>(lanes + 256, part * (DP / 4), a.dim, a.scale * pow2(-up), live && ok, any, dq + orow * a.dim);
      tc_fence_before();
    }
    if (!ok) report_failure(a, KERNEL_DQ);
  }
  __syncwarp();      // the lanes of a role that one lane drained
  __syncthreads();
  tc_fence_after();
  __syncwarp();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// -------------------------------------------------------------------------------- dkv
template <int DP, bool BIAS>
struct DkvCfg {
  static constexpr int kTile = DP / 64 * kBlk;
  static constexpr int kOffV = kTile;
  static constexpr int kOffQ = 2 * kTile;
  static constexpr int kOffG = 4 * kTile;
  static constexpr int kOffB = 6 * kTile;
  static constexpr int kCols = (BIAS && DP == 128) ? 1 : 2;       // what shared memory leaves
  static constexpr int kOffCol = kOffB + (BIAS ? 2 * kBlk : 0);   // kCols x 128 x (x, y, z)
  static constexpr int kOffBar = kOffCol + kCols * kTileRows * 12;
  static constexpr int kSmem = kOffBar + 256 + 1024;
  static_assert(kSmem <= 232448, "dkv exceeds 227 KB of shared memory");
};

template <int DP, bool BIAS, typename T>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dkv_kernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnArgs a) {
  using C = DkvCfg<DP, BIAS>;
  constexpr bool E = !(BIAS && DP == 128);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = smem + C::kOffV;
  uint8_t* sQ = smem + C::kOffQ;
  uint8_t* sG = smem + C::kOffG;
  uint8_t* sB = smem + C::kOffB;
  float* sC = reinterpret_cast<float*>(smem + C::kOffCol);   // [buffer][x: 128, y: 128, z: 128]
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* kv_empty = kv_full + 1;
  uint64_t* q_full = kv_full + 2;
  uint64_t* q_empty = kv_full + 4;
  uint64_t* g_full = kv_full + 6;
  uint64_t* g_empty = kv_full + 8;
  uint64_t* b_full = kv_full + 10;
  uint64_t* b_empty = kv_full + 11;
  uint64_t* c_full = kv_full + 12;   // 2
  uint64_t* c_empty = kv_full + 14;  // 2
  uint64_t* s_full = kv_full + 16;
  uint64_t* p_ready = kv_full + 17;
  uint64_t* dp_full = kv_full + 18;
  uint64_t* ds_ready = kv_full + 19;
  uint64_t* acc_full = kv_full + 20;
  uint64_t* drain = kv_full + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_full + 22);
  int* red = reinterpret_cast<int*>(tmem_slot + 1);   // 2

  const int warp = uniform<E>(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 22; ++i)
      mbar_init(kv_full + i, i == 11 || i == 14 || i == 15 || i == 17 || i == 19 ? kElemWarps : 1);
    fence_mbar_init();
    red[0] = red[1] = 0;
  }
  // rows of a query tile that no load writes (128 is no multiple of the group): zero once
  {
    const int used = a.group * a.tq;
    if (used < kTileRows) {
      for (int t = warp; t < 4; t += kBwdThreads / 32)
        zero_rows_from<DP>(sQ + t * C::kTile, used, lane);
      fence_proxy_async_smem();
    }
  }
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform<E>(*tmem_slot);
  grid_dep_wait();
  grid_dep_release();
  int up = 0;      // of dS^T; P^T, which it is formed of, has 2^kLiftP in it
  if (kLift<T>) {
    const float2 top = largest_norms(a, red);
    up = lift(top.x, top.y);
  }
  const float rest = kLift<T> ? pow2(up - kLiftP) : 1.f;
  // columns: S^T / P^T 0, dP^T / dS^T 128, dV 256, dK 384
  int n = blockIdx.x;
  Item it;

  if (warp == kTmaWarp) {
    const uint32_t q_bytes = DP / 64 * 128u * (a.group * a.tq);
    int in = 0, qn = 0;
    bool ok = true;
    int col_tok[4];          // token of this lane's columns (past all tiles: none), and the place of
    size_t col_off[4];       // its constants behind the tile's first
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int r = w * 32 + lane, tok = r / a.group;
      col_tok[w] = r < a.group * a.tq ? tok : INT_MAX;
      col_off[w] = static_cast<size_t>(r - tok * a.group) * a.q_rows + tok;
    }
    for (; ok && walk_item<true>(a, n, it); n += gridDim.x) {
      if (it.kt1 <= it.kt0) continue;
      ok = mbar_wait_warp(kv_empty, (in & 1) ^ 1, a.err, err_code(KERNEL_DKV, ROLE_PRODUCER, 1));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(kv_full, 2 * C::kTile);
        load_tile4<DP>(&maps.k, kv_full, sK, it.head, it.k0 + it.tile * kTileRows, 0);
        load_tile4<DP>(&maps.v, kv_full, sV, it.head, it.k0 + it.tile * kTileRows, 0);
      }
      ++in;
      for (int t = it.kt0; t < it.kt1; ++t) {
        const int s = qn & 1;
        const uint32_t ph = ((qn >> 1) & 1) ^ 1;
        ok = !(a.test_stall == STALL_DKV && blockIdx.x == 0 && qn == 0) &&
             mbar_wait_warp(&q_empty[s], ph, a.err, err_code(KERNEL_DKV, ROLE_PRODUCER, 2)) &&
             mbar_wait_warp(&g_empty[s], ph, a.err, err_code(KERNEL_DKV, ROLE_PRODUCER, 3)) &&
             (!BIAS || mbar_wait_warp(b_empty, (qn & 1) ^ 1, a.err, err_code(KERNEL_DKV, ROLE_PRODUCER, 4)));
        if (!ok) break;
        if (lane == 0) {
          const int row = it.q0 + t * a.tq;
          mbar_arrive_expect_tx(&q_full[s], q_bytes);
          load_tile4<DP>(&maps.q, &q_full[s], sQ + s * C::kTile, 0, it.head, row);
          mbar_arrive_expect_tx(&g_full[s], q_bytes);
          load_tile4<DP>(&maps.g, &g_full[s], sG + s * C::kTile, 0, it.head, row);
          if (BIAS) {
            mbar_arrive_expect_tx(b_full, 2 * kBlk);
            for (int h = 0; h < 2; ++h)
              tma_load_4d(&maps.bias, b_full, sB + h * kBlk, it.tile * kTileRows + h * 64, t * a.tq, it.head,
                          it.seq / a.bias_seqs);
          }
        }
        ++qn;
        __syncwarp();
        // the constants of this tile's queries, one per column of S^T: four loads in flight
        // (behind conditions they came one after the other, 4900 clocks a tile)
        float4 st[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int left = it.nq - t * a.tq;
          const bool live = col_tok[w] < left;
          const size_t at = live ? static_cast<size_t>(it.head) * a.group * a.q_rows + it.q0 + t * a.tq + col_off[w] : 0;
          st[w] = a.bstats[at];
          if (kLift<T>) {
            (BIAS ? st[w].y : st[w].x) -= kLiftP;
            st[w].z *= rest;
          }
          if (!live) st[w] = make_float4(BIAS ? 0.f : INFINITY, INFINITY, 0.f, 0.f);   // p = 0
        }
        const int cn = qn - 1, cb = cn % C::kCols;
        ok = mbar_wait_warp(&c_empty[cb], ((cn / C::kCols) & 1) ^ 1, a.err, err_code(KERNEL_DKV, ROLE_PRODUCER, 5));
        if (!ok) break;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int r = w * 32 + lane;
          sC[cb * 384 + r] = st[w].x;
          sC[cb * 384 + 128 + r] = st[w].y;
          sC[cb * 384 + 256 + r] = st[w].z;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&c_full[cb]);
      }
    }
    if (lane == 0) {
      if (in) mbar_wait_drain(kv_full, (in - 1) & 1);
      for (int i = qn > 2 ? qn - 2 : 0; i < qn; ++i) {
        mbar_wait_drain(&q_full[i & 1], (i >> 1) & 1);
        mbar_wait_drain(&g_full[i & 1], (i >> 1) & 1);
      }
      if (BIAS && qn) mbar_wait_drain(b_full, (qn - 1) & 1);
    }
  } else if (warp == kMmaWarp) {
    constexpr uint32_t id_s = idesc_f16(IsBf16<T>::v, 128, 128, 0, 0);
    constexpr uint32_t id_o = idesc_f16(IsBf16<T>::v, 128, DP, 0, 1);
    const uint32_t k_addr = uniform<E>(smem_u32(sK)), v_addr = uniform<E>(smem_u32(sV));
    int in = 0, qn = 0;
    bool ok = true;
    // waits for a tile of Q or g; rows behind the sequence's end are cleared, since their zero
    // weights meet them in the accumulating products
    auto arrived = [&](uint64_t* full, uint8_t* tiles, int i, int t, int site) -> bool {
      const int s = i & 1;
      if (!mbar_wait_warp(&full[s], (i >> 1) & 1, a.err, err_code(KERNEL_DKV, ROLE_MMA, site))) return false;
      const int valid = rows_held(it.nq - t * a.tq, a.tq, a.group);
      if (valid < a.group * a.tq) {
        zero_rows_from<DP>(tiles + s * C::kTile, valid, lane);
        fence_proxy_async_smem();
        __syncwarp();
      }
      tc_fence_after();
      return true;
    };
    for (; ok && walk_item<true>(a, n, it); n += gridDim.x) {
      const int tiles = it.kt1 - it.kt0;
      if (tiles <= 0) continue;
      ok = mbar_wait_warp(kv_full, in & 1, a.err, err_code(KERNEL_DKV, ROLE_MMA, 1));
      ++in;
      for (int j = -1; ok && j < tiles; ++j) {
        // (j = -1: only the first tile's scores)
        const int i = qn + j;
        const uint32_t s = uniform<E>(i & 1), t = uniform<E>((i + 1) & 1), more = uniform<E>(j > 0);
        const uint32_t g_at = uniform<E>(smem_u32(sG + s * C::kTile)), q_at = uniform<E>(smem_u32(sQ + s * C::kTile));
        const uint32_t g_next = uniform<E>(smem_u32(sG + t * C::kTile)), q_next = uniform<E>(smem_u32(sQ + t * C::kTile));
        if (j >= 0) {
          ok = mbar_wait_warp(p_ready, i & 1, a.err, err_code(KERNEL_DKV, ROLE_MMA, 2));
          if (!ok) break;
          tc_fence_after();
          if (issuer<E>(lane)) {
            mma_cols<E>(tmem + 256, tmem, g_at, id_o, more);
            umma_commit(&g_empty[s]);
          }
          __syncwarp();
        }
        if (j + 1 < tiles) {   // behind dV in the pipe, so S^T may overwrite P^T
          ok = arrived(q_full, sQ, i + 1, it.kt0 + j + 1, 3);
          if (!ok) break;
          if (issuer<E>(lane)) {
            mma_rows<E>(tmem, k_addr, q_next, id_s, a.ksteps);
            umma_commit(s_full);
          }
          __syncwarp();
        }
        if (j >= 0) {
          ok = mbar_wait_warp(ds_ready, i & 1, a.err, err_code(KERNEL_DKV, ROLE_MMA, 4));
          if (!ok) break;
          tc_fence_after();
          if (issuer<E>(lane)) {
            mma_cols<E>(tmem + 384, tmem + 128, q_at, id_o, more);
            umma_commit(&q_empty[s]);
          }
          __syncwarp();
        }
        if (j + 1 < tiles) {
          ok = arrived(g_full, sG, i + 1, it.kt0 + j + 1, 5);
          if (!ok) break;
          if (issuer<E>(lane)) {
            mma_rows<E>(tmem + 128, v_addr, g_next, id_s, a.ksteps);
            umma_commit(dp_full);
          }
          __syncwarp();
        } else if (issuer<E>(lane)) {
          umma_commit(acc_full);
          umma_commit(kv_empty);
        }
        __syncwarp();
      }
      qn += tiles;
    }
    if (!ok) report_failure(a, KERNEL_DKV);
    if (issuer<E>(lane)) {
      umma_commit(drain);
      mbar_wait_drain(drain, 0);
    }
  } else {
    const int quad = warp & 3, part = warp >> 2;   // columns 32 part and on
    const int row = quad * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c = log2_scale(a.scale);
    T *dk = static_cast<T*>(a.dk), *dv = static_cast<T*>(a.dv);
    if (a.walk == WALK_LIST && a.kv_splits == 1) {
      const long long per = static_cast<long long>(a.kv_heads) * a.dim / 8;
      zero_outside(a.cu_k, a.seqs, a.kv_rows, per, dk, threadIdx.x, kElemWarps * 32);
      zero_outside(a.cu_k, a.seqs, a.kv_rows, per, dv, threadIdx.x, kElemWarps * 32);
    }
    int qn = 0, in = 0;
    bool ok = true;
    // A failed wait is carried to the next barrier, where the quarter's warps leave together.
    for (; walk_item<true>(a, n, it); n += gridDim.x) {
      const int key = it.tile * kTileRows + row;
      const bool live = key < it.klen;
      const size_t orow = (static_cast<size_t>(it.k0) + key) * a.kv_heads + it.head;
      bool on = live;
      if (on && a.key_mask) on = a.key_mask[static_cast<size_t>(it.k0) + key] != 0;
      const bool gone = __any_sync(0xffffffffu, !on);
      for (int t = it.kt0; t < it.kt1; ++t, ++qn) {
        const int cb = qn % C::kCols;
        // queries in front of the first one that sees this key (causal): columns below `lo`
        const int lo = a.causal ? columns_before(key - it.off - t * a.tq, a.group) : 0;
        const bool cut = gone || __any_sync(0xffffffffu, lo > 0);
        const float* col = sC + cb * 384;
        ok = ok && mbar_wait_warp(&c_full[cb], (qn / C::kCols) & 1, a.err, err_code(KERNEL_DKV, ROLE_EPILOGUE, 1));
        if (BIAS) ok = ok && mbar_wait_warp(b_full, qn & 1, a.err, err_code(KERNEL_DKV, ROLE_EPILOGUE, 2));
        ok = ok && mbar_wait_warp(s_full, qn & 1, a.err, err_code(KERNEL_DKV, ROLE_EPILOGUE, 3));
        tc_fence_after();
        uint32_t r[32];
        FTM_TMEM_LD32_NOWAIT(lanes + part * 32, r);
        tmem_wait_ld();
        if (BIAS) {
          // the bias of (query, this key): rows of the tile are queries
          const uint8_t* bt = sB + (row >> 6) * kBlk + (row & 7) * 2;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const T bv = *reinterpret_cast<const T*>(bt + sw128_off(part * 32 + e, (row & 63) >> 3));
            r[e] = __float_as_uint(fmaf(__uint_as_float(r[e]), a.scale, static_cast<float>(bv)));
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(b_empty);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 x4 = *reinterpret_cast<const float4*>(col + part * 32 + e);
          const float xs[4] = {x4.x, x4.y, x4.z, x4.w};
          float ys[4] = {0.f, 0.f, 0.f, 0.f};
          if (BIAS) {
            const float4 y4 = *reinterpret_cast<const float4*>(col + 128 + part * 32 + e);
            ys[0] = y4.x; ys[1] = y4.y; ys[2] = y4.z; ys[3] = y4.w;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = __uint_as_float(r[e + k]);
            r[e + k] = __float_as_uint(ex2(BIAS ? fmaf(x - xs[k], kLog2e, -ys[k]) : fmaf(x, c, -xs[k])));
          }
        }
        if (cut) {
          const uint32_t bits = on ? ~bits_below(lo, part) : 0u;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(bits & (1u << e))) r[e] = 0u;
        }
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) pk[e / 2] = pack16<T>(__uint_as_float(r[e]), __uint_as_float(r[e + 1]));
        ok = named_barrier_all(1 + quad, 128, ok);   // the whole row of S^T has been read: P^T goes over it
        if (!ok) break;
        tmem_st16(lanes + part * 16, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
        ok = mbar_wait_warp(dp_full, qn & 1, a.err, err_code(KERNEL_DKV, ROLE_EPILOGUE, 4));
        tc_fence_after();
        uint32_t d[32];
        FTM_TMEM_LD32_NOWAIT(lanes + 128 + part * 32, d);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 z = *reinterpret_cast<const float4*>(col + 256 + part * 32 + e);
          const float zs[4] = {z.x, z.y, z.z, z.w};
          float x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float y = kLift<T> ? fmaf(__uint_as_float(d[e + k]), rest, -zs[k]) : __uint_as_float(d[e + k]) - zs[k];
            x[k] = __uint_as_float(r[e + k]) * y;
            if (cut) x[k] = r[e + k] ? x[k] : 0.f;
          }
          pk[e / 2] = pack16<T>(x[0], x[1]);
          pk[e / 2 + 1] = pack16<T>(x[2], x[3]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&c_empty[cb]);
        ok = named_barrier_all(1 + quad, 128, ok);
        if (!ok) break;
        tmem_st16(lanes + 128 + part * 16, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ds_ready);
      }
      const bool any = it.kt1 > it.kt0;
      if (any) {
        if (!ok) break;
        ok = mbar_wait_warp(acc_full, in & 1, a.err, err_code(KERNEL_DKV, ROLE_EPILOGUE, 5));
        ++in;
        tc_fence_after();
      }
      const float fk = a.scale * pow2(-up), fv = kLift<T> ? pow2(-kLiftP) : 1.f;
      if (a.kv_splits > 1) {
        const size_t all = static_cast<size_t>(a.kv_rows) * a.kv_heads * a.dim;
        float* to = a.dkv_part + 2 * it.slot * all + orow * a.dim;
        store_part<DP / 4>(lanes + 384, part * (DP / 4), a.dim, fk, live && ok, any, to);
        store_part<DP / 4>(lanes + 256, part * (DP / 4), a.dim, fv, live && ok, any, to + all);
      } else {
        store_acc<DP / 4>(lanes + 256, part * (DP / 4), a.dim, fv, live && ok, any, dv + orow * a.dim);
        store_acc<DP / 4>(lanes + 384, part * (DP / 4), a.dim, fk, live && ok, any, dk + orow * a.dim);
      }
      tc_fence_before();
    }
    if (!ok) report_failure(a, KERNEL_DKV);
  }
  __syncwarp();      // the lanes of a role that one lane drained
  __syncthreads();
  tc_fence_after();
  __syncwarp();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------------ dbias
template <int DP>
struct DbCfg {
  static constexpr int kTile = DP / 64 * kBlk;
  static constexpr int kStages = DP == 64 ? 2 : 1;
  static constexpr int kStage = 4 * kTile;    // Q, g, K, V
  static constexpr int kOffB = kStages * kStage;
  static constexpr int kOffT = kOffB + 2 * kBlk;          // a tile of 32 rows x 16 columns per warp
  static constexpr int kOffBar = kOffT + kElemWarps * 32 * 17 * 4;
  static constexpr int kSmem = kOffBar + 256 + 1024;
  static_assert(kSmem <= 232448, "dbias exceeds 227 KB of shared memory");
};

template <int DP, typename T>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dbias_kernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnArgs a) {
  using C = DbCfg<DP>;
  constexpr bool E = DP == 64;
  constexpr int NS = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sB = smem + C::kOffB;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + 2;
  uint64_t* t_full = full + 4;
  uint64_t* t_empty = full + 6;
  uint64_t* b_full = full + 8;
  uint64_t* b_empty = full + 9;
  uint64_t* drain = full + 10;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + 11);
  const int warp = uniform<E>(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 11; ++i) mbar_init(full + i, i == 6 || i == 7 || i == 9 ? kElemWarps : 1);
    fence_mbar_init();
  }
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform<E>(*tmem_slot);
  grid_dep_wait();
  grid_dep_release();

  const int biases = a.seqs / a.bias_seqs;
  const int items = a.splits * biases * a.heads * a.q_tiles * a.k_tiles;
  int split = 0, bb = 0, head = 0, qt = 0, kt = 0, r0 = 0, r1 = 0;
  auto item = [&](int i) {
    kt = i % a.k_tiles;
    i /= a.k_tiles;
    qt = i % a.q_tiles;
    i /= a.q_tiles;
    head = i % a.heads;
    i /= a.heads;
    bb = i % biases;
    split = i / biases;
    r0 = static_cast<int>(static_cast<long long>(a.bias_seqs) * split / a.splits);
    r1 = static_cast<int>(static_cast<long long>(a.bias_seqs) * (split + 1) / a.splits);
  };

  if (warp == kTmaWarp) {
    if (lane == 0) {
      int rn = 0, in = 0;
      bool ok = true;
      for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
        item(i);
        ok = mbar_wait(b_empty, (in & 1) ^ 1, a.err, err_code(KERNEL_DBIAS, ROLE_PRODUCER, 1));
        if (!ok) break;
        mbar_arrive_expect_tx(b_full, 2 * kBlk);
        for (int h = 0; h < 2; ++h)
          tma_load_4d(&maps.bias, b_full, sB + h * kBlk, kt * kTileRows + h * 64, qt * kTileRows, head, bb);
        ++in;
        for (int r = r0; r < r1; ++r, ++rn) {
          const int s = rn % NS;
          ok = mbar_wait(&empty[s], ((rn / NS) & 1) ^ 1, a.err, err_code(KERNEL_DBIAS, ROLE_PRODUCER, 2));
          if (!ok) break;
          const int seq = bb * a.bias_seqs + r;
          const int q0 = seq * a.q_len + qt * kTileRows, k0 = seq * a.k_len + kt * kTileRows;
          uint8_t* st = smem + s * C::kStage;
          mbar_arrive_expect_tx(&full[s], C::kStage);
          load_tile4<DP>(&maps.q, &full[s], st, 0, head, q0);
          load_tile4<DP>(&maps.g, &full[s], st + C::kTile, 0, head, q0);
          load_tile4<DP>(&maps.k, &full[s], st + 2 * C::kTile, head, k0, 0);
          load_tile4<DP>(&maps.v, &full[s], st + 3 * C::kTile, head, k0, 0);
        }
      }
      for (int i = rn > NS ? rn - NS : 0; i < rn; ++i) mbar_wait_drain(&full[i % NS], (i / NS) & 1);
      if (in) mbar_wait_drain(b_full, (in - 1) & 1);
    }
  } else if (warp == kMmaWarp) {
    constexpr uint32_t id_s = idesc_f16(IsBf16<T>::v, 128, 128, 0, 0);
    int rn = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
      item(i);
      for (int r = r0; r < r1; ++r, ++rn) {
        const uint32_t s = uniform<E>(rn % NS), tb = uniform<E>(rn & 1);
        const uint32_t st = uniform<E>(smem_u32(smem + s * C::kStage));
        ok = mbar_wait_warp(&full[s], (rn / NS) & 1, a.err, err_code(KERNEL_DBIAS, ROLE_MMA, 1)) &&
             mbar_wait_warp(&t_empty[tb], ((rn >> 1) & 1) ^ 1, a.err, err_code(KERNEL_DBIAS, ROLE_MMA, 2));
        if (!ok) break;
        tc_fence_after();
        if (issuer<E>(lane)) {
          mma_rows<E>(tmem + tb * 256, st, st + 2 * C::kTile, id_s, a.ksteps);
          mma_rows<E>(tmem + tb * 256 + 128, st + C::kTile, st + 3 * C::kTile, id_s, a.ksteps);
          umma_commit(&t_full[tb]);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
    }
    if (!ok) report_failure(a, KERNEL_DBIAS);
    if (issuer<E>(lane)) {
      umma_commit(drain);
      mbar_wait_drain(drain, 0);
    }
  } else {
    const int quad = warp & 3, part = warp >> 2;   // columns 32 part and on
    const int row = quad * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    int rn = 0, in = 0;
    bool ok = true;
    for (int i = blockIdx.x; ok && i < items; i += gridDim.x) {
      item(i);
      const int pos = qt * kTileRows + row;
      const bool live = pos < a.q_len;
      Item it;
      it.klen = a.k_len;
      ok = mbar_wait_warp(b_full, in & 1, a.err, err_code(KERNEL_DBIAS, ROLE_EPILOGUE, 1));
      if (!ok) break;
      ++in;
      float acc[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) acc[e] = 0.f;
      for (int r = r0; r < r1; ++r, ++rn) {
        const int tb = rn & 1, seq = bb * a.bias_seqs + r;
        it.k0 = seq * a.k_len;
        const uint32_t on = key_word(a, it, kt, part, lane);
        const float4 st = live ? a.bstats[static_cast<size_t>(head) * a.q_rows + static_cast<size_t>(seq) * a.q_len + pos]
                               : make_float4(0.f, INFINITY, 0.f, 0.f);
        ok = mbar_wait_warp(&t_full[tb], (rn >> 1) & 1, a.err, err_code(KERNEL_DBIAS, ROLE_EPILOGUE, 2));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t x[16], d[16];
          tmem_ld16_nowait(lanes + tb * 256 + part * 32 + q * 16, x);
          tmem_ld16_nowait(lanes + tb * 256 + 128 + part * 32 + q * 16, d);
          tmem_wait_ld();
#pragma unroll
          for (int e8 = 0; e8 < 2; ++e8) {
            const uint4 b4 = *reinterpret_cast<const uint4*>(sB + (part >> 1) * kBlk +
                                                             sw128_off(row, (part & 1) * 4 + q * 2 + e8));
            const uint32_t bw[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int k = e8 * 8 + e;
              const float2 f = unpack2<T>(bw[e >> 1]);
              const float t = fmaf(__uint_as_float(x[k]), a.scale, e & 1 ? f.y : f.x);
              const float p = ex2(fmaf(t - st.x, kLog2e, -st.y));
              const float ds = p * (__uint_as_float(d[k]) - st.z);
              acc[q * 16 + k] += on & (1u << (q * 16 + k)) ? ds : 0.f;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&t_empty[tb]);
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(b_empty);
      // transposed in shared memory, so that 16 lanes write neighbours of a row: each lane
      // writing along its own row cost a sector per element (16 heads of N = 1001: 340 us)
      float* tile = reinterpret_cast<float*>(smem + C::kOffT) + warp * 32 * 17;
      const int row0 = qt * kTileRows + quad * 32, rows = min(32, a.q_len - row0);
      const size_t all = static_cast<size_t>(biases) * a.heads * a.q_len * a.k_len;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int e = 0; e < 16; ++e) tile[lane * 17 + e] = acc[q * 16 + e];
        __syncwarp();
        const int col = kt * kTileRows + part * 32 + q * 16 + (lane & 15);
        if (col < a.k_len) {
          for (int y = lane >> 4; y < rows; y += 2) {
            const size_t at = ((static_cast<size_t>(bb) * a.heads + head) * a.q_len + row0 + y) * a.k_len + col;
            const float v = tile[y * 17 + (lane & 15)];
            if (a.splits == 1) static_cast<T*>(a.dbias)[at] = T(v);
            else a.dbias_part[split * all + at] = v;
          }
        }
        __syncwarp();
      }
    }
    if (!ok) report_failure(a, KERNEL_DBIAS);
  }
  __syncwarp();      // the lanes of a role that one lane drained
  __syncthreads();
  tc_fence_after();
  __syncwarp();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// dk and dv = sums of the parts, in order; rows of no sequence, which no part wrote, are zero
template <typename T>
__global__ void __launch_bounds__(256)
attn_dkv_reduce_kernel(const __grid_constant__ AttnArgs a) {
  grid_dep_wait();
  const long long per = static_cast<long long>(a.kv_heads) * a.dim, all = per * a.kv_rows;
  int lo = 0, hi = a.kv_rows;
  if (a.walk == WALK_LIST) {
    lo = min(max(a.cu_k[0], 0), a.kv_rows);
    hi = min(max(a.cu_k[a.seqs], lo), a.kv_rows);
  }
  for (long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 4; i < 2 * all;
       i += static_cast<long long>(gridDim.x) * 1024) {
    const bool second = i >= all;
    const long long e = second ? i - all : i;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    const long long row = e / per;
    if (row >= lo && row < hi)
      for (int k = 0; k < a.kv_splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(a.dkv_part + 2 * k * all + i);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
      }
    *reinterpret_cast<uint2*>(static_cast<T*>(second ? a.dv : a.dk) + e) =
        make_uint2(pack16<T>(s.x, s.y), pack16<T>(s.z, s.w));
  }
  grid_dep_release();
}

// dbias = sum of the splits' parts, in order
template <typename T>
__global__ void __launch_bounds__(256)
attn_dbias_reduce_kernel(const float* __restrict__ part, T* __restrict__ out, long long n, int splits) {
  grid_dep_wait();
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * 256) {
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += part[k * n + i];
    out[i] = T(s);
  }
  grid_dep_release();
}

int item_grid(const AttnLaunch& l, bool kv) {
  const AttnArgs& a = l.a;
  long long items;
  if (a.walk == WALK_LIST)
    items = ((kv ? (static_cast<long long>(a.kv_rows) + kTileRows - 1) / kTileRows
                 : (static_cast<long long>(a.q_rows) + a.tq - 1) / a.tq) + a.seqs) * a.kv_heads;
  else
    items = static_cast<long long>(a.seqs) * (kv ? a.k_tiles : a.q_tiles) * a.kv_heads;
  if (kv) items *= a.kv_splits;
  return static_cast<int>(items < l.sms ? items : l.sms);
}

template <typename Kern>
cudaError_t go(Kern kern, const AttnLaunch& l, int grid, int smem) {
  const cudaError_t e = set_smem_once(reinterpret_cast<const void*>(kern), smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(grid), dim3(kBwdThreads), smem, l.stream, nullptr, 0, l.m, l.a);
}

}  // namespace

// Threads that share a row of the delta kernel, and its blocks: 8 per SM at most, enough for the rows
// of g and, in fp16, those of V (few queries on many keys: 16 on 100 000, 8 heads of 64, a step 7.2 ms with
// blocks for g alone, 2.4 with these, 2.3 in bf16).
static int delta_lanes(const AttnLaunch& l) { return l.a.dim <= 32 ? 4 : l.a.dim <= 64 ? 8 : 16; }
int attn_delta_grid(const AttnLaunch& l) {
  const long long per = 256 / delta_lanes(l), cap = static_cast<long long>(l.sms) * kDeltaBlocks;
  long long n = static_cast<long long>(l.a.q_rows) * l.a.heads;
  const long long nv = static_cast<long long>(l.a.kv_rows) * l.a.kv_heads;
  if (!l.bf16 && nv > n) n = nv;
  const long long need = (n + per - 1) / per;
  return static_cast<int>(need < cap ? need : cap);
}

cudaError_t launch_attn_delta(const AttnLaunch& l) {
  const int lanes = delta_lanes(l);
  const dim3 grid(attn_delta_grid(l));
  if (l.bf16) return launch_pdl(attn_delta_kernel<__nv_bfloat16>, grid, dim3(256), 0, l.stream, nullptr, 0, l.a, lanes, l.bias);
  return launch_pdl(attn_delta_kernel<__half>, grid, dim3(256), 0, l.stream, nullptr, 0, l.a, lanes, l.bias);
}

#define FTM_BY_SHAPE(KERN, CFG, GRID)                                                                        \
  if (l.dp == 64) {                                                                                          \
    if (l.bias) return l.bf16 ? go(KERN<64, true, __nv_bfloat16>, l, GRID, CFG(64, true)) : go(KERN<64, true, __half>, l, GRID, CFG(64, true));       \
    return l.bf16 ? go(KERN<64, false, __nv_bfloat16>, l, GRID, CFG(64, false)) : go(KERN<64, false, __half>, l, GRID, CFG(64, false));               \
  }                                                                                                          \
  if (l.bias) return l.bf16 ? go(KERN<128, true, __nv_bfloat16>, l, GRID, CFG(128, true)) : go(KERN<128, true, __half>, l, GRID, CFG(128, true));     \
  return l.bf16 ? go(KERN<128, false, __nv_bfloat16>, l, GRID, CFG(128, false)) : go(KERN<128, false, __half>, l, GRID, CFG(128, false));

cudaError_t launch_attn_dq(const AttnLaunch& l) {
  const int grid = item_grid(l, false);
#define DQ_SMEM(D, B) (DqCfg<D, B>::kSmem)
  FTM_BY_SHAPE(attn_dq_kernel, DQ_SMEM, grid)
}

cudaError_t launch_attn_dkv(const AttnLaunch& l) {
  const int grid = item_grid(l, true);
#define DKV_SMEM(D, B) (DkvCfg<D, B>::kSmem)
  FTM_BY_SHAPE(attn_dkv_kernel, DKV_SMEM, grid)
}

cudaError_t launch_attn_dkv_reduce(const AttnLaunch& l) {
  const long long n = static_cast<long long>(l.a.kv_rows) * l.a.kv_heads * l.a.dim / 2;   // float4s of both
  const long long need = (n + 255) / 256, cap = static_cast<long long>(l.sms) * 8;
  const dim3 grid(static_cast<unsigned>(need < cap ? need : cap));
  if (l.bf16) return launch_pdl(attn_dkv_reduce_kernel<__nv_bfloat16>, grid, dim3(256), 0, l.stream, nullptr, 0, l.a);
  return launch_pdl(attn_dkv_reduce_kernel<__half>, grid, dim3(256), 0, l.stream, nullptr, 0, l.a);
}

cudaError_t launch_attn_dbias(const AttnLaunch& l) {
  const AttnArgs& a = l.a;
  const int biases = a.seqs / a.bias_seqs;
  const long long items = static_cast<long long>(a.splits) * biases * a.heads * a.q_tiles * a.k_tiles;
  const int grid = static_cast<int>(items < l.sms ? items : l.sms);
  cudaError_t e;
  if (l.dp == 64)
    e = l.bf16 ? go(attn_dbias_kernel<64, __nv_bfloat16>, l, grid, DbCfg<64>::kSmem)
               : go(attn_dbias_kernel<64, __half>, l, grid, DbCfg<64>::kSmem);
  else
    e = l.bf16 ? go(attn_dbias_kernel<128, __nv_bfloat16>, l, grid, DbCfg<128>::kSmem)
               : go(attn_dbias_kernel<128, __half>, l, grid, DbCfg<128>::kSmem);
  if (e != cudaSuccess || a.splits == 1) return e;
  const long long n = static_cast<long long>(biases) * a.heads * a.q_len * a.k_len;
  const long long need = (n + 255) / 256, cap = static_cast<long long>(l.sms) * 8;
  const dim3 rg(static_cast<unsigned>(need < cap ? need : cap));
  if (l.bf16)
    return launch_pdl(attn_dbias_reduce_kernel<__nv_bfloat16>, rg, dim3(256), 0, l.stream, nullptr, 0,
                      static_cast<const float*>(a.dbias_part), static_cast<__nv_bfloat16*>(a.dbias), n, a.splits);
  return launch_pdl(attn_dbias_reduce_kernel<__half>, rg, dim3(256), 0, l.stream, nullptr, 0,
                    static_cast<const float*>(a.dbias_part), static_cast<__half*>(a.dbias), n, a.splits);
}

}  // namespace ftm
