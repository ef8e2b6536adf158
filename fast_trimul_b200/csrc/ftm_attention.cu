// Attention forward (sm_100a): o = softmax(scale q k^T + bias) v over the keys each query
// may see, with grouped heads, packed sequences, a key mask, an additive bias shared by a
// run of sequences, or a cache whose lengths live on the device.
//
// One pass over the keys with the running maximum m and sum l of each row (fp32): a tile
// of scores S = Q K^T (tcgen05, 128 x 128, fp32 in TMEM) is read by one thread per row,
// turned into p = 2^(c (s - m)), written back to TMEM as a 16-bit operand over S, and
// O += P V accumulates in TMEM. The rounding of p to the inputs' type is the only one
// before the output's. O is rescaled only when a row's maximum grew by more than 2^8
// (p <= 256 then, harmless in fp32 sums and 16-bit p alike), so almost never.
//
// Roles of a block: warps 0-3 softmax and epilogue, warp 4 TMA, warp 5 MMA. Two blocks
// per SM (256 TMEM columns each: S / P 128, O up to 128), so one block's MMAs run under the
// other's exponentials. A 128 x 128 tile costs 8 dim clocks of MMA and 1024 clocks of the
// special function unit, so dim 128 is balanced between the two, and for smaller heads the
// exponentials are the floor. Neither bounds the kernel: at N = 384, 4 heads of 32, the counters
// show 39 % of the exponentials' rate and 14 % of the matrix instructions', and warps that wait
// for their own last result.
//
// Measured, bf16: 2 sequences of 8192 tokens, 16 heads, dim 128, 1000 us (1100 TFLOP/s);
// one of them, causal, 300 us (917); triangle attention at N = 384, 4 heads of 32, 149 us, the
// exponentials alone 49; one token over 16 caches of 9000 to 16384 tokens, 8 heads of 128
// shared by 32, 154 us (6.0 TB/s).
//
// Persistent grid. Packed sequences: a one-block kernel lists (sequence, tile) by
// descending number of key tiles, so the long ones start first. Cache: the key tiles of
// all sequences and heads are cut into equal runs, one per block; a sequence that spans
// blocks leaves partial (O, m, l) results that a second kernel joins in a fixed order.
#include "ftm_attention.cuh"

namespace ftm {
namespace {

enum : int { KERNEL_ATTN = 4 };
constexpr int kFwdThreads = 192;

template <int DP, bool BIAS>
struct FwdCfg {
  static constexpr int kTile = DP / 64 * kBlk;
  static constexpr int kStages = (DP == 64 && !BIAS) ? 2 : 1;   // K and V each
  // TMEM columns: S 0 - 127, O from 128. At DP = 64 there is room for P behind O, so the next
  // tile's scores need not wait for P V; at DP = 128 P lies over S.
  static constexpr bool kOwnP = DP == 64;
  static constexpr int kUnroll = (DP == 64 && !BIAS) ? 2 : 1;
  static constexpr int kColP = kOwnP ? 192 : 0;
  static constexpr int kOffK = kTile;
  static constexpr int kOffV = kOffK + kStages * kTile;
  static constexpr int kOffB = kOffV + kStages * kTile;
  static constexpr int kOffM = kOffB + (BIAS ? 2 * kBlk : 0);   // key bits: 2 x 16 bytes
  static constexpr int kOffBar = kOffM + 32;
  static constexpr int kSmem = kOffBar + 256 + 1024;
};

// Cache walk: block c of n takes key tiles [c per, (c + 1) per) of the concatenation over
// (sequence, head); `t` runs over it. Sequences are found from the lengths on the device.
struct CacheWalk {
  int t, end;         // this block's tiles
  int first;          // the first tile of the block's run (partials are told apart by it)
  int seq, head, base, tiles;   // current sequence: its first tile overall, tiles per head
};

__device__ __forceinline__ int cache_total(const AttnArgs& a, int lane) {
  int s = 0;
  for (int i = lane; i < a.seqs; i += 32) s += (cache_len(a, i) + kTileRows - 1) / kTileRows;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s * a.kv_heads;
}
__device__ __forceinline__ int cache_per_block(int total, int blocks) { return (total + blocks - 1) / blocks; }

__device__ __forceinline__ void cache_start(const AttnArgs& a, int lane, CacheWalk& w) {
  const int total = cache_total(a, lane);
  const int per = cache_per_block(total, gridDim.x);
  w.t = w.first = min(total, static_cast<int>(blockIdx.x) * per);
  w.end = min(total, w.t + per);
  // the sequence that holds tile w.t: a warp-wide scan over the lengths
  w.seq = 0;
  w.base = 0;
  for (int i0 = 0; i0 < a.seqs && w.t < w.end; i0 += 32) {
    const int i = i0 + lane;
    const int n = i < a.seqs ? (cache_len(a, i) + kTileRows - 1) / kTileRows * a.kv_heads : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const int all = __shfl_sync(0xffffffffu, inc, 31);
    if (w.base + all > w.t) {
      const uint32_t hit = __ballot_sync(0xffffffffu, w.base + inc > w.t);
      const int l = __ffs(hit) - 1;
      w.seq = i0 + l;
      w.base += __shfl_sync(0xffffffffu, inc - n, l);
      break;
    }
    w.base += all;
  }
}

// next run of tiles of one (sequence, head); false when the block is done
__device__ __forceinline__ bool cache_next(const AttnArgs& a, CacheWalk& w, Item& it) {
  if (w.t >= w.end) return false;
  int tiles = (cache_len(a, w.seq) + kTileRows - 1) / kTileRows;
  while (w.t >= w.base + tiles * a.kv_heads) {     // w.t < total: a later sequence holds it
    w.base += tiles * a.kv_heads;
    ++w.seq;
    tiles = (cache_len(a, w.seq) + kTileRows - 1) / kTileRows;
  }
  const int head = (w.t - w.base) / tiles;
  const int t0 = w.base + head * tiles;            // first tile of this (sequence, head)
  q_item(a, w.seq, 0, head, it);
  it.kt0 = w.t - t0;
  const int stop = min(w.end, t0 + tiles);
  it.kt1 = stop - t0;
  if (it.kt0 > 0 || it.kt1 < tiles) it.slot = 2 * blockIdx.x + (w.t == w.first ? 0 : 1);
  w.t = stop;
  return true;
}

// the items of this block, in order; every role of the block walks the same ones
struct FwdWalk {
  int n;
  CacheWalk c;
  __device__ __forceinline__ void start(const AttnArgs& a, int lane) {
    n = blockIdx.x;
    if (a.walk == WALK_CACHE) cache_start(a, lane, c);
  }
  __device__ __forceinline__ bool next(const AttnArgs& a, Item& it) {
    if (a.walk == WALK_CACHE) return cache_next(a, c, it);
    if (!walk_item<false>(a, n, it)) return false;
    n += gridDim.x;
    return true;
  }
};

// A row of scores is read twice, 32 columns at a time, the next 32 on their way under these
// ones' arithmetic: once for the maximum, once for the weights. Held in registers it would
// spill, and spilled words miss the little L1 that the tiles leave (2 x 8192 tokens, 16 heads
// of 128: 636 against 842 TFLOP/s). CUT: some keys are not seen, and their scores become -inf in
// the first pass; without, no instruction is spent on that. UN: halves of the row per step of
// the loop; 2 where the registers allow it (N = 384, 4 heads of 32 without a bias: 112 against
// 123 us), 1 with a bias (147 against 194 us, whose spills came back from L2).
template <bool BIAS, bool CUT, int UN, typename T>
__device__ __forceinline__ float row_max(uint32_t taddr, const uint8_t* sB, int row, float scale, float m,
                                         const uint32_t (&keep)[4], int lim) {
  uint32_t r[2][32];
  float top[4] = {m, -INFINITY, -INFINITY, -INFINITY};
  FTM_TMEM_LD32_NOWAIT(taddr, r[0]);
#pragma unroll UN
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int q = half * 2 + h;
      uint32_t(&x)[32] = r[h];
      tmem_wait_ld();
      if (q < 3) FTM_TMEM_LD32_NOWAIT(taddr + (q + 1) * 32, r[h ^ 1]);
      // scores with the bias go back over the plain ones
      if (BIAS) add_bias<T>(x, sB + half * kBlk, row, h * 4, scale);
      if (CUT) {
        const uint32_t bits = (half ? keep[2 + h] : keep[h]) & bits_below(lim, q);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(bits & (1u << e))) x[e] = 0xff800000u;   // -inf
      }
      if (BIAS || CUT) tmem_st32(taddr + q * 32, x);
#pragma unroll
      for (int e = 0; e < 32; e += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          top[k] = fmaxf(fmaxf(top[k], __uint_as_float(x[e + k])), __uint_as_float(x[e + k + 4]));
    }
  }
  if (BIAS || CUT) tmem_wait_st();
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// Weights 2^(c (t - ref)) of a row, written as 16-bit pairs to 64 columns at `paddr` (which may
// be the scores' own first columns: those have been read by then); their sum. `before_store`
// runs in front of the first store, `all_read` once the last scores are in registers. FAR: the
// difference first (see the call).
// (A polynomial on the FMA pipe for a fourth to a half of the exponentials measured the same
// time within 2 %: these loops are bound by latency, not by the special function unit.)
template <bool FAR, int UN, typename T, typename F, typename G>
__device__ __forceinline__ float row_weights(uint32_t taddr, uint32_t paddr, float c, float ref, F before_store,
                                             G all_read) {
  uint32_t r[2][32];
  const float nref = -ref * c;
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  FTM_TMEM_LD32_NOWAIT(taddr, r[0]);
#pragma unroll UN
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int q = half * 2 + h;
      uint32_t(&x)[32] = r[h];
      tmem_wait_ld();
      if (q < 3) FTM_TMEM_LD32_NOWAIT(taddr + (q + 1) * 32, r[h ^ 1]);
      else all_read();
      uint32_t pk[16];
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        float2 y = make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1]));
        if (FAR) y = make_float2((y.x - ref) * c, (y.y - ref) * c);
        else y = __ffma2_rn(y, make_float2(c, c), make_float2(nref, nref));
        y = make_float2(ex2(y.x), ex2(y.y));
        sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], y);
        pk[e >> 1] = pack16<T>(y.x, y.y);
      }
      if (q == 0) before_store();
      tmem_st16(paddr + q * 16, pk);
    }
  }
  return (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
}

template <int DP, bool BIAS, typename T>
__global__ void __launch_bounds__(kFwdThreads, 2)
attn_fwd_kernel(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnArgs a) {
  using C = FwdCfg<DP, BIAS>;
  constexpr int NS = C::kStages;
  constexpr bool E = !(BIAS && DP == 128);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::kOffK;
  uint8_t* sV = smem + C::kOffV;
  uint8_t* sB = smem + C::kOffB;
  uint32_t* sM = reinterpret_cast<uint32_t*>(smem + C::kOffM);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_full + 2;
  uint64_t* k_empty = k_full + NS;
  uint64_t* v_full = k_empty + NS;
  uint64_t* v_empty = v_full + NS;
  uint64_t* b_full = v_empty + NS;
  uint64_t* b_empty = b_full + 1;
  uint64_t* s_full = b_empty + 1;
  uint64_t* p_ready = s_full + 1;
  uint64_t* o_full = p_ready + 1;
  uint64_t* drain = o_full + 1;
  uint64_t* m_full = drain + 1;     // 2: key bits of a tile, written by the TMA warp
  uint64_t* m_empty = drain + 3;    // 2: read by the softmax warps and the MMA warp
  uint64_t* pv_done = drain + 5;    // O and P of a tile free again (own P columns only)
  uint64_t* s_empty = drain + 6;    // a tile's scores are all read (own P columns only)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 7);

  const int warp = uniform<E>(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < NS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(b_full, 1);
    mbar_init(b_empty, 4);
    mbar_init(s_full, 1);
    mbar_init(s_empty, 4);
    mbar_init(p_ready, 4);
    mbar_init(o_full, 1);
    mbar_init(drain, 1);
    mbar_init(pv_done, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&m_full[s], 1);
      mbar_init(&m_empty[s], 5);
    }
    fence_mbar_init();
  }
  if (warp == 5) tmem_alloc(tmem_slot, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform<E>(*tmem_slot);
  grid_dep_wait();
  grid_dep_release();

  FwdWalk walk;
  walk.start(a, lane);
  Item it;

  if (warp == 4) {
    // ------------------------------------------------------------------------ TMA
    const uint32_t q_bytes = DP / 64 * 128u * (a.group * a.tq);
    int qn = 0, kn = 0, kf = 0, vf = 0, bn = 0;   // items, tiles; loads issued of K, V, bias
    bool ok = true;
    Item next;
    for (bool more = walk.next(a, next); ok && more;) {
      it = next;
      more = walk.next(a, next);
      if (more && next.kt1 > next.kt0 && lane == 0) {
        // the next item's first tiles on their way to L2: its Q can only be loaded once the
        // last scores of this one are formed, and from HBM would come too late
#pragma unroll
        for (int h = 0; h < DP / 64; ++h) {
          tma_prefetch_l2_4d(&maps.q, h * 64, 0, next.head, next.q0);
          tma_prefetch_l2_4d(&maps.k, h * 64, next.head, next.k0 + next.kt0 * kTileRows, next.kb);
          tma_prefetch_l2_4d(&maps.v, h * 64, next.head, next.k0 + next.kt0 * kTileRows, next.kb);
        }
      }
      if (it.kt1 <= it.kt0) continue;
      ok = mbar_wait_warp(q_empty, (qn & 1) ^ 1, a.err, err_code(KERNEL_ATTN, ROLE_PRODUCER, 1));
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, q_bytes);
        load_tile4<DP>(&maps.q, q_full, sQ, 0, it.head, it.q0);
      }
      ++qn;
      for (int t = it.kt0; t < it.kt1; ++t) {
        const int s = kn % NS;
        const uint32_t ph = ((kn / NS) & 1) ^ 1;
        ok = mbar_wait_warp(&k_empty[s], ph, a.err, err_code(KERNEL_ATTN, ROLE_PRODUCER, 2)) &&
             !(a.test_stall == STALL_FWD && kn == 0);   // (then every wait of the block expires)
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&k_full[s], C::kTile);
          load_tile4<DP>(&maps.k, &k_full[s], sK + s * C::kTile, it.head, it.k0 + t * kTileRows, it.kb);
        }
        ++kf;
        if (a.key_mask) {
          // here, while the tile before is being worked on: the loads' latency is nobody else's
          const int mb = kn & 1;
          uint32_t keep[4];
          key_bits(a, it, t, lane, keep);
          ok = mbar_wait_warp(&m_empty[mb], ((kn >> 1) & 1) ^ 1, a.err, err_code(KERNEL_ATTN, ROLE_PRODUCER, 5));
          if (!ok) break;
          if (lane == 0) {
            *reinterpret_cast<uint4*>(sM + mb * 4) = make_uint4(keep[0], keep[1], keep[2], keep[3]);
            mbar_arrive(&m_full[mb]);
          }
        }
        if (BIAS) {
          ok = mbar_wait_warp(b_empty, (kn & 1) ^ 1, a.err, err_code(KERNEL_ATTN, ROLE_PRODUCER, 3));
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(b_full, 2 * kBlk);
            for (int h = 0; h < 2; ++h)
              tma_load_4d(&maps.bias, b_full, sB + h * kBlk, t * kTileRows + h * 64, it.pos0, it.head,
                          it.seq / a.bias_seqs);
          }
          ++bn;
        }
        ok = mbar_wait_warp(&v_empty[s], ph, a.err, err_code(KERNEL_ATTN, ROLE_PRODUCER, 4));
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&v_full[s], C::kTile);
          load_tile4<DP>(&maps.v, &v_full[s], sV + s * C::kTile, it.head, it.k0 + t * kTileRows, it.kb);
        }
        ++vf;
        ++kn;
      }
    }
    if (!ok) report_failure(a, KERNEL_ATTN);
    if (lane == 0) {   // copies in flight land before the block may exit
      if (qn) mbar_wait_drain(q_full, (qn - 1) & 1);
      for (int i = kf > NS ? kf - NS : 0; i < kf; ++i) mbar_wait_drain(&k_full[i % NS], (i / NS) & 1);
      for (int i = vf > NS ? vf - NS : 0; i < vf; ++i) mbar_wait_drain(&v_full[i % NS], (i / NS) & 1);
      if (bn) mbar_wait_drain(b_full, (bn - 1) & 1);
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------------ MMA
    constexpr uint32_t id_s = idesc_f16(IsBf16<T>::v, 128, 128, 0, 0);
    constexpr uint32_t id_o = idesc_f16(IsBf16<T>::v, 128, DP, 0, 1);
    const uint32_t q_addr = uniform<E>(smem_u32(sQ));
    int qn = 0, kn = 0;        // items with keys; key tiles
    bool ok = true;
    Item next;                 // found while this item's tiles are at work
    for (bool more = walk.next(a, next); ok && more;) {
      it = next;
      const int n = it.kt1 - it.kt0;
      if (n <= 0) {
        more = walk.next(a, next);
        continue;
      }
      ok = mbar_wait_warp(q_full, qn & 1, a.err, err_code(KERNEL_ATTN, ROLE_MMA, 1));
      auto arrived = [&](int j) -> bool {
        const int kj = kn + j;
        return mbar_wait_warp(&k_full[kj % NS], (kj / NS) & 1, a.err, err_code(KERNEL_ATTN, ROLE_MMA, 4));
      };
      auto scores = [&](int j) {
        const uint32_t s = uniform<E>((kn + j) % NS);
        const uint32_t k_addr = uniform<E>(smem_u32(sK + s * C::kTile)), last = uniform<E>(j == n - 1);
        tc_fence_after();
        if (issuer<E>(lane)) {
          mma_rows<E>(tmem, q_addr, k_addr, id_s, a.ksteps);
          umma_commit(s_full);
          umma_commit(&k_empty[s]);
          if (last) umma_commit(q_empty);
        }
        __syncwarp();
      };
      ok = ok && arrived(0);
      if (ok) scores(0);
      more = walk.next(a, next);
      for (int j = 0; ok && j < n; ++j) {
        // P V of tile j and the scores of tile j + 1. Where P lies over S the scores come
        // second (the tensor pipe runs in order), else as soon as tile j's have been read.
        const int kj = kn + j, s = kj % NS;
        const int kt = it.kt0 + j;
        if (C::kOwnP && j + 1 < n) {
          ok = arrived(j + 1) && mbar_wait_warp(s_empty, kj & 1, a.err, err_code(KERNEL_ATTN, ROLE_MMA, 6));
          if (!ok) break;
          scores(j + 1);
        }
        ok = mbar_wait_warp(&v_full[s], (kj / NS) & 1, a.err, err_code(KERNEL_ATTN, ROLE_MMA, 2));
        if (ok && a.key_mask)
          ok = mbar_wait_warp(&m_full[kj & 1], (kj >> 1) & 1, a.err, err_code(KERNEL_ATTN, ROLE_MMA, 5));
        if (!ok) break;
        const int valid = it.klen - kt * kTileRows;
        if (a.key_mask) {
          const uint4 w = *reinterpret_cast<const uint4*>(sM + (kj & 1) * 4);
          const uint32_t keep[4] = {w.x, w.y, w.z, w.w};
          __syncwarp();
          if (lane == 0) mbar_arrive(&m_empty[kj & 1]);
          if ((keep[0] & keep[1] & keep[2] & keep[3]) != 0xffffffffu) {
            zero_rows_masked<DP>(sV + s * C::kTile, keep, lane);
            fence_proxy_async_smem();
            __syncwarp();
          }
        } else if (valid < kTileRows) {
          zero_rows_from<DP>(sV + s * C::kTile, valid, lane);
          fence_proxy_async_smem();
          __syncwarp();
        }
        ok = mbar_wait_warp(p_ready, kj & 1, a.err, err_code(KERNEL_ATTN, ROLE_MMA, 3));
        if (!ok) break;
        tc_fence_after();
        {
          const uint32_t v_addr = uniform<E>(smem_u32(sV + s * C::kTile)), su = uniform<E>(s);
          const uint32_t more = uniform<E>(j > 0), last = uniform<E>(j + 1 == n);
          if (issuer<E>(lane)) {
            mma_cols<E>(tmem + 128, tmem + C::kColP, v_addr, id_o, more);
            umma_commit(&v_empty[su]);
            if (C::kOwnP) umma_commit(pv_done);
            if (last) umma_commit(o_full);
          }
        }
        __syncwarp();
        if (!C::kOwnP && j + 1 < n) {
          ok = arrived(j + 1);
          if (ok) scores(j + 1);
        }
      }
      kn += n;
      ++qn;
    }
    if (!ok) report_failure(a, KERNEL_ATTN);
    if (issuer<E>(lane)) {
      umma_commit(drain);
      mbar_wait_drain(drain, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax, epilogue
    const int row = threadIdx.x;
    const int tok = row / a.group, gi = row - tok * a.group;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const float c = BIAS ? kLog2e : log2_scale(a.scale);     // scores to powers of two
    int kn = 0, on = 0;
    T* out = static_cast<T*>(a.out);
    if (a.walk == WALK_LIST) {
      // rows of no sequence: in front of the first, behind the last
      const int lo = min(max(a.cu_q[0], 0), a.q_rows), hi = min(max(a.cu_q[a.seqs], lo), a.q_rows);
      const long long per = static_cast<long long>(a.heads) * a.dim / 8;
      const long long gone = (static_cast<long long>(lo) + a.q_rows - hi) * per;
      for (long long i = static_cast<long long>(blockIdx.x) * 128 + row; i < gone;
           i += static_cast<long long>(gridDim.x) * 128)
        reinterpret_cast<uint4*>(out)[i < lo * per ? i : hi * per + (i - lo * per)] = make_uint4(0, 0, 0, 0);
    }
    bool ok = true;
    for (bool more = walk.next(a, it); ok && more;) {
      const bool live = tok < it.nq && row < a.group * a.tq;
      const int seen = a.causal ? min(it.klen, it.pos0 + tok + it.off + 1) : it.klen;
      float m = -INFINITY, l = 0.f;
      for (int kt = it.kt0; kt < it.kt1; ++kt, ++kn) {
        uint32_t keep[4];
        const int lim = seen - kt * kTileRows;
        bool cut = lim < kTileRows;
        if (a.key_mask) {
          ok = mbar_wait_warp(&m_full[kn & 1], (kn >> 1) & 1, a.err, err_code(KERNEL_ATTN, ROLE_EPILOGUE, 4));
          if (!ok) break;
          const uint4 w = *reinterpret_cast<const uint4*>(sM + (kn & 1) * 4);
          keep[0] = w.x; keep[1] = w.y; keep[2] = w.z; keep[3] = w.w;
          __syncwarp();
          if (lane == 0) mbar_arrive(&m_empty[kn & 1]);
          cut = cut || (keep[0] & keep[1] & keep[2] & keep[3]) != 0xffffffffu;
        } else {
          keep[0] = keep[1] = keep[2] = keep[3] = 0xffffffffu;
        }
        cut = __any_sync(0xffffffffu, cut);
        if (BIAS) {
          ok = mbar_wait_warp(b_full, kn & 1, a.err, err_code(KERNEL_ATTN, ROLE_EPILOGUE, 1));
          if (!ok) break;
        }
        ok = mbar_wait_warp(s_full, kn & 1, a.err, err_code(KERNEL_ATTN, ROLE_EPILOGUE, 2));
        if (!ok) break;
        tc_fence_after();
        float mt;
        if (cut) mt = row_max<BIAS, true, 1, T>(lanes, sB, row, a.scale, m, keep, lim);
        else mt = row_max<BIAS, false, C::kUnroll, T>(lanes, sB, row, a.scale, m, keep, lim);
        if (BIAS) {
          __syncwarp();
          if (lane == 0) mbar_arrive(b_empty);
        }
        // P V of the tile before has read P and written O
        auto pv_wait = [&] {
          if (C::kOwnP && kn > 0) {
            ok = ok && mbar_wait_warp(pv_done, (kn - 1) & 1, a.err, err_code(KERNEL_ATTN, ROLE_EPILOGUE, 5));
            tc_fence_after();
          }
        };
        // keep the old maximum as the reference while it is within 2^8 of the new one
        const bool grow = (mt - m) * c > 8.f || (m == -INFINITY && mt > m);
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? (m == -INFINITY ? 0.f : ex2((m - mt) * c)) : 1.f;
          if (grow) {
            m = mt;
            l *= f;
          }
          if (kt > it.kt0) {
            pv_wait();
            __syncwarp();
#pragma unroll 1
            for (int q = 0; q * 32 < a.dim; ++q) {
              uint32_t o[32];
              FTM_TMEM_LD32_NOWAIT(lanes + 128 + q * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st32(lanes + 128 + q * 32, o);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        // c t - c ref in one rounding, unless a bias has put the whole row far from 0 (down to
        // the type's lowest value, used as a mask): then the difference first, which is exact
        const bool far = BIAS && __any_sync(0xffffffffu, fabsf(ref) > 1024.f);
        auto all_read = [&] {
          if (!C::kOwnP) return;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_empty);
          __syncwarp();
        };
        if (far) l += row_weights<true, 1, T>(lanes, lanes + C::kColP, c, ref, pv_wait, all_read);
        else l += row_weights<false, C::kUnroll, T>(lanes, lanes + C::kColP, c, ref, pv_wait, all_read);
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready);
      }
      if (!ok) break;
      const bool any = it.kt1 > it.kt0;
      const int slot = it.slot;
      const size_t orow = (static_cast<size_t>(it.q0) + tok) * a.heads + it.head * a.group + gi;
      more = walk.next(a, it);     // (some hundred clocks of divisions: under the last P V)
      if (any) {
        ok = mbar_wait_warp(o_full, on & 1, a.err, err_code(KERNEL_ATTN, ROLE_EPILOGUE, 3));
        if (!ok) break;
        ++on;
        tc_fence_after();
      }
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll 1
      for (int q = 0; q * 32 < a.dim; ++q) {
        uint32_t o[32];
        __syncwarp();
        if (any) {
          FTM_TMEM_LD32_NOWAIT(lanes + 128 + q * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (!live) continue;
        if (slot >= 0) {
          float* po = a.part_o + (static_cast<size_t>(slot) * a.group + gi) * DP + q * 32;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            reinterpret_cast<uint4*>(po)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (q * 32 + e * 8 >= a.dim) break;
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(o[e * 8 + k]) * inv;
            uint32_t w[4], low[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              w[k] = pack16<T>(f[2 * k], f[2 * k + 1]);
              const float2 r = unpack2<T>(w[k]);
              low[k] = pack16<T>(f[2 * k] - r.x, f[2 * k + 1] - r.y);
            }
            const size_t at = orow * a.dim + q * 32 + e * 8;
            *reinterpret_cast<uint4*>(out + at) = make_uint4(w[0], w[1], w[2], w[3]);
            if (a.out_low) *reinterpret_cast<uint4*>(static_cast<T*>(a.out_low) + at) = make_uint4(low[0], low[1], low[2], low[3]);
          }
        }
      }
      if (live && slot >= 0) a.part_ml[static_cast<size_t>(slot) * a.group + gi] = make_float2(m, l);
      if (live && a.stats)   // a row without keys: p = 2^-inf = 0 in the backward
        a.stats[orow] = l > 0.f || l != l ? make_float2(m, __log2f(l)) : make_float2(0.f, INFINITY);
      tc_fence_before();   // O read before the next item's first P V is released by p_ready
    }
    if (!ok) report_failure(a, KERNEL_ATTN);
  }
  __syncwarp();      // the lanes of a role that one lane drained
  __syncthreads();
  tc_fence_after();
  __syncwarp();
  if (warp == 5) tmem_dealloc(tmem, 256);
}

// Joins the partial results of a cache walk: block (sequence, head) x query head of the group.
// A (sequence, head) whose tiles lie in one block of the walk was written by it.
template <int DP, typename T>
__global__ void __launch_bounds__(DP)
attn_combine_kernel(const __grid_constant__ AttnArgs a, int blocks) {
  grid_dep_wait();
  const int seq = blockIdx.x / a.kv_heads, head = blockIdx.x % a.kv_heads, gi = blockIdx.y;
  __shared__ int red[2][DP / 32];
  int before = 0, all = 0;
  for (int i = threadIdx.x; i < a.seqs; i += DP) {
    const int n = (cache_len(a, i) + kTileRows - 1) / kTileRows;
    all += n;
    if (i < seq) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if ((threadIdx.x & 31) == 0) {
    red[0][threadIdx.x >> 5] = before;
    red[1][threadIdx.x >> 5] = all;
  }
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < DP / 32; ++w) {
    before += red[0][w];
    all += red[1][w];
  }
  const int tiles = (cache_len(a, seq) + kTileRows - 1) / kTileRows;
  const int per = cache_per_block(all * a.kv_heads, blocks);
  const int d = threadIdx.x;
  const size_t orow = (static_cast<size_t>(seq) * a.heads + head * a.group + gi) * a.dim + d;
  T* out = static_cast<T*>(a.out);
  if (tiles == 0) {          // no keys: zeros
    if (d < a.dim) out[orow] = T(0.f);
    return;
  }
  const int t0 = before * a.kv_heads + head * tiles, t1 = t0 + tiles;
  const int c0 = t0 / per, c1 = (t1 - 1) / per;
  if (c0 == c1) return;
  const float c = log2_scale(a.scale);
  float m = -INFINITY;
  for (int b = c0; b <= c1; ++b) {
    const int slot = 2 * b + (b == c0 && t0 != b * per ? 1 : 0);
    m = fmaxf(m, a.part_ml[static_cast<size_t>(slot) * a.group + gi].x);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f, o = 0.f;
#pragma unroll 4
  for (int b = c0; b <= c1; ++b) {
    const int slot = 2 * b + (b == c0 && t0 != b * per ? 1 : 0);
    const size_t i = static_cast<size_t>(slot) * a.group + gi;
    const float2 ml = a.part_ml[i];
    const float f = ml.x == -INFINITY && ml.y == 0.f ? 0.f : ex2((ml.x - ref) * c);
    l = fmaf(ml.y, f, l);
    o = fmaf(a.part_o[i * DP + d], f, o);
  }
  if (d < a.dim) out[orow] = T(l > 0.f || l != l ? o / l : 0.f);
}

// Lists of a packed batch's tiles, (sequence, tile), by descending number of tiles of the
// other side they meet: block 0 the query tiles, block 1 the key tiles. A counting sort
// over that number; the order within equal ones varies and changes no result.
__global__ void __launch_bounds__(1024)
attn_lists_kernel(const __grid_constant__ AttnArgs a, int2* q_list, int q_cap, int2* k_list, int k_cap,
                  int* counts) {
  constexpr int kBuckets = 1024;
  __shared__ int hist[kBuckets], warp_sum[32];
  const bool kv = blockIdx.x == 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  hist[threadIdx.x] = 0;
  grid_dep_wait();
  __syncthreads();
  for (int pass = 0; pass < 2; ++pass) {
    for (int s = warp; s < a.seqs; s += 32) {
      int q0, qn, k0, kn;
      seq_range(a.cu_q, s, 0, a.q_rows, q0, qn);
      seq_range(a.cu_k, s, 0, a.kv_rows, k0, kn);
      const int tiles = kv ? (kn + kTileRows - 1) / kTileRows : (qn + a.tq - 1) / a.tq;
      for (int t = lane; t < tiles; t += 32) {
        Item it;
        if (kv) kv_item(a, s, t, 0, it);
        else q_item(a, s, t, 0, it);
        const int cost = min(kBuckets - 1, it.kt1 - it.kt0);
        const int at = atomicAdd(&hist[kBuckets - 1 - cost], 1);
        if (pass == 1 && at < (kv ? k_cap : q_cap)) (kv ? k_list : q_list)[at] = make_int2(s, t);
      }
    }
    __syncthreads();
    if (pass == 0) {     // counts -> first places
      const int n = hist[threadIdx.x];
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) warp_sum[warp] = inc;
      __syncthreads();
      if (warp == 0) {
        int w = warp_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, w, o);
          if (lane >= o) w += v;
        }
        warp_sum[lane] = w;
      }
      __syncthreads();
      const int end = inc + (warp ? warp_sum[warp - 1] : 0);
      hist[threadIdx.x] = end - n;
      if (threadIdx.x == kBuckets - 1) counts[kv ? 1 : 0] = min(end, kv ? k_cap : q_cap);
      __syncthreads();
    }
  }
  grid_dep_release();
}

// Rows of `cols` 16-bit elements, any distance apart, to rows a multiple of 8 elements apart
// (16-byte aligned): a thread makes 8 elements of a destination row from the aligned words
// around them. Elements past `cols` are whatever follows, never read by the copies of the
// kernels above, whose maps end at `cols`.
__global__ void __launch_bounds__(256)
pad_rows_kernel(const uint16_t* __restrict__ src, long long src_stride, uint4* __restrict__ dst, int dst_vecs,
                long long rows, int cols) {
  grid_dep_wait();
  const long long n = rows * dst_vecs;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n;
       i += static_cast<long long>(gridDim.x) * 256) {
    const long long r = i / dst_vecs;
    const int c = static_cast<int>(i - r * dst_vecs) * 8;
    const uint16_t* p = src + r * src_stride + c;
    uint32_t w[4];
    if (c + 8 < cols) {     // the word behind the 8 elements still belongs to the row
      const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
      if (reinterpret_cast<uintptr_t>(p) & 2) {
        uint32_t x = q[0];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t y = q[k + 1];
          w[k] = __funnelshift_r(x, y, 16);
          x = y;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = q[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = (c + 2 * k < cols ? p[2 * k] : 0u) | ((c + 2 * k + 1 < cols ? p[2 * k + 1] : 0u) << 16);
    }
    dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  grid_dep_release();
}

template <int DP, bool BIAS, typename T>
cudaError_t go_fwd(const AttnLaunch& l) {
  auto kern = attn_fwd_kernel<DP, BIAS, T>;
  using C = FwdCfg<DP, BIAS>;
  const cudaError_t e = set_smem_once(reinterpret_cast<const void*>(kern), C::kSmem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(attn_fwd_grid(l)), dim3(kFwdThreads), C::kSmem, l.stream, nullptr, 0, l.m,
                    l.a);
}

template <bool BIAS>
cudaError_t go_fwd_dp(const AttnLaunch& l) {
  if (l.dp == 64) return l.bf16 ? go_fwd<64, BIAS, __nv_bfloat16>(l) : go_fwd<64, BIAS, __half>(l);
  return l.bf16 ? go_fwd<128, BIAS, __nv_bfloat16>(l) : go_fwd<128, BIAS, __half>(l);
}

}  // namespace

// Two blocks per SM (one with a bias at DP = 128, whose shared memory allows no second), never
// more than there are items: an item of the list per head, or a key tile of the cache.
int attn_fwd_grid(const AttnLaunch& l) {
  const AttnArgs& a = l.a;
  const long long slots = static_cast<long long>(l.sms) * ((l.bias && l.dp == 128) ? 1 : 2);
  long long items;
  if (a.walk == WALK_LIST)
    items = (static_cast<long long>(a.q_rows + a.tq - 1) / a.tq + a.seqs) * a.kv_heads;
  else if (a.walk == WALK_UNIFORM)
    items = static_cast<long long>(a.seqs) * a.q_tiles * a.kv_heads;
  else
    items = static_cast<long long>(a.seqs) * a.kv_heads * ((a.kv_rows + kTileRows - 1) / kTileRows);
  return static_cast<int>(items < slots ? (items > 0 ? items : 1) : slots);
}

cudaError_t launch_attn_fwd(const AttnLaunch& l) { return l.bias ? go_fwd_dp<true>(l) : go_fwd_dp<false>(l); }

cudaError_t launch_attn_combine(const AttnLaunch& l, int grid_fwd) {
  const dim3 grid(l.a.seqs * l.a.kv_heads, l.a.group);
  if (l.dp == 64)
    return l.bf16 ? launch_pdl(attn_combine_kernel<64, __nv_bfloat16>, grid, dim3(64), 0, l.stream, nullptr, 0, l.a, grid_fwd)
                  : launch_pdl(attn_combine_kernel<64, __half>, grid, dim3(64), 0, l.stream, nullptr, 0, l.a, grid_fwd);
  return l.bf16 ? launch_pdl(attn_combine_kernel<128, __nv_bfloat16>, grid, dim3(128), 0, l.stream, nullptr, 0, l.a, grid_fwd)
                : launch_pdl(attn_combine_kernel<128, __half>, grid, dim3(128), 0, l.stream, nullptr, 0, l.a, grid_fwd);
}

cudaError_t launch_pad_rows(const void* src, long long src_stride, void* dst, long long dst_stride, long long rows,
                            int cols, int sms, cudaStream_t stream) {
  const long long need = (rows * (dst_stride / 8) + 255) / 256, cap = static_cast<long long>(sms) * 8;
  return launch_pdl(pad_rows_kernel, dim3(static_cast<unsigned>(need < cap ? need : cap)), dim3(256), 0, stream,
                    nullptr, 0, static_cast<const uint16_t*>(src), src_stride, static_cast<uint4*>(dst),
                    static_cast<int>(dst_stride / 8), rows, cols);
}

cudaError_t launch_attn_lists(const AttnLaunch& l, int2* q_list, int q_cap, int2* k_list, int k_cap,
                              int* counts) {
  return launch_pdl(attn_lists_kernel, dim3(k_list ? 2 : 1), dim3(1024), 0, l.stream, nullptr, 0, l.a, q_list,
                    q_cap, k_list, k_cap, counts);
}

}  // namespace ftm
