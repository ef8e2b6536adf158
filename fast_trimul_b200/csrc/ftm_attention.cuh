// Shared pieces of the attention kernels (forward and backward): the problem as the
// kernels see it, the walk over its tiles, and the tcgen05 forms they need beside
// ftm_common.cuh's.
//
// A tile of queries is up to 128 rows of one key / value head: row = token * G + g over
// the G query heads that share the head, so grouped heads read K and V once, and one new
// token of a sequence still fills G rows. A tile of keys is 128 positions. Head
// dimensions are padded to DP = 64 or 128 in shared memory by the zero fill of TMA.
#pragma once

#include "ftm_kernels.h"

namespace ftm {

constexpr int kTileRows = 128;
constexpr float kLog2e = 1.4426950408889634f;

// how the items of a launch are numbered
enum : int { WALK_LIST = 0, WALK_UNIFORM = 1, WALK_CACHE = 2 };

struct AttnArgs {
  int heads, kv_heads, group, dim;
  int tq;                    // tokens per query tile: 128 / group
  int ksteps;                // 16-element steps of the head dimension
  int seqs, q_rows, kv_rows; // kv_rows: rows of one batch entry of a cache
  int q_len, k_len;          // every sequence's, where cu_q is null
  int walk;
  int q_tiles, k_tiles;      // per sequence (uniform walk)
  int causal;
  float scale;
  const int* cu_q;           // seqs + 1 first rows, on the device; null: uniform
  const int* cu_k;
  const int* k_lens;         // cache walk: keys of each sequence
  const int2* list;          // list walk: (sequence, tile), longest first
  const int* count;          // entries of the list
  const uint8_t* key_mask;   // one byte per key row, 0: not seen; may be null
  int bias_seqs;             // consecutive sequences that share a bias
  int splits;                // bias gradient: parts of those sequences
  int kv_splits;             // dk, dv: parts of the query tiles of a key tile
  float* dkv_part;           // their partial sums: [part][dk, dv][row][kv head][dim]
  // outputs and operands that are read by plain loads; contiguous unless strides follow
  void* out;
  const void* o;             // forward output (backward)
  const void* g;             // its gradient: strides in elements
  long long g_row, g_head;
  const void* v;             // (backward in fp16: its row norms)
  long long v_row, v_head;
  float2* norms;             // largest row norms (of g, of v), a pair per block of the delta kernel
  int norm_parts;
  void* out_low;             // what rounding left of the output, for the backward; or null
  float2* stats;             // (row maximum m, log2 of the row sum) per (row, head)
  float4* bstats;            // backward: (see attn_delta_kernel)
  float* part_o;             // cache walk: partial results of split sequences
  float2* part_ml;
  void* dq;
  void* dk;
  void* dv;
  void* dbias;
  float* dbias_part;
  int* err;                  // device error word the waits poll
  int* host_err;             // pinned host word that learns of an expired wait; may be null
  bool dbias_direct;         // the dq kernel writes dbias: one row per bias, all tiles met
  int test_stall;            // withhold a tile (failure tests): STALL_*
};

// a role that gave up tells the host: polling a host word in the waits themselves would cross
// PCIe on every poll (measured: 50x slower kernels), so only this write goes there. The device word
// may have been cleared since; that a kernel gave up is told all the same.
__device__ __forceinline__ void report_failure(const AttnArgs& a, int kernel) {
  if (a.host_err) {
    const int code = *reinterpret_cast<volatile int*>(a.err);
    *reinterpret_cast<volatile int*>(a.host_err) = code ? code : err_code(kernel, 0, 0);
    __threadfence_system();
  }
}

struct Item {
  int seq, head;      // sequence, key / value head
  int q0, nq;         // first global token row of the query tile, its tokens
  int pos0;           // position of that token in its sequence
  int k0, klen;       // first key row, keys of the sequence
  int kb;             // batch coordinate of the key maps
  int off;            // query i sees keys j <= i + off (causal)
  int kt0, kt1;       // tiles of keys (or of queries, in the kv walk)
  int slot;           // partial result, -1: none
  int tile;
};

__device__ __forceinline__ void seq_range(const int* cu, int i, int len, int rows, int& s, int& n) {
  if (cu) {   // clamped: whatever the array holds, no row outside the tensors is touched
    s = min(max(cu[i], 0), rows);
    n = min(max(cu[i + 1], s), rows) - s;
  } else {
    s = i * len;
    n = len;
  }
}

__device__ __forceinline__ int cache_len(const AttnArgs& a, int i) {
  return min(max(a.k_lens[i], 0), a.kv_rows);
}

// the query tile `tile` of sequence `seq` and head `head`, with the tiles of keys it sees
__device__ __forceinline__ void q_item(const AttnArgs& a, int seq, int tile, int head, Item& it) {
  int qs, qn;
  seq_range(a.cu_q, seq, a.q_len, a.q_rows, qs, qn);
  if (a.k_lens) {
    it.k0 = 0;
    it.klen = cache_len(a, seq);
    it.kb = seq;
  } else {
    seq_range(a.cu_k, seq, a.k_len, a.kv_rows, it.k0, it.klen);
    it.kb = 0;
  }
  it.seq = seq;
  it.head = head;
  it.tile = tile;
  it.pos0 = tile * a.tq;
  it.q0 = qs + it.pos0;
  it.nq = min(a.tq, qn - it.pos0);
  it.off = it.klen - qn;
  int seen = it.klen;
  if (a.causal) seen = max(0, min(seen, it.pos0 + it.nq + it.off));
  it.kt0 = 0;
  it.kt1 = (seen + kTileRows - 1) / kTileRows;
  it.slot = -1;
}

// the key tile `tile`, with the query tiles that see it
__device__ __forceinline__ void kv_item(const AttnArgs& a, int seq, int tile, int head, Item& it) {
  int qs, qn;
  seq_range(a.cu_q, seq, a.q_len, a.q_rows, qs, qn);
  seq_range(a.cu_k, seq, a.k_len, a.kv_rows, it.k0, it.klen);
  it.kb = 0;
  it.seq = seq;
  it.head = head;
  it.tile = tile;
  it.q0 = qs;
  it.nq = qn;
  it.pos0 = 0;
  it.off = it.klen - qn;
  it.kt1 = (qn + a.tq - 1) / a.tq;
  it.kt0 = a.causal ? min(it.kt1, max(0, tile * kTileRows - it.off) / a.tq) : 0;
  it.slot = -1;
}

template <bool KV>
__device__ __forceinline__ bool walk_item_whole(const AttnArgs& a, int n, Item& it) {
  if (a.walk == WALK_LIST) {
    const int w = n / a.kv_heads;
    if (w >= *a.count) return false;
    const int2 e = a.list[w];
    if (KV) kv_item(a, e.x, e.y, n % a.kv_heads, it);
    else q_item(a, e.x, e.y, n % a.kv_heads, it);
    return true;
  }
  const int tiles = KV ? a.k_tiles : a.q_tiles;
  const int rest = n / tiles;
  if (rest >= a.seqs * a.kv_heads) return false;
  if (KV) kv_item(a, rest / a.kv_heads, n % tiles, rest % a.kv_heads, it);
  else q_item(a, rest / a.kv_heads, n % tiles, rest % a.kv_heads, it);
  return true;
}

template <bool KV>
__device__ __forceinline__ bool walk_item(const AttnArgs& a, int n, Item& it) {
  if (KV && a.kv_splits > 1) {   // the parts of an item are neighbours
    const int part = n % a.kv_splits;
    if (!walk_item_whole<KV>(a, n / a.kv_splits, it)) return false;
    const int t = it.kt1 - it.kt0, t0 = it.kt0;
    it.kt0 = t0 + t * part / a.kv_splits;
    it.kt1 = t0 + t * (part + 1) / a.kv_splits;
    it.slot = part;
    return true;
  }
  return walk_item_whole<KV>(a, n, it);
}

enum : int { STALL_FWD = 1, STALL_DQ = 2, STALL_DKV = 3 };

// Named barrier that also tells whether `ok` holds in all of its threads: the warps that meet there
// go on together or leave together, so none waits for one that gave up on an expired wait.
__device__ __forceinline__ bool named_barrier_all(int id, int nthreads, bool ok) {
  int all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %3, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, %2, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(id), "r"(nthreads), "r"(ok ? 1 : 0)
      : "memory");
  __syncwarp();
  return all != 0;
}

// ------------------------------------------------------------------- tcgen05 forms
// TMEM loads, stores and (de)allocations are instructions of a whole warp (.sync.aligned). Behind a
// branch that some lanes take alone the lanes meet first: by a vote on a wait, else by __syncwarp().
// D (+)= A[tmem] * B[smem desc]; A: 16-bit pairs, 8 columns per 16-element step
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) { return pack_half2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) { return pack_bf162(a, b); }

template <typename T>
struct IsBf16 { static constexpr int v = 0; };
template <>
struct IsBf16<__nv_bfloat16> { static constexpr int v = 1; };

// two 16-bit values of a word
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (IsBf16<T>::v) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------------- MMA shapes
// Tiles in shared memory: DP / 64 blocks of 128 rows x 128 bytes (128-byte swizzle).
constexpr int kBlk = kTileRows * 128;   // bytes of one 64-element block

// The lane of a converged warp that issues its matrix instructions. These take descriptors
// from uniform registers. Behind `elect.sync` the compiler keeps the (warp-uniform) operands
// there; behind `lane == 0` it moves each one over before every instruction: about 120 clocks
// per issued MMA, 950 for one P V, which bound the whole kernel. The lanes meet first: an
// election among some of them would pick another lane, whose commits do not cover the MMAs of
// the first one.
// E: which of the two. The kernels with a bias at DP = 128 keep lane 0: with the election they once
// ended with an illegal address whose cause is not known. A check of every descriptor and TMEM
// address found none out of range, and those of the forward, dq and dkv are the same without a
// bias, where the elected form runs. Lanes that a branch had parted could then reach TMEM accesses
// one after the other, which is undefined; that is mended in all kernels. The kernels with a bias
// stay in the form that was tested.
template <bool E>
__device__ __forceinline__ bool issuer(int lane) {
  if (!E) return lane == 0;
  uint32_t p;
  __syncwarp();
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// A value that is the same in all lanes, where the compiler cannot see that it is: a broadcast
// puts it into a uniform register once. Every address a matrix instruction takes goes through
// this in front of the issuing branch; addresses that depend on loop counters otherwise cost
// moves per instruction there, 128 clocks for each 128 x 128 x 16 product instead of its 64.
template <bool E>
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return E ? __shfl_sync(0xffffffffu, x, 0) : x; }

// D[128 x 128] = A[128 rows x dim] B[128 rows x dim]^T, both K-major; `steps` 16-element steps
template <bool E>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int steps) {
  if (!E) {
    for (int k = 0; k < steps; ++k) {
      const uint32_t o = (k >> 2) * kBlk + (k & 3) * 32;
      umma_f16(d, kmajor_desc(a + o), kmajor_desc(b + o), idesc, k > 0 ? 1u : 0u);
    }
    return;
  }
  const uint64_t ad = kmajor_desc(a), bd = kmajor_desc(b);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < steps) {   // descriptor addresses count 16 bytes
      const uint64_t o = ((k >> 2) * kBlk + (k & 3) * 32) >> 4;
      umma_f16(d, ad + o, bd + o, idesc, k > 0 ? 1u : 0u);
    }
}
// D[128 x DP] (+)= A[tmem, 128 x 128] B[128 rows x DP], B MN-major
template <bool E>
__device__ __forceinline__ void mma_cols(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  if (!E) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      umma_f16_ts(d, a_tmem + k * 8, sw128_desc(b + k * 2048, kBlk, 1024), idesc, (accumulate || k > 0) ? 1u : 0u);
    return;
  }
  const uint64_t bd = sw128_desc(b, kBlk, 1024);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    umma_f16_ts(d, a_tmem + k * 8, bd + ((k * 2048) >> 4), idesc, k > 0 ? 1u : accumulate);
}

template <int DP>
__device__ __forceinline__ void load_tile4(const CUtensorMap* map, uint64_t* bar, uint8_t* dst, int c1,
                                           int c2, int c3) {
#pragma unroll
  for (int h = 0; h < DP / 64; ++h) tma_load_4d(map, bar, dst + h * kBlk, h * 64, c1, c2, c3);
}

// Rows [first, 128) of a tile set to zero by one warp: rows behind a sequence's end belong
// to somebody else, and a zero weight times what they hold need not be zero.
template <int DP>
__device__ __forceinline__ void zero_rows_from(uint8_t* tile, int first, int lane) {
  for (int h = 0; h < DP / 64; ++h)
    for (int i = first * 8 + lane; i < kTileRows * 8; i += 32)
      reinterpret_cast<uint4*>(tile + h * kBlk)[i] = make_uint4(0, 0, 0, 0);
}
// the same for the rows whose bit is clear: 32 rows at a time, DP / 8 lanes a row
template <int DP>
__device__ __forceinline__ void zero_rows_masked(uint8_t* tile, const uint32_t (&keep)[4], int lane) {
  constexpr int kLanes = DP / 8, kRows = 32 / kLanes;
  const int l = lane % kLanes;
  uint8_t* at = tile + (l >> 3) * kBlk + (l & 7) * 16;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (keep[w] == 0xffffffffu) continue;
#pragma unroll 4
    for (int i = lane / kLanes; i < 32; i += kRows)
      if (!((keep[w] >> i) & 1u)) *reinterpret_cast<uint4*>(at + (w * 32 + i) * 128) = make_uint4(0, 0, 0, 0);
  }
}

// bits of the keys of a tile that exist and are not masked (the same in every lane)
__device__ __forceinline__ void key_bits(const AttnArgs& a, const Item& it, int kt, int lane,
                                         uint32_t (&w)[4]) {
  const int c0 = kt * kTileRows;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + i * 32 + lane;
    bool on = c < it.klen;
    if (on && a.key_mask) on = a.key_mask[static_cast<size_t>(it.k0) + c] != 0;
    w[i] = __ballot_sync(0xffffffffu, on);
  }
}

// r = scale r + bias for 32 columns: chunks `chunk0` to chunk0 + 3 of row `row` of a bias block
template <typename T>
__device__ __forceinline__ void add_bias(uint32_t (&r)[32], const uint8_t* block, int row, int chunk0, float scale) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint4 b4 = *reinterpret_cast<const uint4*>(block + sw128_off(row, chunk0 + q));
    const uint32_t bw[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = q * 8 + 2 * e;
      const float2 t = __ffma2_rn(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])),
                                  make_float2(scale, scale), unpack2<T>(bw[e]));
      r[i] = __float_as_uint(t.x);
      r[i + 1] = __float_as_uint(t.y);
    }
  }
}

// The kv walk, causal: columns of a query tile in front of the first query that sees a key. `ahead`:
// tokens from the tile's first to that query. They are cut to a tile before they are multiplied:
// tokens times the heads of a group may pass 32 bits (17e6 keys in front of one query of 128 heads).
__host__ __device__ __forceinline__ int columns_before(int ahead, int group) {
  const int t = ahead < 0 ? 0 : ahead < kTileRows ? ahead : kTileRows;
  return t * group < kTileRows ? t * group : kTileRows;
}

// Rows of a query tile that hold queries, where `left` tokens of the sequence remain from its first
// token on; cut before they are multiplied, as above (a negative product would clear memory in front
// of the tile).
__host__ __device__ __forceinline__ int rows_held(int left, int tq, int group) {
  return (left < tq ? left : tq) * group;
}

// bits [0, lim) of a 128-bit row
__device__ __forceinline__ uint32_t bits_below(int lim, int word) {
  const int n = lim - word * 32;
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

// Factor from scores to powers of two. A scale of 0 becomes the least normal number: finite
// scores still meet 0, but a masked -inf does not turn into 0 * inf.
__device__ __forceinline__ float log2_scale(float scale) { return fmaxf(scale * kLog2e, 1.17549435e-38f); }

struct AttnMaps {
  CUtensorMap q, k, v, g, bias;
};

// host side ------------------------------------------------------------------------
struct AttnLaunch {
  AttnArgs a;
  AttnMaps m;
  int dp, bf16, bias, sms;
  cudaStream_t stream;
};
cudaError_t launch_attn_fwd(const AttnLaunch& l);
cudaError_t launch_attn_combine(const AttnLaunch& l, int grid_fwd);
cudaError_t launch_attn_lists(const AttnLaunch& l, int2* q_list, int q_cap, int2* k_list, int k_cap,
                              int* counts);
cudaError_t launch_pad_rows(const void* src, long long src_stride, void* dst, long long dst_stride, long long rows,
                            int cols, int sms, cudaStream_t stream);
constexpr int kDeltaBlocks = 8;   // per SM, at most
int attn_delta_grid(const AttnLaunch& l);
cudaError_t launch_attn_delta(const AttnLaunch& l);
cudaError_t launch_attn_dq(const AttnLaunch& l);
cudaError_t launch_attn_dkv(const AttnLaunch& l);
cudaError_t launch_attn_dkv_reduce(const AttnLaunch& l);
cudaError_t launch_attn_dbias(const AttnLaunch& l);
int attn_fwd_grid(const AttnLaunch& l);

}  // namespace ftm
