// C entry points of attention (declared in include/fast_trimul_b200.h): argument checks,
// tensor maps, workspaces and the launch sequences.
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "ftm_attention.cuh"

using namespace ftm;

namespace {

constexpr int64_t kMaxRows = 0x7fffffff - 1024;    // row numbers are 32-bit in the kernels

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// a stride the tensor map can take; dimensions of extent 1 are never stepped over
bool stride_ok(int64_t stride, int64_t extent) {
  return extent <= 1 || (stride > 0 && stride % 8 == 0 && stride < (int64_t(1) << 38));
}

int check(const ftm_attention* p) {
  if (!p || !p->q || !p->k || !p->v || !p->out) return FTM_BAD_ARGUMENT;
  if (p->dtype != FTM_F16 && p->dtype != FTM_BF16) return FTM_BAD_DTYPE;
  if (!(p->scale >= 0.f) || !std::isfinite(p->scale)) return FTM_BAD_ARGUMENT;
  if (p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->heads / p->kv_heads > kTileRows)
    return FTM_BAD_SHAPE;
  if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8) return FTM_BAD_SHAPE;
  if (p->sequences < 1 || p->q_rows < 1 || p->kv_rows < 1 || p->q_rows > kMaxRows || p->kv_rows > kMaxRows)
    return FTM_BAD_SHAPE;
  // item numbers are 32-bit too: tiles of either side times heads (of a cache: of every sequence)
  const int64_t q_tiles = p->q_rows / (kTileRows / (p->heads / p->kv_heads)) + p->sequences;
  const int64_t k_tiles = p->kv_rows / kTileRows + 1;
  if (q_tiles * p->kv_heads > kMaxRows ||
      (p->kv_lengths ? k_tiles * p->kv_heads > kMaxRows / p->sequences
                     : (k_tiles + p->sequences) * p->kv_heads > kMaxRows))
    return FTM_BAD_SHAPE;
  if (p->kv_lengths) {
    if (p->cu_q || p->cu_k || p->key_mask || p->bias || p->causal || p->stats || p->out_low) return FTM_BAD_ARGUMENT;
    if (p->q_len != 1 || p->q_rows != p->sequences) return FTM_BAD_SHAPE;
    if (!stride_ok(p->k_batch_stride, p->sequences) || !stride_ok(p->v_batch_stride, p->sequences))
      return FTM_BAD_ALIGN;
  } else if (p->cu_q || p->cu_k) {
    if (!p->cu_q || !p->cu_k || p->bias) return FTM_BAD_ARGUMENT;
  } else {
    if (p->q_len < 1 || p->kv_len < 1 || int64_t(p->q_len) * p->sequences != p->q_rows ||
        int64_t(p->kv_len) * p->sequences != p->kv_rows)
      return FTM_BAD_SHAPE;
  }
  if (p->bias) {
    if (p->causal) return FTM_BAD_ARGUMENT;     // its gradient's kernel knows key masks only
    if (p->heads != p->kv_heads || p->bias_seqs < 1 || p->sequences % p->bias_seqs) return FTM_BAD_SHAPE;
    if (!aligned(p->bias, 16) || !stride_ok(p->bias_row_stride, p->q_len) ||
        !stride_ok(p->bias_head_stride, p->heads) ||
        !stride_ok(p->bias_batch_stride, p->sequences / p->bias_seqs))
      return FTM_BAD_ALIGN;
  }
  if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->out, 16) ||
      !aligned(p->stats, 8) || !aligned(p->out_low, 16) || !stride_ok(p->q_row_stride, p->q_rows) ||
      !stride_ok(p->q_head_stride, p->heads) || !stride_ok(p->k_row_stride, p->kv_rows) ||
      !stride_ok(p->k_head_stride, p->kv_heads) || !stride_ok(p->v_row_stride, p->kv_rows) ||
      !stride_ok(p->v_head_stride, p->kv_heads))
    return FTM_BAD_ALIGN;
  return FTM_OK;
}

uint64_t bytes_or(int64_t stride, int64_t extent, uint64_t other) {
  return extent > 1 ? static_cast<uint64_t>(stride) * 2 : other;
}

// q or its gradient: (dim, group, kv head, row), boxes of 64 x group x 1 x tq
bool q_map(CUtensorMap* m, const ftm_attention* p, const void* base, int64_t rs, int64_t hs) {
  const uint64_t G = p->heads / p->kv_heads, one = 256;
  const uint64_t dims[4] = {uint64_t(p->head_dim), G, uint64_t(p->kv_heads), uint64_t(p->q_rows)};
  const uint64_t strides[3] = {bytes_or(hs, p->heads, one), bytes_or(hs * int64_t(G), p->kv_heads, one),
                               bytes_or(rs, p->q_rows, one)};
  const uint32_t box[4] = {64, uint32_t(G), 1, uint32_t(kTileRows / G)};
  return make_tensor_map(m, p->dtype == FTM_BF16, 4, base, dims, strides, box);
}

// k or v: (dim, head, row, batch entry), boxes of 64 x 1 x 128 x 1
bool kv_map(CUtensorMap* m, const ftm_attention* p, const void* base, int64_t rs, int64_t hs, int64_t bs) {
  const uint64_t B = p->kv_lengths ? p->sequences : 1, one = 256;
  const uint64_t dims[4] = {uint64_t(p->head_dim), uint64_t(p->kv_heads), uint64_t(p->kv_rows), B};
  const uint64_t strides[3] = {bytes_or(hs, p->kv_heads, one), bytes_or(rs, p->kv_rows, one),
                               bytes_or(bs, int64_t(B), one)};
  const uint32_t box[4] = {64, 1, kTileRows, 1};
  return make_tensor_map(m, p->dtype == FTM_BF16, 4, base, dims, strides, box);
}

bool bias_map(CUtensorMap* m, const ftm_attention* p) {
  const uint64_t B = p->sequences / p->bias_seqs, one = 256;
  const uint64_t dims[4] = {uint64_t(p->kv_len), uint64_t(p->q_len), uint64_t(p->heads), B};
  const uint64_t strides[3] = {bytes_or(p->bias_row_stride, p->q_len, one),
                               bytes_or(p->bias_head_stride, p->heads, one),
                               bytes_or(p->bias_batch_stride, int64_t(B), one)};
  const uint32_t box[4] = {64, kTileRows, 1, 1};
  return make_tensor_map(m, p->dtype == FTM_BF16, 4, p->bias, dims, strides, box);
}

int caps(const ftm_attention* p, int& q_cap, int& k_cap) {
  const int tq = kTileRows / (p->heads / p->kv_heads);
  q_cap = static_cast<int>((p->q_rows + tq - 1) / tq + p->sequences);
  k_cap = static_cast<int>((p->kv_rows + kTileRows - 1) / kTileRows + p->sequences);
  return 0;
}

// lists: [counts 256 B][query tiles][key tiles, when training]
struct FwdSpace {
  size_t q_list, k_list, part_o, part_ml, total;
};
FwdSpace fwd_space(const ftm_attention* p, int train, int sms) {
  FwdSpace w{};
  if (p->kv_lengths) {
    const size_t slots = size_t(4) * sms * (p->heads / p->kv_heads);   // two per block, two blocks per SM
    w.part_ml = slots * 128 * sizeof(float);
    w.total = w.part_ml + up256(slots * sizeof(float2));
  } else if (p->cu_q) {
    int qc, kc;
    caps(p, qc, kc);
    w.q_list = 256;
    w.k_list = w.q_list + up256(size_t(qc) * sizeof(int2));
    w.total = w.k_list + (train ? up256(size_t(kc) * sizeof(int2)) : 0);
  }
  return w;
}

// backward: [row constants][row norms, fp16][parts of dk and dv][parts of the bias gradient]
struct BwdSpace {
  size_t norms, kv_part, part, total;
  int splits, kv_splits;
};
BwdSpace bwd_space(const ftm_attention* p, int want_dbias, int sms) {
  BwdSpace w{};
  w.norms = up256(size_t(p->q_rows) * p->heads * sizeof(float4));
  w.kv_part = w.norms + (p->dtype == FTM_F16 ? up256(size_t(sms) * kDeltaBlocks * sizeof(float2)) : 0);
  w.part = w.kv_part;
  // Few key tiles (one key / value head, a few thousand keys) leave SMs idle: the query tiles of
  // each are split over up to 8 blocks, at least 4 tiles each, and the parts added up. One
  // sequence of 2319 tokens, 8 heads on one, dim 128: the training step 370 us unsplit, 148 us
  // with the parts and their sums. (That shape is the rule's only measurement; it goes by the average
  // length, so that one long sequence among many short ones may stay unsplit.)
  const int64_t tq = kTileRows / (p->heads / p->kv_heads);
  const int64_t k_items = (p->cu_q ? p->kv_rows / kTileRows + p->sequences
                                   : int64_t(p->sequences) * ((p->kv_len + kTileRows - 1) / kTileRows)) * p->kv_heads;
  const int64_t q_tiles = (p->q_rows / p->sequences + tq - 1) / tq;
  int64_t ks = sms / (k_items > 0 ? k_items : 1);
  if (ks > 8) ks = 8;
  if (ks > q_tiles / 4) ks = q_tiles / 4;
  w.kv_splits = ks < 2 ? 1 : static_cast<int>(ks);
  if (w.kv_splits > 1)
    w.part += up256(size_t(2) * w.kv_splits * p->kv_rows * p->kv_heads * p->head_dim * sizeof(float));
  w.total = w.part;
  w.splits = 1;
  if (want_dbias && p->bias) {
    // tiles of the bias are few: the rows that share it are split until the SMs are busy
    const int64_t biases = p->sequences / p->bias_seqs;
    const int64_t tiles = biases * p->heads * ((p->q_len + kTileRows - 1) / kTileRows) *
                          ((p->kv_len + kTileRows - 1) / kTileRows);
    int64_t splits = sms / tiles;      // one item per SM at most: a second wave would be mostly idle
    if (splits > p->bias_seqs) splits = p->bias_seqs;
    if (splits < 1) splits = 1;
    w.splits = static_cast<int>(splits);
    if (splits > 1)
      w.total += up256(size_t(splits) * biases * p->heads * p->q_len * p->kv_len * sizeof(float));
  }
  return w;
}

// everything of a launch that does not depend on the pass
bool fill(AttnLaunch& l, const ftm_attention* p, int dev, int* err, int* host_err, ftm_stream_t stream) {
  l.dp = p->head_dim <= 64 ? 64 : 128;
  l.bf16 = p->dtype == FTM_BF16;
  l.bias = p->bias != nullptr;
  l.sms = device_sms(dev);
  l.stream = reinterpret_cast<cudaStream_t>(stream);
  AttnArgs& a = l.a;
  a.heads = p->heads;
  a.kv_heads = p->kv_heads;
  a.group = p->heads / p->kv_heads;
  a.dim = p->head_dim;
  a.tq = kTileRows / a.group;
  a.ksteps = (p->head_dim + 15) / 16;
  a.seqs = p->sequences;
  a.q_rows = static_cast<int>(p->q_rows);
  a.kv_rows = static_cast<int>(p->kv_rows);
  a.q_len = p->q_len;
  a.k_len = p->kv_len;
  a.walk = p->kv_lengths ? WALK_CACHE : p->cu_q ? WALK_LIST : WALK_UNIFORM;
  if (a.walk == WALK_UNIFORM) {
    a.q_tiles = (p->q_len + a.tq - 1) / a.tq;
    a.k_tiles = (p->kv_len + kTileRows - 1) / kTileRows;
  }
  a.causal = p->causal != 0;
  a.scale = p->scale;
  a.cu_q = p->cu_q;
  a.cu_k = p->cu_k;
  a.k_lens = p->kv_lengths;
  a.key_mask = p->key_mask;
  a.bias_seqs = p->bias ? p->bias_seqs : 1;
  a.splits = a.kv_splits = 1;
  a.out = p->out;
  a.stats = reinterpret_cast<float2*>(p->stats);
  a.out_low = p->out_low;
  a.err = err;
  a.host_err = host_err;
  const char* stall = getenv("FTM_TEST_STALL");
  a.test_stall = !stall ? 0
                 : strcmp(stall, "attention") == 0     ? STALL_FWD
                 : strcmp(stall, "attention_dq") == 0  ? STALL_DQ
                 : strcmp(stall, "attention_dkv") == 0 ? STALL_DKV
                                                       : 0;
  return q_map(&l.m.q, p, p->q, p->q_row_stride, p->q_head_stride) &&
         kv_map(&l.m.k, p, p->k, p->k_row_stride, p->k_head_stride, p->k_batch_stride) &&
         kv_map(&l.m.v, p, p->v, p->v_row_stride, p->v_head_stride, p->v_batch_stride) &&
         (!p->bias || bias_map(&l.m.bias, p));
}

}  // namespace

extern "C" {

size_t ftm_attention_workspace_bytes(const ftm_attention* p, int32_t train) {
  if (check(p) != FTM_OK) return 0;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    const int n = device_sms(dev);
    if (n > 0) sms = n;
  }
  return fwd_space(p, train, sms).total;
}

int ftm_attention_fwd(const ftm_attention* p, int32_t train, void* workspace, size_t workspace_bytes,
                      int* err_word, int* host_word, ftm_stream_t stream) {
  set_last_launch_count(0);
  const int st = check(p);
  if (st != FTM_OK) return st;
  if (!err_word) return FTM_BAD_ARGUMENT;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || ftm_device_supported(dev) != 1) return FTM_UNSUPPORTED_ARCH;
  const FwdSpace w = fwd_space(p, train, device_sms(dev));
  if (w.total && (!workspace || workspace_bytes < w.total)) return FTM_BAD_WORKSPACE;
  if (!aligned(workspace, 256)) return FTM_BAD_ALIGN;
  AttnLaunch l{};
  if (!fill(l, p, dev, err_word, host_word, stream)) return FTM_LAUNCH_FAILED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  int launches = 1;
  if (l.a.walk == WALK_LIST) {
    int qc, kc;
    caps(p, qc, kc);
    int2* ql = reinterpret_cast<int2*>(ws + w.q_list);
    int2* kl = train ? reinterpret_cast<int2*>(ws + w.k_list) : nullptr;
    l.a.list = ql;
    l.a.count = reinterpret_cast<int*>(ws);
    if (launch_attn_lists(l, ql, qc, kl, kc, reinterpret_cast<int*>(ws)) != cudaSuccess) return FTM_LAUNCH_FAILED;
    ++launches;
  } else if (l.a.walk == WALK_CACHE) {
    l.a.part_o = reinterpret_cast<float*>(ws);
    l.a.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  }
  if (launch_attn_fwd(l) != cudaSuccess) return FTM_LAUNCH_FAILED;
  if (l.a.walk == WALK_CACHE) {
    if (launch_attn_combine(l, attn_fwd_grid(l)) != cudaSuccess) return FTM_LAUNCH_FAILED;
    ++launches;
  }
  set_last_launch_count(launches);
  return FTM_OK;
}

int ftm_pad_rows(const void* src, int64_t src_stride, void* dst, int64_t dst_stride, int64_t rows, int32_t cols,
                 ftm_stream_t stream) {
  set_last_launch_count(0);
  if (!src || !dst) return FTM_BAD_ARGUMENT;
  if (rows < 1 || cols < 1 || src_stride < cols || dst_stride < cols || dst_stride % 8 || dst_stride > (1 << 30))
    return FTM_BAD_SHAPE;
  if (!aligned(src, 2) || !aligned(dst, 16)) return FTM_BAD_ALIGN;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || ftm_device_supported(dev) != 1) return FTM_UNSUPPORTED_ARCH;
  if (launch_pad_rows(src, src_stride, dst, dst_stride, rows, cols, device_sms(dev),
                      reinterpret_cast<cudaStream_t>(stream)) != cudaSuccess)
    return FTM_LAUNCH_FAILED;
  set_last_launch_count(1);
  return FTM_OK;
}

size_t ftm_attention_bwd_workspace_bytes(const ftm_attention* p, int32_t want_dbias) {
  if (check(p) != FTM_OK || p->kv_lengths) return 0;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) {
    const int n = device_sms(dev);
    if (n > 0) sms = n;
  }
  return bwd_space(p, want_dbias, sms).total;
}

int ftm_attention_bwd(const ftm_attention* p, const void* grad, int64_t grad_row_stride,
                      int64_t grad_head_stride, void* fwd_workspace, size_t fwd_workspace_bytes,
                      void* workspace, size_t workspace_bytes, void* dq, void* dk, void* dv, void* dbias,
                      int* err_word, int* host_word, ftm_stream_t stream) {
  set_last_launch_count(0);
  const int st = check(p);
  if (st != FTM_OK) return st;
  if (!grad || !p->stats || !err_word || p->kv_lengths || (!dq && !dk && !dbias) || !dk != !dv ||
      (dbias && !p->bias))
    return FTM_BAD_ARGUMENT;
  if (!aligned(grad, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16) ||
      !stride_ok(grad_row_stride, p->q_rows) || !stride_ok(grad_head_stride, p->heads))
    return FTM_BAD_ALIGN;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || ftm_device_supported(dev) != 1) return FTM_UNSUPPORTED_ARCH;
  const int sms = device_sms(dev);
  const BwdSpace w = bwd_space(p, dbias != nullptr, sms);
  const FwdSpace f = fwd_space(p, 1, sms);
  if (!workspace || workspace_bytes < w.total || (f.total && (!fwd_workspace || fwd_workspace_bytes < f.total)))
    return FTM_BAD_WORKSPACE;
  if (!aligned(workspace, 256) || !aligned(fwd_workspace, 256)) return FTM_BAD_ALIGN;
  AttnLaunch l{};
  if (!fill(l, p, dev, err_word, host_word, stream) || !q_map(&l.m.g, p, grad, grad_row_stride, grad_head_stride))
    return FTM_LAUNCH_FAILED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  l.a.o = p->out;
  l.a.g = grad;
  l.a.g_row = p->q_rows > 1 ? grad_row_stride : 0;
  l.a.g_head = p->heads > 1 ? grad_head_stride : 0;
  l.a.v = p->v;
  l.a.v_row = p->kv_rows > 1 ? p->v_row_stride : 0;
  l.a.v_head = p->kv_heads > 1 ? p->v_head_stride : 0;
  l.a.bstats = reinterpret_cast<float4*>(ws);
  l.a.norms = reinterpret_cast<float2*>(ws + w.norms);
  l.a.norm_parts = attn_delta_grid(l);
  l.a.dq = dq;
  l.a.dk = dk;
  l.a.dv = dv;
  l.a.dbias = dbias;
  l.a.dbias_part = reinterpret_cast<float*>(ws + w.part);
  l.a.splits = w.splits;
  l.a.kv_splits = w.kv_splits;
  l.a.dkv_part = reinterpret_cast<float*>(ws + w.kv_part);
  l.a.dbias_direct = dbias && dq && p->bias_seqs == 1 && l.dp == 64;
  int launches = 1;
  if (launch_attn_delta(l) != cudaSuccess) return FTM_LAUNCH_FAILED;
  uint8_t* lists = static_cast<uint8_t*>(fwd_workspace);
  if (dq) {
    if (l.a.walk == WALK_LIST) {
      l.a.list = reinterpret_cast<const int2*>(lists + f.q_list);
      l.a.count = reinterpret_cast<const int*>(lists);
    }
    if (launch_attn_dq(l) != cudaSuccess) return FTM_LAUNCH_FAILED;
    ++launches;
  }
  if (dk) {
    if (l.a.walk == WALK_LIST) {
      l.a.list = reinterpret_cast<const int2*>(lists + f.k_list);
      l.a.count = reinterpret_cast<const int*>(lists) + 1;
    }
    if (launch_attn_dkv(l) != cudaSuccess) return FTM_LAUNCH_FAILED;
    ++launches;
    if (w.kv_splits > 1) {
      if (launch_attn_dkv_reduce(l) != cudaSuccess) return FTM_LAUNCH_FAILED;
      ++launches;
    }
  }
  if (dbias && !l.a.dbias_direct) {
    if (launch_attn_dbias(l) != cudaSuccess) return FTM_LAUNCH_FAILED;
    launches += w.splits > 1 ? 2 : 1;
  }
  set_last_launch_count(launches);
  return FTM_OK;
}

}  // extern "C"
