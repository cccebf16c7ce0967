// C-ABI entry points around the paged cache (include/bw_attn.h): rotary tables
// and rotations, cache writes and reads, decode over the 8-bit cache.  Argument
// checks come before anything touches the device.
#include <cmath>

#include "../../include/bw_attn.h"
#include "kernels.h"

namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// One page of the cache: 8, 16, 32, 64 or a multiple of 64 tokens.
bool page_size_ok(int n) { return n >= 8 && ((n <= 64 && 64 % n == 0) || n % 64 == 0); }

int cache_dtype_ok(int dtype) { return dtype == BW_BF16 || dtype == BW_E4M3; }

constexpr double kTwoPi = 6.283185307179586476925286766559;

// Turns per position of pair i under the scaling; *magnitude: the factor on cos and sin.
int schedule(int R, const bw_rope_scaling* sc, double* turns, double* magnitude) {
  const bw_rope_scaling none = {BW_ROPE_NONE, 10000.0, 1.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
  const bw_rope_scaling& s = sc ? *sc : none;
  if (!(s.base > 1.0) || !std::isfinite(s.base)) return BW_ERR_SHAPE;
  if (s.kind < BW_ROPE_NONE || s.kind > BW_ROPE_BANDS) return BW_ERR_SHAPE;
  if (!(s.attention_factor >= 0.0) || !std::isfinite(s.attention_factor)) return BW_ERR_SHAPE;
  const bool scaled = s.kind != BW_ROPE_NONE;
  if (scaled && (!(s.factor > 0.0) || !std::isfinite(s.factor))) return BW_ERR_SHAPE;
  const bool bands = s.kind == BW_ROPE_YARN || s.kind == BW_ROPE_BANDS;
  if (bands && (!(s.original_length > 0.0) || !std::isfinite(s.original_length))) return BW_ERR_SHAPE;
  // a zero bound means its usual value
  const double fast = s.beta_fast != 0.0 ? s.beta_fast : 32.0, slow = s.beta_slow != 0.0 ? s.beta_slow : 1.0;
  const double low_f = s.low_freq_factor != 0.0 ? s.low_freq_factor : 1.0;
  const double high_f = s.high_freq_factor != 0.0 ? s.high_freq_factor : 4.0;
  if (s.kind == BW_ROPE_YARN && !(fast > 0.0 && slow > 0.0 && std::isfinite(fast) && std::isfinite(slow)))
    return BW_ERR_SHAPE;
  if (s.kind == BW_ROPE_BANDS && !(low_f > 0.0 && high_f > low_f && std::isfinite(high_f))) return BW_ERR_SHAPE;
  double base = s.base;
  if (s.kind == BW_ROPE_NTK) {
    if (R <= 2) return BW_ERR_SHAPE;
    base *= std::pow(s.factor, (double)R / (R - 2));
  }
  double lo = 0.0, hi = 1.0;
  if (s.kind == BW_ROPE_YARN) {
    // the pair that makes n turns over the original length: R ln(L / 2 pi n) / (2 ln base)
    const auto pair_of = [&](double n) { return R * std::log(s.original_length / (kTwoPi * n)) / (2.0 * std::log(base)); };
    lo = std::fmax(std::floor(pair_of(fast)), 0.0);
    hi = std::fmin(std::ceil(pair_of(slow)), R - 1.0);
    if (hi == lo) hi += 0.001;
  }
  for (int i = 0; i < R / 2; ++i) {
    double f = std::pow(base, -2.0 * i / R);   // radians per position
    if (s.kind == BW_ROPE_LINEAR) {
      f /= s.factor;
    } else if (s.kind == BW_ROPE_YARN) {
      const double r = std::fmin(std::fmax((i - lo) / (hi - lo), 0.0), 1.0);
      f = f / s.factor * r + f * (1.0 - r);
    } else if (s.kind == BW_ROPE_BANDS) {
      const double n = s.original_length * f / kTwoPi;   // turns over the original length
      const double r = std::fmin(std::fmax((n - low_f) / (high_f - low_f), 0.0), 1.0);
      f = f / s.factor * (1.0 - r) + f * r;
    }
    turns[i] = f / kTwoPi;
  }
  *magnitude = s.attention_factor > 0.0 ? s.attention_factor
               : s.kind == BW_ROPE_YARN && s.factor > 1.0 ? 0.1 * std::log(s.factor) + 1.0
                                                          : 1.0;
  return BW_OK;
}

// Strides of one rope tensor; a dimension of one element has no stride to check.
int rope_tensor(bw::RopeTensor* t, const void* in, void* out, const int64_t* xs, const int64_t* ys, int B, int H, int S,
                int D, int mult) {
  const int64_t dense[3] = {(int64_t)H * S * D, (int64_t)S * D, D};
  const int n[3] = {B, H, S};
  int64_t x[3], y[3];
  for (int i = 0; i < 3; ++i) {
    x[i] = n[i] == 1 ? 0 : xs ? xs[i] : dense[i];
    y[i] = n[i] == 1 ? 0 : ys ? ys[i] : dense[i];
    if (n[i] > 1 && (x[i] <= 0 || y[i] <= 0 || x[i] % mult || y[i] % mult)) return BW_ERR_ALIGN;
  }
  if (!aligned(in, 16) || !aligned(out, 16)) return BW_ERR_ALIGN;
  t->in = in;
  t->out = out;
  t->in_sb = x[0]; t->in_sh = x[1]; t->in_ss = x[2];
  t->out_sb = y[0]; t->out_sh = y[1]; t->out_ss = y[2];
  t->H = H;
  return BW_OK;
}

bool in_place(const bw::RopeTensor& t) {
  return t.in == t.out && t.in_sb == t.out_sb && t.in_sh == t.out_sh && t.in_ss == t.out_ss;
}

// Most blocks of a decode (its workspace's size does not depend on the device).
constexpr int kMaxDecodeBlocks = 1024;

int decode_groups(int Hkv, int blocks) {
  const int n = blocks / Hkv;
  return n < 1 ? 1 : n;
}

}  // namespace

extern "C" {

int bw_rope_table(float* table, int64_t length, int rotary_dim, int64_t first, const bw_rope_scaling* scaling,
                  void* stream) {
  if (!table) return BW_ERR_NULL;
  if (length <= 0 || rotary_dim < 2 || rotary_dim % 2 || rotary_dim > bw::kMaxRotaryDim || first < 0 ||
      first > (int64_t(1) << 31) - length || length > (int64_t(1) << 31))
    return BW_ERR_SHAPE;
  if (!aligned(table, 4)) return BW_ERR_ALIGN;
  bw::RopeTableParams p{};
  double magnitude = 1.0;
  int rc = schedule(rotary_dim, scaling, p.turns, &magnitude);
  if (rc != BW_OK) return rc;
  bw::DeviceInfo dev;
  rc = bw::device_info(stream, &dev);
  if (rc != BW_OK) return rc;
  p.table = table;
  p.length = length;
  p.first = first;
  p.R = rotary_dim;
  p.magnitude = (float)magnitude;
  return bw::launch_rope_table(p, dev.num_sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? BW_OK : BW_ERR_CUDA;
}

int bw_rope(const void* Q, void* Q_out, const void* K, void* K_out, int dtype, int B, int Hq, int Hkv, int S, int D,
            const int64_t* q_strides, const int64_t* q_out_strides, const int64_t* k_strides,
            const int64_t* k_out_strides, const float* cos_sin_cache, int64_t cache_seq_len, int rotary_dim,
            const int* positions, int pos_offset, int interleaved, int inverse, void* stream) {
  if (!Q || !Q_out || !cos_sin_cache) return BW_ERR_NULL;
  if (!K != !K_out) return BW_ERR_NULL;
  if (dtype != BW_BF16 && dtype != BW_F32) return BW_ERR_SHAPE;
  if (B <= 0 || Hq <= 0 || S <= 0 || (K ? Hkv <= 0 : Hkv != 0) || Hq > 65536 || Hkv > 65536) return BW_ERR_SHAPE;
  if ((Hq + 1) / 2 + (Hkv + 1) / 2 > 65535) return BW_ERR_SHAPE;   // groups of two heads along a grid's axis
  if (D <= 0 || D % 8 || D > bw::kMaxRotaryDim || rotary_dim < 16 || rotary_dim % 16 || rotary_dim > D)
    return BW_ERR_SHAPE;
  if (cache_seq_len < 0 || (int64_t)B * S >= (int64_t(1) << 31)) return BW_ERR_SHAPE;
  if (!aligned(cos_sin_cache, 16) || !aligned(positions, 4)) return BW_ERR_ALIGN;
  bw::RopeParams p{};
  const int mult = dtype == BW_BF16 ? 8 : 4;
  int rc = rope_tensor(&p.q, Q, Q_out, q_strides, q_out_strides, B, Hq, S, D, mult);
  if (rc == BW_OK && K) rc = rope_tensor(&p.k, K, K_out, k_strides, k_out_strides, B, Hkv, S, D, mult);
  if (rc != BW_OK) return rc;
  p.B = B;
  p.S = S;
  p.D = D;
  p.R = rotary_dim;
  // two vectors of 16 bytes a thread; behind the rotary part only where something is to be copied
  p.units = rotary_dim / (2 * mult);
  if (!in_place(p.q) || (K && !in_place(p.k))) p.units += ((D - rotary_dim) / mult + 1) / 2;
  p.fp32 = dtype == BW_F32;
  p.half = interleaved ? 0 : 1;
  p.inverse = inverse ? 1 : 0;
  p.table = cos_sin_cache;
  p.table_len = cache_seq_len;
  p.positions = positions;
  p.pos_offset = pos_offset;
  bw::DeviceInfo dev;
  rc = bw::device_info(stream, &dev);
  if (rc != BW_OK) return rc;
  return bw::launch_rope(p, dev.num_sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? BW_OK : BW_ERR_CUDA;
}

int bw_kv_cache_write(const void* K, const void* V, const int64_t* k_strides, const int64_t* v_strides, int T, int Hkv,
                      int D, void* K_cache, void* V_cache, uint8_t* scales, int cache_dtype, int page_size,
                      int num_pages, const int64_t* slots, const float* cos_sin_cache, int64_t cache_seq_len,
                      int rotary_dim, const int* positions, int interleaved, void* stream) {
  if (T == 0) return BW_OK;   // no token
  if (!K || !V || !K_cache || !V_cache || !slots) return BW_ERR_NULL;
  if (!cache_dtype_ok(cache_dtype) || T < 0 || Hkv <= 0 || (D != 64 && D != 128) || num_pages <= 0 ||
      !page_size_ok(page_size))
    return BW_ERR_SHAPE;
  const int64_t num_slots = (int64_t)num_pages * page_size;
  if (num_slots >= (int64_t(1) << 31) || (int64_t)T * Hkv >= (int64_t(1) << 31)) return BW_ERR_SHAPE;
  if (cache_dtype == BW_E4M3 && !scales) return BW_ERR_NULL;
  if (cos_sin_cache) {
    if (!positions) return BW_ERR_NULL;
    if (cache_seq_len < 0 || rotary_dim < 16 || rotary_dim % 16 || rotary_dim > D) return BW_ERR_SHAPE;
  }
  if (!aligned(K, 16) || !aligned(V, 16) || !aligned(K_cache, 16) || !aligned(V_cache, 16) || !aligned(slots, 8) ||
      !aligned(cos_sin_cache, 16) || !aligned(positions, 4))
    return BW_ERR_ALIGN;
  bw::KvWriteParams p{};
  const int64_t dense[2] = {(int64_t)Hkv * D, D};
  const int64_t *ks = k_strides ? k_strides : dense, *vs = v_strides ? v_strides : dense;
  const int n[2] = {T, Hkv};
  for (int i = 0; i < 2; ++i)
    if (n[i] > 1 && (ks[i] <= 0 || vs[i] <= 0 || ks[i] % 8 || vs[i] % 8)) return BW_ERR_ALIGN;
  p.k = K;
  p.v = V;
  p.k_st = T == 1 ? 0 : ks[0];
  p.v_st = T == 1 ? 0 : vs[0];
  p.k_sh = Hkv == 1 ? 0 : ks[1];
  p.v_sh = Hkv == 1 ? 0 : vs[1];
  p.k_cache = K_cache;
  p.v_cache = V_cache;
  p.scales = scales;
  p.slots = slots;
  p.num_slots = num_slots;
  p.T = T;
  p.Hkv = Hkv;
  p.D = D;
  p.page_size = page_size;
  p.fp8 = cache_dtype == BW_E4M3;
  p.table = cos_sin_cache;
  p.table_len = cache_seq_len;
  p.R = rotary_dim;
  p.half = interleaved ? 0 : 1;
  p.positions = positions;
  bw::DeviceInfo dev;
  const int rc = bw::device_info(stream, &dev);
  if (rc != BW_OK) return rc;
  p.err = dev.err;
  return bw::launch_kv_write(p, static_cast<cudaStream_t>(stream)) == cudaSuccess ? BW_OK : BW_ERR_CUDA;
}

int bw_kv_cache_read(const void* K_cache, const void* V_cache, const uint8_t* scales, int cache_dtype, int page_size,
                     int num_pages, const int* block_table, int max_pages_per_seq, const int* kv_lens,
                     const int* kv_starts, const int64_t* out_offsets, int B, int Hkv, int D, void* K_out, void* V_out,
                     int64_t total_rows, void* stream) {
  if (B == 0 || total_rows == 0) return BW_OK;   // no row to write
  if (!K_cache || !V_cache || !block_table || !kv_lens || !out_offsets || !K_out || !V_out) return BW_ERR_NULL;
  if (!cache_dtype_ok(cache_dtype) || B < 0 || B > 4096 || Hkv <= 0 || (D != 64 && D != 128) || num_pages <= 0 ||
      max_pages_per_seq <= 0 || !page_size_ok(page_size) || total_rows < 0)
    return BW_ERR_SHAPE;
  if ((int64_t)num_pages * page_size >= (int64_t(1) << 31) ||
      (int64_t)max_pages_per_seq * page_size > (int64_t(1) << 30))
    return BW_ERR_SHAPE;
  if (Hkv > 65536) return BW_ERR_SHAPE;
  if (cache_dtype == BW_E4M3 && !scales) return BW_ERR_NULL;
  if (!aligned(K_cache, 16) || !aligned(V_cache, 16) || !aligned(K_out, 16) || !aligned(V_out, 16) ||
      !aligned(block_table, 4) || !aligned(kv_lens, 4) || !aligned(kv_starts, 4) || !aligned(out_offsets, 8))
    return BW_ERR_ALIGN;
  bw::KvReadParams p{};
  p.k_cache = K_cache;
  p.v_cache = V_cache;
  p.scales = scales;
  p.block_table = block_table;
  p.kv_lens = kv_lens;
  p.kv_starts = kv_starts;
  p.out_offsets = out_offsets;
  p.k_out = K_out;
  p.v_out = V_out;
  p.total_rows = total_rows;
  p.B = B;
  p.Hkv = Hkv;
  p.D = D;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.max_pages = max_pages_per_seq;
  p.fp8 = cache_dtype == BW_E4M3;
  bw::DeviceInfo dev;
  const int rc = bw::device_info(stream, &dev);
  if (rc != BW_OK) return rc;
  p.err = dev.err;
  return bw::launch_kv_read(p, dev.num_sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? BW_OK : BW_ERR_CUDA;
}

size_t bw_gqa_decode_paged_fp8_workspace_size(int B, int Hq, int Hkv, int D) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || D <= 0) return 0;
  const size_t groups = (size_t)decode_groups(Hkv, kMaxDecodeBlocks);
  const size_t parts = (groups + B) * Hkv, G = (size_t)(Hq / Hkv);
  return align256((size_t)(B + 1) * 4) + align256(parts * G * 4) + parts * G * D * 4;
}

int bw_gqa_decode_paged_fp8(const void* Q, const void* K_cache, const void* V_cache, const uint8_t* scales,
                            const int* block_table, const int* kv_lens, void* O, float* LSE, int B, int Hq, int Hkv,
                            int D, int page_size, int num_pages, int max_pages_per_seq, float scale, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (!Q || !K_cache || !V_cache || !scales || !block_table || !kv_lens || !O || !workspace) return BW_ERR_NULL;
  if (B <= 0 || B > 4096 || Hkv <= 0 || Hkv > kMaxDecodeBlocks || Hq <= 0 || Hq % Hkv != 0) return BW_ERR_SHAPE;
  const int G = Hq / Hkv;
  if (G > 16 || (D != 64 && D != 128) || num_pages <= 0 || max_pages_per_seq <= 0 || !page_size_ok(page_size))
    return BW_ERR_SHAPE;
  const int64_t max_tokens = (int64_t)max_pages_per_seq * page_size;
  if ((int64_t)num_pages * page_size >= (int64_t(1) << 31) || max_tokens > (int64_t(1) << 30) ||
      max_tokens * B > (int64_t(1) << 36))
    return BW_ERR_SHAPE;
  if (!(scale > 0.f) || !std::isfinite(scale)) return BW_ERR_SHAPE;
  if (!aligned(Q, 16) || !aligned(K_cache, 16) || !aligned(V_cache, 16) || !aligned(scales, 16) || !aligned(O, 16) ||
      !aligned(workspace, 16) || !aligned(block_table, 4) || !aligned(kv_lens, 4) || !aligned(LSE, 4))
    return BW_ERR_ALIGN;
  if (workspace_bytes < bw_gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D)) return BW_ERR_WORKSPACE;
  bw::Fp8DecodeParams p{};
  bw::DeviceInfo dev;
  const int rc = bw::device_info(stream, &dev);
  if (rc != BW_OK) return rc;
  p.err = dev.err;
  p.timeout_ns = dev.timeout_ns;
  p.debug_flags = dev.debug_flags;
  p.Q = Q;
  p.k_cache = K_cache;
  p.v_cache = V_cache;
  p.scales = scales;
  p.block_table = block_table;
  p.kv_lens = kv_lens;
  p.O = O;
  p.LSE = LSE;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = G;
  p.D = D;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.max_pages = max_pages_per_seq;
  p.max_tokens = (int)max_tokens;
  p.page_shift = -1;
  for (int i = 3; i < 31; ++i)
    if (page_size == 1 << i) p.page_shift = i;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int blocks = bw::decode_fp8_blocks(dev.num_sms);
  p.groups = decode_groups(Hkv, blocks < kMaxDecodeBlocks ? blocks : kMaxDecodeBlocks);
  bw::Fp8DecodeMaps maps;
  const int64_t rows = (int64_t)num_pages * page_size;
  const int box_rows = page_size < 64 ? page_size : 64;
  if (bw::make_map_bytes(&maps.k, K_cache, (int64_t)Hkv * D, rows, D, box_rows) != BW_OK ||
      bw::make_map_bytes(&maps.v, V_cache, (int64_t)Hkv * D, rows, D, box_rows) != BW_OK)
    return BW_ERR_CUDA;
  const size_t parts = (size_t)(p.groups + B) * Hkv;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.prefix = reinterpret_cast<int*>(ws);
  p.lse_part = reinterpret_cast<float*>(ws + align256((size_t)(B + 1) * 4));
  p.o_part = reinterpret_cast<float*>(ws + align256((size_t)(B + 1) * 4) + align256(parts * G * 4));
  return bw::launch_decode_fp8(p, maps, static_cast<cudaStream_t>(stream)) == cudaSuccess ? BW_OK : BW_ERR_CUDA;
}

}  // extern "C"
