// The paged key-value cache: new tokens' K and V written into their slots (K
// rotated on the way, both quantised to 8 bits where the cache is 8-bit), and
// spans of sequences read back as contiguous bf16 rows.
//
// Cache: [pages, page_size, Hkv, D] bf16 or e4m3; 8-bit rows have a scale byte
// in scales [pages, Hkv, 2 (K, V), page_size] (rope_math.cuh: rows, rounding).
// Slot = page * page_size + place in the page.
#include <cuda_bf16.h>

#include <type_traits>

#include "early_launch.cuh"
#include "kernels.h"
#include "rope_math.cuh"

namespace bw {
namespace {

constexpr int kThreads = 256;

// Rows (token, KV head, K or V) one after the other, D / 16 lanes a row, 16
// elements a lane: two chunks of 8 in the rotary part, R / 2 apart, or 16
// consecutive elements.
template <int D, bool FP8, bool ROPE, bool HALF>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvWriteParams p) {
  constexpr int LPR = D / 16;
  after_previous_kernel();
  const int64_t idx = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t rows = (int64_t)p.T * p.Hkv * 2;
  int64_t row = idx / LPR;
  const int sub = threadIdx.x % LPR;
  bool live = row < rows;
  if (!live) row = 0;   // stays for the warp's shuffles
  const uint32_t th = (uint32_t)(row >> 1);   // T * Hkv is below 2^31
  const int is_v = (int)(row & 1);
  const int64_t t = p.by_heads.div(th);
  const int h = (int)(th - (uint32_t)t * p.Hkv);
  const int64_t slot = p.slots[t];
  if (slot < 0) {
    live = false;   // padding
  } else if (slot >= p.num_slots) {
    if (live && sub == 0) atomicCAS(p.err, 0, kErrIndexBit);
    live = false;
  }
  int e0 = 16 * sub, e1 = e0 + 8;
  bool turns = false;
  if constexpr (ROPE) {
    turns = !is_v && sub < (p.R >> 4);
    if (turns) {
      e0 = 8 * sub;
      e1 = e0 + (p.R >> 1);
    }
  }
  const __nv_bfloat16* in = static_cast<const __nv_bfloat16*>(is_v ? p.v : p.k) +
                            (is_v ? t * p.v_st + h * p.v_sh : t * p.k_st + h * p.k_sh);
  uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  if (live) {
    raw[0] = *reinterpret_cast<const uint4*>(in + e0);
    raw[1] = *reinterpret_cast<const uint4*>(in + e1);
  }
  float x[16];
  bf16x8_to_f32(raw[0], x);
  bf16x8_to_f32(raw[1], x + 8);
  if constexpr (ROPE) {
    if (turns && live) {
      const int64_t pos = p.positions[t];
      if (pos >= 0 && pos < p.table_len) {
        float c[8], sn[8];
        const float* cs = p.table + pos * p.R;
        load_angles<8, HALF>(cs, e0, e1, c);
        load_angles<8, HALF>(cs + (p.R >> 1), e0, e1, sn);
        rotate<8, HALF>(x, c, sn);
        raw[0] = f32_to_bf16x8(x);
        raw[1] = f32_to_bf16x8(x + 8);
      }
    }
  }
  const int64_t at = (slot * p.Hkv + h) * D;
  if constexpr (!FP8) {
    if (live) {
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(is_v ? p.v_cache : p.k_cache) + at;
      *reinterpret_cast<uint4*>(out + e0) = raw[0];
      *reinterpret_cast<uint4*>(out + e1) = raw[1];
    }
  } else {
    // The row's largest finite magnitude; infinities and NaN are stored as NaN
    // and leave the scale of the row's other elements alone.
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float a = fabsf(x[i]);
      amax = a < INFINITY ? fmaxf(amax, a) : amax;
    }
#pragma unroll
    for (int off = LPR / 2; off; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
    const int e = row_exponent(amax);
    const float inv = pow2i(-e);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = fabsf(x[i]) < INFINITY ? x[i] * inv : __uint_as_float(0x7fffffffu);
    if (live) {
      uint8_t* out = static_cast<uint8_t*>(is_v ? p.v_cache : p.k_cache) + at;
      const uint2 lo = make_uint2(f32_to_e4m3x4(x[0], x[1], x[2], x[3]), f32_to_e4m3x4(x[4], x[5], x[6], x[7]));
      const uint2 hi = make_uint2(f32_to_e4m3x4(x[8], x[9], x[10], x[11]), f32_to_e4m3x4(x[12], x[13], x[14], x[15]));
      *reinterpret_cast<uint2*>(out + e0) = lo;
      *reinterpret_cast<uint2*>(out + e1) = hi;
      if (sub == 0) {
        const uint32_t page = p.by_page.div((uint32_t)slot), place = (uint32_t)slot - page * p.page_size;
        p.scales[(((int64_t)page * p.Hkv + h) * 2 + is_v) * p.page_size + place] = (uint8_t)(e + 127);
      }
    }
  }
}

// blockIdx.y = sequence; a block takes block_tokens tokens at a time.  Its threads
// walk the (token, 8-element unit) pairs of them, kUnroll pairs of K and V loads
// in flight a thread; neighbouring threads write neighbouring 16 bytes, so every
// store covers whole sectors.
constexpr int kUnroll = 4;

template <int D, bool FP8>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvReadParams p) {
  constexpr int LPR = D / 8;
  using Raw = typename std::conditional<FP8, uint2, uint4>::type;   // 8 elements
  const int b = blockIdx.y;
  after_previous_kernel();
  const int len = p.kv_lens[b];
  if (len <= 0) return;
  const int64_t start = p.kv_starts ? p.kv_starts[b] : 0;
  const int64_t out0 = p.out_offsets[b];
  // (out0 + len might pass 2^63)
  if (start < 0 || start + len > (int64_t)p.max_pages * p.page_size || out0 < 0 || out0 > p.total_rows - len) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(p.err, 0, kErrIndexBit);
    return;
  }
  const uint32_t upr = (uint32_t)p.Hkv * LPR;   // units a token
  const int* bt = p.block_table + (int64_t)b * p.max_pages;
  for (int tok0 = blockIdx.x * p.block_tokens; tok0 < len; tok0 += gridDim.x * p.block_tokens) {
    const uint32_t n = (uint32_t)min(p.block_tokens, len - tok0) * upr;
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += kThreads * kUnroll) {
      Raw raw[kUnroll][2];
      uint8_t sc[kUnroll][2];
      int64_t dst[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const uint32_t i = i0 + u * kThreads;
        dst[u] = -1;
        if (i >= n) continue;
        const uint32_t tok = p.by_units.div(i), unit = i - tok * upr;
        const uint32_t at = (uint32_t)start + tok0 + tok;
        const uint32_t pi = p.by_page.div(at), place = at - pi * p.page_size;
        const int page = bt[pi];
        if ((unsigned)page >= (unsigned)p.num_pages) {
          atomicCAS(p.err, 0, kErrIndexBit);
          continue;
        }
        const int64_t src = ((int64_t)page * p.page_size + place) * p.Hkv * D + 8 * unit;
        dst[u] = (out0 + tok0 + tok) * p.Hkv * D + 8 * unit;
        const int64_t esz = FP8 ? 1 : 2;
        raw[u][0] = *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(p.k_cache) + src * esz);
        raw[u][1] = *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(p.v_cache) + src * esz);
        if constexpr (FP8) {
          const uint8_t* s = p.scales + ((int64_t)page * p.Hkv + unit / LPR) * 2 * p.page_size + place;
          sc[u][0] = s[0];
          sc[u][1] = s[p.page_size];
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (dst[u] < 0) continue;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint4 o;
          if constexpr (FP8) {
            const float scale = __uint_as_float((uint32_t)sc[u][w] << 23);
            float f[8];
            e4m3x4_to_f32(raw[u][w].x, f);
            e4m3x4_to_f32(raw[u][w].y, f + 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= scale;
            o = f32_to_bf16x8(f);
          } else {
            o = raw[u][w];
          }
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(w ? p.v_out : p.k_out) + dst[u]) = o;
        }
      }
    }
  }
}

template <int D, bool FP8>
cudaError_t write_launch(KvWriteParams p, cudaStream_t stream) {
  p.by_heads = FastDiv(p.Hkv);
  p.by_page = FastDiv(p.page_size);
  const int64_t threads = (int64_t)p.T * p.Hkv * 2 * (D / 16);
  const dim3 blocks((unsigned)((threads + kThreads - 1) / kThreads));
  auto kern = p.table == nullptr ? kv_write_kernel<D, FP8, false, false>
              : p.half           ? kv_write_kernel<D, FP8, true, true>
                                 : kv_write_kernel<D, FP8, true, false>;
  return launch_early(kern, blocks, dim3(kThreads), 0, stream, p);
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteParams& p, cudaStream_t stream) {
  if (p.D == 128) return p.fp8 ? write_launch<128, true>(p, stream) : write_launch<128, false>(p, stream);
  return p.fp8 ? write_launch<64, true>(p, stream) : write_launch<64, false>(p, stream);
}

cudaError_t launch_kv_read(KvReadParams p, int num_sms, cudaStream_t stream) {
  const int upr = p.Hkv * (p.D / 8);
  p.by_units = FastDiv(upr);
  p.by_page = FastDiv(p.page_size);
  // Blocks for the longest span that the table's width or the output's rows
  // allow, at most about 16 an SM over all sequences.
  int64_t most = (int64_t)p.max_pages * p.page_size;
  if (most > p.total_rows) most = p.total_rows;
  // Of a block's tokens: four units a thread, fewer where the rows would not make
  // two blocks an SM (3 sequences of 305 to 1094 tokens, 16 heads of 64, bf16, with
  // their write: 7.3 -> 6.2 us against 16 tokens for every shape; 32768 tokens: 41.8
  // -> 41.6).
  const int64_t spread = p.total_rows / ((int64_t)num_sms * 2), full = kThreads * kUnroll / upr;
  p.block_tokens = (int)(spread < full ? spread : full);
  if (p.block_tokens < 1) p.block_tokens = 1;
  int64_t bx = (most + p.block_tokens - 1) / p.block_tokens;
  const int64_t cap = ((int64_t)num_sms * 16 + p.B - 1) / p.B;
  if (bx > cap) bx = cap;
  auto kern = p.D == 128 ? (p.fp8 ? kv_read_kernel<128, true> : kv_read_kernel<128, false>)
                         : (p.fp8 ? kv_read_kernel<64, true> : kv_read_kernel<64, false>);
  return launch_early(kern, dim3((unsigned)bx, (unsigned)p.B), dim3(kThreads), 0, stream, p);
}

}  // namespace bw
