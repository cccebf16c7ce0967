// Single-token GQA decode over a paged 8-bit cache (e4m3 codes and a
// power-of-two scale per row, rope_math.cuh), split over the tokens and joined.
//
//   x_t = scale (q . k_t) 2^ek_t,  p_t = e^(x_t - max x),
//   o = sum_t p_t 2^ev_t v_t / sum_t p_t,  LSE = max x + ln sum_t p_t
// with k_t, v_t the codes of token t.
//
// Split: the 64-token tiles of all sequences, one after the other, are dealt
// to `groups` token groups in equal contiguous runs, so the load is even
// whatever the lengths are; a group has one block per KV head (the heads of a
// token are neighbours in memory and are read at the same time).  A run meets
// a sequence in one segment.  A segment that holds the whole sequence writes
// the result itself; the others leave (O, LSE) partials that the join kernel
// merges in segment order, so results do not depend on timing.
#include <cuda_bf16.h>

#include "kernels.h"
#include "ptx.cuh"
#include "rope_math.cuh"

namespace bw {
namespace {

constexpr int kTile = 64;      // tokens
constexpr int kMinTiles = 4;   // tiles of a run, at least
constexpr int kThreads = 128;

// Tokens of sequence b: kv_lens[b], at least 0 and at most what its row of the
// block table can hold.
__device__ __forceinline__ int seq_len(const Fp8DecodeParams& p, int b) {
  const int len = p.kv_lens[b];
  return len < 0 ? 0 : min(len, p.max_tokens);
}

// prefix[b] = tiles before sequence b (prefix[B] = all), by the whole block.
__device__ void tile_prefix(const Fp8DecodeParams& p, int* prefix, int* warp_sum) {
  const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.B + nth - 1) / nth;
  const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += (seq_len(p, b) + kTile - 1) / kTile;
  int x = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  if (lane == 31) warp_sum[warp] = x;
  __syncthreads();
  int before = x - mine;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  for (int b = b0; b < b1; ++b) {
    prefix[b] = before;
    before += (seq_len(p, b) + kTile - 1) / kTile;
  }
  if (tid == nth - 1) prefix[p.B] = before;
  __syncthreads();
}

__device__ __forceinline__ int tiles_per_group(int total, int groups) {
  return max((total + groups - 1) / groups, kMinTiles);
}

template <int D>
__global__ void __launch_bounds__(kThreads) decode_fp8_kernel(const Fp8DecodeParams p) {
  extern __shared__ int prefix[];
  __shared__ int warp_sum[kThreads / 32];
  __shared__ float qs[16][D], sc[16][kTile], vscale[kTile], m_s[16], l_s[16], corr_s[16];
  tile_prefix(p, prefix, warp_sum);
  const int tid = threadIdx.x;
  const int grp = blockIdx.x / p.Hkv, kvh = blockIdx.x - grp * p.Hkv;
  const int total = prefix[p.B], per = tiles_per_group(total, p.groups);
  if (blockIdx.x == 0)
    for (int b = tid; b <= p.B; b += kThreads) p.prefix[b] = prefix[b];
  int t0 = min(grp * per, total);
  const int t1 = min(t0 + per, total);
  while (t0 < t1) {
    int lo = 0, hi = p.B - 1;   // the last sequence that begins at or before t0 (and so holds it)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= t0) lo = mid; else hi = mid - 1;
    }
    const int b = lo, end = min(t1, prefix[b + 1]);
    const int len = seq_len(p, b);
    const int tok0 = (t0 - prefix[b]) * kTile, tok1 = min((end - prefix[b]) * kTile, len);
    for (int i = tid; i < p.G * D; i += kThreads)
      qs[i / D][i % D] = __bfloat162float(static_cast<const __nv_bfloat16*>(p.Q)[((int64_t)b * p.Hq + kvh * p.G) * D + i]);
    if (tid < 16) {
      m_s[tid] = -INFINITY;
      l_s[tid] = 0.f;
    }
    float acc[16 * D / kThreads] = {};
    __syncthreads();
    for (int t = tok0; t < tok1; t += kTile) {
      const int nt = min(kTile, tok1 - t);
      for (int i = tid; i < p.G * kTile; i += kThreads) {
        const int g = i / kTile, j = i % kTile;
        float s = -INFINITY;
        if (j < nt) {
          const int at = t + j, pi = at / p.page_size, place = at - pi * p.page_size;
          int page = p.block_table[(int64_t)b * p.max_pages + pi];
          if (page < 0 || page >= p.num_pages) {
            atomicCAS(p.err, 0, kErrIndexBit);
            page = 0;
          }
          const uint8_t* k = static_cast<const uint8_t*>(p.k_cache) + (((int64_t)page * p.page_size + place) * p.Hkv + kvh) * D;
          const uint8_t* bytes = p.scales + (((int64_t)page * p.Hkv + kvh) * 2) * p.page_size + place;
          float dot = 0.f;
          for (int d = 0; d < D; d += 2) {
            const float2 kk = e4m3x2_to_f32(*reinterpret_cast<const uint16_t*>(k + d));
            dot = fmaf(qs[g][d], kk.x, fmaf(qs[g][d + 1], kk.y, dot));
          }
          s = dot * __uint_as_float((uint32_t)bytes[0] << 23) * p.scale_log2;
          if (g == 0) vscale[j] = __uint_as_float((uint32_t)bytes[p.page_size] << 23);
        }
        sc[g][j] = s;
      }
      __syncthreads();
      if (tid < p.G) {
        float m = m_s[tid];
        for (int j = 0; j < nt; ++j) m = fmaxf(m, sc[tid][j]);
        const float sub = m == -INFINITY ? 0.f : m;
        corr_s[tid] = exp2f(m_s[tid] - sub);
        float l = l_s[tid] * corr_s[tid];
        for (int j = 0; j < nt; ++j) {
          sc[tid][j] = exp2f(sc[tid][j] - sub);
          l += sc[tid][j];
        }
        m_s[tid] = m;
        l_s[tid] = l;
      }
      __syncthreads();
      for (int j = 0; j < nt; ++j) {
        const int at = t + j, pi = at / p.page_size, place = at - pi * p.page_size;
        int page = p.block_table[(int64_t)b * p.max_pages + pi];
        if (page < 0 || page >= p.num_pages) page = 0;
        const uint8_t* v = static_cast<const uint8_t*>(p.v_cache) + (((int64_t)page * p.page_size + place) * p.Hkv + kvh) * D;
#pragma unroll
        for (int u = 0; u < 16 * D / kThreads; ++u) {
          const int i = tid + u * kThreads, g = i / D, d = i % D;
          if (g < p.G) {
            if (j == 0) acc[u] *= corr_s[g];
            acc[u] = fmaf(sc[g][j] * vscale[j], e4m3x2_to_f32(v[d]).x, acc[u]);
          }
        }
      }
      __syncthreads();
    }
    const bool whole = tok0 == 0 && tok1 == len;
    const int64_t part = (int64_t)(grp + b) * p.Hkv + kvh;
#pragma unroll
    for (int u = 0; u < 16 * D / kThreads; ++u) {
      const int i = tid + u * kThreads, g = i / D, d = i % D;
      if (g >= p.G) continue;
      const float o = acc[u] / l_s[g];
      const int64_t row = (int64_t)b * p.Hq + kvh * p.G + g;
      if (whole) static_cast<__nv_bfloat16*>(p.O)[row * D + d] = __float2bfloat16(o);
      else p.o_part[(part * p.G + g) * D + d] = o;
      if (d == 0) {
        const float lse = (m_s[g] + log2f(l_s[g])) * 0.69314718055994531f;
        if (!whole) p.lse_part[part * p.G + g] = lse;
        else if (p.LSE) p.LSE[row] = lse;
      }
    }
    __syncthreads();
    t0 = end;
  }
}

// One block per (sequence, query head): the segments of the sequence are the
// groups whose runs meet its tiles.
template <int D>
__global__ void __launch_bounds__(128) decode_fp8_join_kernel(const Fp8DecodeParams p) {
  constexpr int kLanes = D / 4;              // 4 columns a thread
  constexpr int kRows = 128 / kLanes;        // segments in flight
  __shared__ float4 part[kRows][kLanes];
  __shared__ float wsum_s[kRows], max_s[4];
  const int hq = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int kvh = hq / p.G, g = hq - kvh * p.G;
  const int first = p.prefix[b], last = p.prefix[b + 1], per = tiles_per_group(p.prefix[p.B], p.groups);
  const int64_t row = (int64_t)b * p.Hq + hq;
  __nv_bfloat16* O = static_cast<__nv_bfloat16*>(p.O) + row * D;
  if (first == last) {                       // no tokens
    for (int d = tid; d < D; d += 128) O[d] = __float2bfloat16(0.f);
    if (p.LSE && tid == 0) p.LSE[row] = -INFINITY;
    return;
  }
  const int g0 = first / per, n = (last - 1) / per - g0 + 1;
  if (n == 1) return;                        // written by its segment
  const int64_t base = ((int64_t)(g0 + b) * p.Hkv + kvh) * p.G + g, step = (int64_t)p.Hkv * p.G;
  float mx = -INFINITY;
  for (int i = tid; i < n; i += 128) mx = fmaxf(mx, p.lse_part[base + i * step]);
#pragma unroll
  for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  if ((tid & 31) == 0) max_s[tid >> 5] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(max_s[0], max_s[1]), fmaxf(max_s[2], max_s[3]));
  const float sub = mx == -INFINITY ? 0.f : mx;
  const int lane = tid % kLanes, r = tid / kLanes;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float wsum = 0.f;
  for (int i = r; i < n; i += kRows) {
    const float w = __expf(p.lse_part[base + i * step] - sub);
    const float4 v = *reinterpret_cast<const float4*>(p.o_part + (base + i * step) * D + 4 * lane);
    wsum += w;
    acc.x = fmaf(w, v.x, acc.x);
    acc.y = fmaf(w, v.y, acc.y);
    acc.z = fmaf(w, v.z, acc.z);
    acc.w = fmaf(w, v.w, acc.w);
  }
  part[r][lane] = acc;
  if (lane == 0) wsum_s[r] = wsum;
  __syncthreads();
  if (r == 0) {
    for (int i = 1; i < kRows; ++i) {
      const float4 v = part[i][lane];
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      wsum += wsum_s[i];
    }
    const float inv = 1.f / wsum;
    *reinterpret_cast<uint2*>(O + 4 * lane) =
        make_uint2(f32_to_bf16x2(acc.x * inv, acc.y * inv), f32_to_bf16x2(acc.z * inv, acc.w * inv));
    if (p.LSE && lane == 0) p.LSE[row] = sub + __logf(wsum);
  }
}

template <int D>
cudaError_t launch(const Fp8DecodeParams& p, cudaStream_t stream) {
  const int bytes = (p.B + 1) * 4;
  decode_fp8_kernel<D><<<p.groups * p.Hkv, kThreads, bytes, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  decode_fp8_join_kernel<D><<<dim3(p.Hq, p.B), 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_decode_fp8(const Fp8DecodeParams& p, cudaStream_t stream) {
  return p.D == 128 ? launch<128>(p, stream) : launch<64>(p, stream);
}

}  // namespace bw
