// Rotary positions beside the attention kernels: the cos | sin table for a
// (possibly scaled) frequency schedule, and the rotation of Q and K with a
// position of its own for every token.
//
// Table row p of a rotary dimension R (the layout bw_qk_norm_rope reads):
//   t[p][i] = m cos(p f_i),  t[p][R/2 + i] = m sin(p f_i),  i < R/2.
// Rotation of the first R of a head's D elements, pairs (i, i + R/2) or
// (2i, 2i + 1):
//   a' = a c - b s,  b' = a s + b c;   inverse: s -> -s, the transpose, which
// is also the gradient with respect to (a, b) (m included).
// Elements R.. of the head and tokens whose position is outside the table pass
// through unchanged, as in bw_qk_norm_rope.
#include <cuda_bf16.h>

#include "early_launch.cuh"
#include "kernels.h"
#include "rope_math.cuh"

namespace bw {
namespace {

// One thread owns one pair (its frequency stays in a register) and walks rows.
// The angle is kept in quarter turns and in fp64 until only the part around the
// nearest whole number of them is left: p f has an absolute error near p f 2^-52,
// so positions of millions keep full fp32 accuracy; the rest, at most half a
// quarter turn, goes to fp32.  Adding 1.5 * 2^52 rounds to a whole number whose
// low bits are the quadrant, which saves the conversions between fp64 and
// integers.  The series and the product with the magnitude are fp32, as the table
// is (3.5e-8 of the result off at 131072 rows with YaRN, an fp64 series rounded
// once 2.7e-8): fp64 would be the bound instead of the stores.
constexpr int kTableThreads = 256, kTableBlocks = 6;   // resident blocks an SM, by registers

__global__ void __launch_bounds__(kTableThreads, kTableBlocks) rope_table_kernel(const RopeTableParams p) {
  constexpr double kRound = 6755399441055744.0;   // 1.5 * 2^52
  const int i = threadIdx.x;
  const int half = p.R >> 1;
  const double f = 4.0 * p.turns[i];
  after_previous_kernel();
  const int64_t r0 = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  if (r0 >= p.length) return;
  double pos = (double)(p.first + r0);
  const double pos_step = (double)step;
  float* out = p.table + r0 * p.R + i;
  const int64_t out_step = step * p.R;
  for (int64_t n = (p.length - r0 - 1) / step + 1; n > 0; --n, pos += pos_step, out += out_step) {
    const double quarters = f * pos;
    const double whole = quarters + kRound;
    const float x = (float)((quarters - (whole - kRound)) * 1.5707963267948966);   // |x| <= pi / 4
    const float x2 = x * x;
    // Taylor series; the terms left out are below 2^-28 of sin x and 2^-32 of cos x at pi / 4
    const float s = fmaf(x * x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), x);
    const float c = fmaf(
        x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    // turned by q quarters: (c, s), (-s, c), (-c, -s), (s, -c)
    const uint32_t q = (uint32_t)__double2loint(whole);
    const float cc = (q & 1) ? s : c, ss = (q & 1) ? c : s;
    out[0] = __uint_as_float(__float_as_uint(cc * p.magnitude) ^ (((q + 1) & 2) << 30));
    out[half] = __uint_as_float(__float_as_uint(ss * p.magnitude) ^ ((q & 2) << 30));
  }
}

// 16 bytes of a head: V elements.
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ void get(const uint4& v, float* x) { bf16x8_to_f32(v, x); }
  static __device__ __forceinline__ uint4 set(const float* x) { return f32_to_bf16x8(x); }
};
template <>
struct Vec<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ void get(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 set(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

constexpr int kRopeThreads = 128, kRopeBlocks = 8;   // resident blocks an SM, at four heads a thread

// A thread owns one unit of a token: two vectors of 16 bytes, R / 2 elements
// apart, that rotate with each other (half layout) or each within itself, or two
// vectors behind the rotary part; neighbouring threads read neighbouring
// vectors.  It reads its cos and sin once and applies them to kHeads heads, whose
// loads are all in flight together.
template <typename T, bool HALF, int kHeads>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  constexpr int V = Vec<T>::V;
  after_previous_kernel();
  const uint32_t in_block = p.by_units.div(threadIdx.x);   // token of the block
  const int64_t tok = (int64_t)blockIdx.x * p.block_tokens + in_block;
  if (in_block >= (uint32_t)p.block_tokens || tok >= (int64_t)p.B * p.S) return;
  const int unit = (int)(threadIdx.x - in_block * p.units);
  const int b = (int)p.by_s.div((uint32_t)tok), s = (int)tok - b * p.S;
  const bool is_k = (int)blockIdx.y >= p.q_groups;
  const RopeTensor& t = is_k ? p.k : p.q;
  const int h0 = ((int)blockIdx.y - (is_k ? p.q_groups : 0)) * kHeads;
  const T* in = static_cast<const T*>(t.in) + b * t.in_sb + s * t.in_ss + h0 * t.in_sh;
  T* out = static_cast<T*>(t.out) + b * t.out_sb + s * t.out_ss + h0 * t.out_sh;

  const int rot = p.R / (2 * V);   // rotary units
  const bool turns = unit < rot;
  const int rest = (p.D - p.R) / V;   // vectors behind the rotary part
  const int e0 = turns ? V * unit : p.R + V * (unit - rot);
  const int e1 = turns ? e0 + (p.R >> 1) : e0 + V * ((rest + 1) / 2);
  const bool two = e1 < p.D;
  uint4 x[kHeads][2];
#pragma unroll
  for (int u = 0; u < kHeads; ++u)
    if (h0 + u < t.H) {
      x[u][0] = *reinterpret_cast<const uint4*>(in + u * t.in_sh + e0);
      if (two) x[u][1] = *reinterpret_cast<const uint4*>(in + u * t.in_sh + e1);
    }
  if (turns) {
    const int64_t pos = (int64_t)(p.positions ? p.positions[tok] : s) + p.pos_offset;
    if (pos >= 0 && pos < p.table_len) {
      float c[V], sn[V];
      const float* cs = p.table + pos * p.R;
      load_angles<V, HALF>(cs, e0, e1, c);
      load_angles<V, HALF>(cs + (p.R >> 1), e0, e1, sn);
      if (p.inverse) {
#pragma unroll
        for (int i = 0; i < V; ++i) sn[i] = -sn[i];
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u)
        if (h0 + u < t.H) {
          float y[2 * V];
          Vec<T>::get(x[u][0], y);
          Vec<T>::get(x[u][1], y + V);
          rotate<V, HALF>(y, c, sn);
          x[u][0] = Vec<T>::set(y);
          x[u][1] = Vec<T>::set(y + V);
        }
    }
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u)
    if (h0 + u < t.H) {
      *reinterpret_cast<uint4*>(out + u * t.out_sh + e0) = x[u][0];
      if (two) *reinterpret_cast<uint4*>(out + u * t.out_sh + e1) = x[u][1];
    }
}

template <typename T, int kHeads>
cudaError_t launch(RopeParams p, unsigned token_blocks, cudaStream_t stream) {
  p.q_groups = (p.q.H + kHeads - 1) / kHeads;
  const int k_groups = (p.k.H + kHeads - 1) / kHeads;
  return launch_early(p.half ? rope_kernel<T, true, kHeads> : rope_kernel<T, false, kHeads>,
                      dim3(token_blocks, (unsigned)(p.q_groups + k_groups)), dim3(kRopeThreads), 0, stream, p);
}

// Four heads a thread re-use its angles and keep eight loads in flight; where that
// leaves less than a wave of blocks, two heads spread the work (2960 x 3 tokens, 6 + 2
// heads of 80: 4.8 -> 4.5 us, 7 + 1 heads 4.8 -> 5.1; 1777 x 3 tokens, 12 + 4 heads of
// 64 in fp32, more than a wave: 8.7 us with four heads, 9.4 with two; 4 x 4096 tokens,
// 40 heads: 55.3, 57.8).
template <typename T>
cudaError_t launch_heads(RopeParams p, int num_sms, cudaStream_t stream) {
  p.block_tokens = kRopeThreads / p.units;   // units: at most 64
  p.by_units = FastDiv(p.units);
  p.by_s = FastDiv(p.S);
  const int64_t tokens = (int64_t)p.B * p.S;
  const int64_t bx = (tokens + p.block_tokens - 1) / p.block_tokens;
  const int64_t blocks = bx * ((p.q.H + 3) / 4 + (p.k.H + 3) / 4);
  return blocks >= (int64_t)num_sms * kRopeBlocks ? launch<T, 4>(p, (unsigned)bx, stream)
                                                  : launch<T, 2>(p, (unsigned)bx, stream);
}

}  // namespace

cudaError_t launch_rope_table(const RopeTableParams& p, int num_sms, cudaStream_t stream) {
  const int half = p.R / 2;
  const dim3 block((unsigned)half, (unsigned)(kTableThreads / half));   // half: at most 256
  int64_t blocks = (p.length + block.y - 1) / block.y;
  const int64_t cap = (int64_t)num_sms * kTableBlocks;
  if (blocks > cap) blocks = cap;
  return launch_early(rope_table_kernel, dim3((unsigned)blocks), block, 0, stream, p);
}

cudaError_t launch_rope(const RopeParams& p, int num_sms, cudaStream_t stream) {
  return p.fp32 ? launch_heads<float>(p, num_sms, stream) : launch_heads<__nv_bfloat16>(p, num_sms, stream);
}

}  // namespace bw
