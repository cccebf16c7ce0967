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

#include "kernels.h"
#include "rope_math.cuh"

namespace bw {
namespace {

// One thread owns one pair (its frequency stays in a register) and walks rows.
// The angle is kept in turns and in fp64 until only the quarter turn around it
// is left: p f / 2 pi has an absolute error near p f 2^-53, so positions of
// millions keep full fp32 accuracy; |rest| <= 1/2 quarter turn goes to fp32.
__global__ void rope_table_kernel(const RopeTableParams p) {
  const int i = threadIdx.x;
  const int half = p.R >> 1;
  const double f = p.turns[i];
  for (int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y; r < p.length; r += (int64_t)gridDim.x * blockDim.y) {
    const double quarters = 4.0 * (f * (double)(p.first + r));
    const double whole = rint(quarters);
    const float rest = (float)(quarters - whole);
    float s, c;
    sincospif(0.5f * rest, &s, &c);
    const int q = (int)((long long)whole & 3);
    float cc = (q & 1) ? s : c, ss = (q & 1) ? c : s;   // turn by q quarters
    if (q == 1 || q == 2) cc = -cc;
    if (q >= 2) ss = -ss;
    float* row = p.table + r * p.R;
    row[i] = cc * p.magnitude;
    row[half + i] = ss * p.magnitude;
  }
}

template <typename T>
struct Chunk8;   // eight consecutive elements
template <>
struct Chunk8<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = v; }
  __device__ __forceinline__ void get(float* x) const { bf16x8_to_f32(v, x); }
  __device__ __forceinline__ void set(const float* x) { v = f32_to_bf16x8(x); }
};
template <>
struct Chunk8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + 4) = b;
  }
  __device__ __forceinline__ void get(float* x) const {
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ __forceinline__ void set(const float* x) {
    a = make_float4(x[0], x[1], x[2], x[3]);
    b = make_float4(x[4], x[5], x[6], x[7]);
  }
};

// A thread owns one unit of a token: 16 elements that rotate among themselves
// (two chunks of 8: c0 = 8u and c0 + R/2, or 16u and 16u + 8), or two chunks
// behind the rotary part.  It reads its 8 cos and 8 sin once and applies them
// to kHeads heads, whose loads are all in flight together.
template <typename T, bool HALF, int kHeads>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t tok = idx / p.units;
  if (tok >= (int64_t)p.B * p.S) return;
  const int unit = (int)(idx - tok * p.units);
  const int b = (int)(tok / p.S), s = (int)(tok - (int64_t)b * p.S);
  const bool is_k = (int)blockIdx.y >= p.q_groups;
  const RopeTensor& t = is_k ? p.k : p.q;
  const int h0 = ((int)blockIdx.y - (is_k ? p.q_groups : 0)) * kHeads;
  const T* in = static_cast<const T*>(t.in) + b * t.in_sb + s * t.in_ss + h0 * t.in_sh;
  T* out = static_cast<T*>(t.out) + b * t.out_sb + s * t.out_ss + h0 * t.out_sh;

  const int rot = p.R >> 4;   // rotary units
  const bool turns = unit < rot;
  const int e0 = turns ? (HALF ? 8 * unit : 16 * unit) : p.R + 16 * (unit - rot);
  const int e1 = turns ? (HALF ? 8 * unit + (p.R >> 1) : 16 * unit + 8) : e0 + 8;
  const bool two = e1 < p.D;   // D - R may be an odd number of chunks
  Chunk8<T> x[kHeads][2];
#pragma unroll
  for (int u = 0; u < kHeads; ++u)
    if (h0 + u < t.H) {
      x[u][0].load(in + u * t.in_sh + e0);
      if (two) x[u][1].load(in + u * t.in_sh + e1);
    }
  if (turns) {
    const int64_t pos = (int64_t)(p.positions ? p.positions[tok] : s) + p.pos_offset;
    if (pos >= 0 && pos < p.table_len) {
      float c[8], sn[8];
      const float* cs = p.table + pos * p.R + 8 * unit;
      load8(cs, c);
      load8(cs + (p.R >> 1), sn);
      if (p.inverse) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u)
        if (h0 + u < t.H) {
          float y[16];
          x[u][0].get(y);
          x[u][1].get(y + 8);
          rotate16<HALF>(y, c, sn);
          x[u][0].set(y);
          x[u][1].set(y + 8);
        }
    }
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u)
    if (h0 + u < t.H) {
      x[u][0].store(out + u * t.out_sh + e0);
      if (two) x[u][1].store(out + u * t.out_sh + e1);
    }
}

template <typename T, int kHeads>
cudaError_t launch(RopeParams p, cudaStream_t stream) {
  p.q_groups = (p.q.H + kHeads - 1) / kHeads;
  const int k_groups = (p.k.H + kHeads - 1) / kHeads;
  const int64_t threads = (int64_t)p.B * p.S * p.units;
  // Few tokens: small blocks, so that the work spreads over the SMs.
  const int block = threads <= 148 * 64 ? 64 : 256;
  const dim3 grid((unsigned)((threads + block - 1) / block), (unsigned)(p.q_groups + k_groups));
  if (p.half) rope_kernel<T, true, kHeads><<<grid, block, 0, stream>>>(p);
  else rope_kernel<T, false, kHeads><<<grid, block, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope_table(const RopeTableParams& p, int num_sms, cudaStream_t stream) {
  const int half = p.R / 2;
  const dim3 block((unsigned)half, (unsigned)(half >= 256 ? 1 : 256 / half));
  int64_t blocks = (p.length + block.y - 1) / block.y;
  const int64_t cap = (int64_t)num_sms * 8;
  if (blocks > cap) blocks = cap;
  rope_table_kernel<<<(unsigned)blocks, block, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_rope(const RopeParams& p, cudaStream_t stream) {
  return p.fp32 ? launch<float, 2>(p, stream) : launch<__nv_bfloat16, 4>(p, stream);
}

}  // namespace bw
