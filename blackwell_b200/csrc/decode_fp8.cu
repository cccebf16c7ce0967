// Single-token GQA decode over a paged 8-bit cache (e4m3 codes and a
// power-of-two scale per row, rope_math.cuh), split over the tokens and joined.
//
//   x_t = scale (q . k_t) 2^ek_t,  p_t = e^(x_t - max x),
//   o = sum_t p_t 2^ev_t v_t / sum_t p_t,  LSE = max x + ln sum_t p_t
// with k_t, v_t the codes of token t.
//
// Split: the tiles of all sequences, one after the other, are dealt to `groups`
// token groups in equal contiguous runs, so the load is even whatever the
// lengths are; a group has one block per KV head (the heads of a token are
// neighbours in memory and are read at the same time).  A run meets a sequence
// in one segment.  A segment that holds the whole sequence writes the result
// itself; the others leave (O, LSE) partials that the join kernel merges in
// segment order, so results do not depend on timing.  Runs are of whole tiles:
// finer ones balance better but cut short sequences in two, and a segment costs
// about 2 us (16 ragged sequences, heads of 64: 11 us against 12.5 with runs of
// 64 tokens).
//
// 2 G flops a byte: bound by HBM.  The products take 13 to 18 % of the tensor
// pipe through mma.sync; a tcgen05 product would want the f16 operands in shared
// memory, where the codes are not, and 128 rows.  What had to be kept small
// beside them is the work per code: the conversions (two codes an instruction,
// no repacking) and the softmax, and the copies a page needs.
//
// Measured on B200 (device time; share of the 6.45 TB/s that a copy reaches):
//   64 sequences of 1024 to 32768 tokens, 8 KV heads, G = 8, D = 128
//     pages of 64   329 - 356 us   97 - 105 %   (by box; the bf16 cache has twice the bytes)
//     pages of 16   335 us         103 %
//     pages of 8    390 us          88 %         one tensor copy per 8 rows
//     D = 64        179 us          97 %
//   32 sequences of 1000 to 32768, 4 KV heads, G = 16: 104 us, 83 %: two products
//     and softmaxes a code on the same 8 consumer warps an SM.  They issue in 50 % of
//     the cycles (G = 8: 42 %) and wait for memory a quarter as long (0.5 against 2.0
//     warps an issue): what bounds them is the latency of their own instructions, and
//     168 registers leave no room to start the next tile under it
//   1 sequence of 131072: 50 us, 84 %: start, last merge and join take 7
//   1 sequence of 517: 7.5 us: launch 0.4, tile counts 1, page index and first tile
//     2.1, products 0.8, merge 0.9, join 2
#include <cuda_bf16.h>

#include <atomic>
#include <type_traits>

#include "early_launch.cuh"
#include "kernels.h"
#include "ptx.cuh"
#include "rope_math.cuh"

namespace bw {
namespace {

constexpr int kStep = 64;   // tokens of a step: 16 a consumer warp
// Steps of a tile, which a warp takes at once (so many independent chains of
// products in flight).  Heads of 64 have half the bytes a token and so twice the
// softmax per byte; more steps hide its latency.
__host__ __device__ constexpr int tile_steps(int D) { return D == 128 ? 2 : 4; }
__host__ __device__ constexpr int tile_tokens(int D) { return kStep * tile_steps(D); }
constexpr int kMaxB = 4096;
constexpr int kWarps = 4;      // consumers; one producer warp more for K and one for V
constexpr int kThreads = 32 * (kWarps + 2);
// Resident blocks an SM: 97 KB of stages and up to 168 registers a thread each.
// Three blocks of smaller tiles were slower (337 -> 349 us at the first shape
// above), four too (355).
constexpr int kBlocksPerSm = 2;

// Tokens of sequence b: kv_lens[b], at least 0 and at most what its row of the
// block table can hold.
__device__ __forceinline__ int seq_len(const Fp8DecodeParams& p, int b) {
  const int len = p.kv_lens[b];
  return len < 0 ? 0 : min(len, p.max_tokens);
}

// prefix[b] = tiles before sequence b (prefix[B] = all), by the whole block.  Every
// length is read once, so that the counts fit together whatever happens to
// kv_lens meanwhile.
template <int kTile>
__device__ void tile_prefix(const Fp8DecodeParams& p, int* prefix, int* warp_sum) {
  const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.B + nth - 1) / nth;
  const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int tiles = (seq_len(p, b) + kTile - 1) / kTile;
    prefix[b] = tiles;
    mine += tiles;
  }
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
    const int tiles = prefix[b];
    prefix[b] = before;
    before += tiles;
  }
  if (tid == nth - 1) prefix[p.B] = before;
  __syncthreads();
}

__device__ __forceinline__ int tiles_per_group(int total, int groups) { return max((total + groups - 1) / groups, 1); }

// ------------------------------------------------------------------ shared memory of a block
// A stage is one tile: K and V codes (pieces of bh = min(64, page size) rows, D
// bytes a row, 16-byte chunks swizzled by the tensor map) and the scale bytes of
// K, then of V.
template <int D>
struct Cfg {
  static constexpr int kTile = tile_tokens(D);
  static constexpr int kHalf = kTile * D;            // K (or V) codes of a stage
  static constexpr int kStage = 2 * kHalf;           // 32 KB
  static constexpr int kStages = 3;
  static constexpr int kScales = kStages * kStage;
  static constexpr int kRed = kScales + kStages * 2 * kTile;    // m, l, M of 4 warps x 16 heads
  static constexpr int kBars = kRed + 3 * kWarps * 16 * 4;
  static constexpr int kPrefix = kBars + 256;
};
template <int D>
struct Bars {
  uint64_t full[Cfg<D>::kStages], empty[Cfg<D>::kStages];
  int abort_flag;
  int stop;   // what the consumers make of abort_flag at the end of a segment
  int warp_sum[kThreads / 32];
};
static_assert(sizeof(Bars<64>) <= 256 && sizeof(Bars<128>) <= 256, "barriers fit their 256 bytes");

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }
// Asynchronous copy of N = 4 or 8 bytes.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
// The thread arrives on `bar` when its copies so far have landed.
__device__ __forceinline__ void arrive_after_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

struct Segment {
  int b, len, tok0, tok1;   // tokens [tok0, tok1) of sequence b
};
// The first tile from t on with which a sequence begins (or the end of all).
__device__ __forceinline__ int sequence_start(const int* prefix, int B, int t) {
  int lo = 0, hi = B;   // the first b with prefix[b] >= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] < t) lo = mid + 1; else hi = mid;
  }
  return prefix[lo];
}
// The segment that begins at tile t0 of the run [t0, t1); t0 moves behind it.
template <int kTile>
__device__ __forceinline__ Segment next_segment(const Fp8DecodeParams& p, const int* prefix, int& t0, int t1) {
  int lo = 0, hi = p.B - 1;   // the last sequence that begins at or before t0, and so holds it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= t0) lo = mid; else hi = mid - 1;
  }
  Segment s;
  s.b = lo;
  // The last tile decides the length; the tiles are the prefix's: a length that the
  // caller has changed since (an error) must not lead to a segment without tokens,
  // nor the warps of a block to different tiles.
  const int tiles = prefix[lo + 1] - prefix[lo];
  s.len = min(max(seq_len(p, lo), (tiles - 1) * kTile + 1), tiles * kTile);
  const int end = min(t1, prefix[lo + 1]);
  s.tok0 = (t0 - prefix[lo]) * kTile;
  s.tok1 = min((end - prefix[lo]) * kTile, s.len);
  t0 = end;
  return s;
}

// Two producer warps stream the tiles of the block's run through a ring of
// stages; four consumer warps take 16 tokens of every step each, keep their own
// running softmax and output, and merge at the end of a segment.
//
// The products run with tokens (then columns d) as the 16 rows of m16n8k16 and
// the heads of the group as its 8 columns, so a group of up to 8 fills the
// instruction (NT = 1; NT = 2 for up to 16):
//   S^T[16 tokens, 8 heads] = K[16, D] Q^T,   O^T[D, 8] += V^T[D, 16] P^T[16, 8].
// Codes go to f16 in registers (every e4m3 value is one): four bytes that
// ldmatrix hands a lane are d = 4 q4 .. 4 q4 + 3 of its token, taken as the
// k-columns 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9 of a step of 16 (Q in the same
// order); of V they are columns 2g, 2g + 1 of two tokens, taken as the rows g
// and g + 8 of a step of 16.
//
// Scales: x = (q k) 2^ek qs with the group's softmax scale and a power of two of
// the Q row in qs (Q is brought to [1, 2) for f16).  2^ev must not be multiplied
// into an f16 weight; the weight is 2^(x + ev - M) with M the running maximum of
// x + ev, so the largest contribution is in [1, 2^8] whatever the scales are.
// The denominator has its own reference m (the maximum of x): one more ex2 an
// element.  Both references follow their maximum only when it has moved by more
// than 2^8; m is per thread, M per warp (votes; shuffles only when it moves).
// A value row of zeros has no part in M (see there).
//
// Rounded to fewer bits than 32: Q to f16 (nothing down to 2^-14 of its row's
// largest) and the weight to f16 (2^-11 of itself; the bf16 decode's are bf16,
// 2^-8), since the product wants both as the codes are.  Sums, the denominator and
// the references are fp32.  Against 64 bits the output is as far off as one from
// fp32 weights (1.6e-3 of its norm, the rounding to bf16); the two differ by single
// bf16 steps (1.4e-4 to 6.5e-4 of the norm).
//
// WHOLE: runs begin and end with a sequence, so that none is cut and no join follows.
template <int D, int NT, bool WHOLE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    decode_fp8_kernel(const Fp8DecodeParams p, const __grid_constant__ Fp8DecodeMaps maps) {
  using C = Cfg<D>;
  constexpr int U = tile_steps(D), kTile = C::kTile;
  constexpr int kScaleBytes = kTile / 32;   // of K (or V), a producer lane
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars<D>& bars = *reinterpret_cast<Bars<D>*>(smem + C::kBars);
  int* prefix = reinterpret_cast<int*>(smem + C::kPrefix);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&bars.full[s], 2 * (1 + 32));   // of either producer: the codes' byte count, each lane's scale bytes
      mbar_init(&bars.empty[s], kWarps);
    }
    bars.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp >= kWarps && lane == 0) prefetch_tmap(warp == kWarps ? &maps.k : &maps.v);
  after_previous_kernel();
  let_next_kernel_start();
  tile_prefix<kTile>(p, prefix, bars.warp_sum);   // synchronises the block
  const int grp = blockIdx.x / p.Hkv, kvh = blockIdx.x - grp * p.Hkv;
  const int total = prefix[p.B], per = tiles_per_group(total, p.groups);
  if (blockIdx.x == 0)
    for (int b = tid; b <= p.B; b += kThreads) p.prefix[b] = prefix[b];
  int t0 = min(grp * per, total), t1 = min(t0 + per, total);
  if constexpr (WHOLE) {
    t0 = sequence_start(prefix, p.B, t0);
    t1 = sequence_start(prefix, p.B, t1);
  }
  const WaitCtl wc{&bars.abort_flag, p.err, p.timeout_ns, 48 + warp};
  const uint32_t sbase = smem_u32(smem);
  const int bh = p.page_size < 64 ? p.page_size : 64;   // rows of a piece

  if (warp >= kWarps) {
    // ------------------------------------------------------------ producers
    // One warp copies K, one V: a tensor copy a piece, one lane each (the
    // hardware takes them from a warp one after the other, which is why there
    // are two warps), and the scale bytes of 2 U tokens by every lane.
    const int is_v = warp - kWarps;
    const CUtensorMap* map = is_v ? &maps.v : &maps.k;
    const int np = kTile / bh;
    const auto page_of = [&](int tok) { return p.page_shift >= 0 ? tok >> p.page_shift : tok / p.page_size; };
    uint32_t n = 0;
    bool ok = true;
    while (ok && t0 < t1) {
      const Segment sg = next_segment<kTile>(p, prefix, t0, t1);
      const int* bt = p.block_table + (int64_t)sg.b * p.max_pages;
      const int last_page = page_of(sg.tok1 - 1);
      // Page indices: a lane holds one of 32 consecutive ones, and the next 32 are on their way.
      int base = page_of(sg.tok0);
      int held = bt[min(base + lane, last_page)], next = bt[min(base + 32 + lane, last_page)];
      for (int t = sg.tok0; t < sg.tok1; t += kTile, ++n) {
        const uint32_t s = n % C::kStages;
        if (page_of(t) >= base + 32) {
          base += 32;
          held = next;
          next = bt[min(base + 32 + lane, last_page)];
        }
        const auto page_at = [&](int pi) {   // a tile's pages may reach into the next 32
          const int a = __shfl_sync(0xffffffffu, held, pi - base), b = __shfl_sync(0xffffffffu, next, pi - base);
          int page = pi - base < 32 ? a : b;
          if ((unsigned)page >= (unsigned)p.num_pages) {
            atomicCAS(p.err, 0, kErrIndexBit);
            page = 0;
          }
          return page;
        };
        // Only what the segment has: a piece (a lane's scale bytes) that begins past its end stays what it was.
        const int live = min(np, (sg.tok1 - t + bh - 1) / bh);   // pieces
        const int tok = t + (lane < live ? lane : 0) * bh, pi = page_of(tok);
        const int row = page_at(pi) * p.page_size + (tok - pi * p.page_size);
        const bool has_sc = t + lane * kScaleBytes < sg.tok1;
        const int tok_sc = has_sc ? t + lane * kScaleBytes : t, pi_sc = page_of(tok_sc);
        const uint8_t* src = p.scales + (((int64_t)page_at(pi_sc) * p.Hkv + kvh) * 2 + is_v) * p.page_size +
                             (tok_sc - pi_sc * p.page_size);
        bool got = true;
        if (lane == 0) {
          got = wc.wait(&bars.empty[s], ((n / C::kStages) & 1) ^ 1);
          if (got) mbar_arrive_expect_tx(&bars.full[s], live * bh * D);
        }
        if (!__shfl_sync(0xffffffffu, got, 0)) {
          ok = false;
          break;
        }
        const bool withheld = (p.debug_flags & 1) && !is_v && n == 0;
        if (lane < live && !withheld)
          tma_load_2d(smem + s * C::kStage + is_v * C::kHalf + lane * bh * D, map, &bars.full[s], kvh * D, row);
        if (has_sc) copy_async<kScaleBytes>(sbase + C::kScales + (s * 2 + is_v) * kTile + lane * kScaleBytes, src);
        arrive_after_copies(&bars.full[s]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      // Copies in flight must land before the block gives its memory back, also when
      // this producer got all its stages and the consumers have given up on one (else
      // they wait for the same barriers, and this costs nothing).  A stage that the
      // other producer no longer filled stays open: the bound ends it.
      for (uint32_t i = n > C::kStages ? n - C::kStages : 0; i < n; ++i)
        drain_wait(&bars.full[i % C::kStages], (i / C::kStages) & 1, kDrainNs);
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int g = lane >> 2, q4 = lane & 3;
  float* red_m = reinterpret_cast<float*>(smem + C::kRed);   // [warp][16]
  float* red_l = red_m + kWarps * 16;
  float* red_M = red_l + kWarps * 16;
  // This lane's ldmatrix row: token (lane >> 3 & 1) * 8 + (lane & 7) of the warp's 16 of a step, chunk (lane >> 4) of a pair.
  // 16-byte chunk c of tile row r lies at chunk c ^ (r & 7) of its row (128-byte rows), c ^ (r >> 1 & 3) (64-byte rows).
  const int lrow = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
  const uint32_t row_off = (uint32_t)lrow * D;   // pieces follow one another: a row's place does not depend on bh
  const uint32_t swz = D == 128 ? (lrow & 7) : ((lrow >> 1) & 3);
  const uint32_t chunk0 = lane >> 4;
  if constexpr (WHOLE)   // the sequences without tokens are written here, not by the join
    for (int b = grp; b < p.B; b += p.groups) {
      if (prefix[b + 1] != prefix[b]) continue;
      const int64_t row = (int64_t)b * p.Hq + kvh * p.G;
      for (int i = tid; i < p.G * D / 8; i += kWarps * 32)
        reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.O) + row * D)[i] = make_uint4(0u, 0u, 0u, 0u);
      if (p.LSE && tid < p.G) p.LSE[row + tid] = -INFINITY;
    }
  uint32_t n = 0;
  while (t0 < t1) {
    const Segment sg = next_segment<kTile>(p, prefix, t0, t1);
    // Q of head 8 nt + g as f16, brought to [1, 2) by a power of two; columns in the codes' order
    uint32_t qb[NT][D / 16][2];
    float qs[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const __nv_bfloat16* Q = static_cast<const __nv_bfloat16*>(p.Q) + ((int64_t)sg.b * p.Hq + kvh * p.G + h) * D;
      uint2 raw[D / 16];
      uint32_t top = 0;   // largest magnitude's bits
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        raw[j] = h < p.G ? *reinterpret_cast<const uint2*>(Q + 16 * j + 4 * q4) : make_uint2(0u, 0u);
        top = max(top, max(max(raw[j].x & 0x7fffu, (raw[j].x >> 16) & 0x7fffu),
                           max(raw[j].y & 0x7fffu, (raw[j].y >> 16) & 0x7fffu)));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int ex = min(max((int)(top >> 7), 2), 252);   // biased exponent
      const float down = __uint_as_float((uint32_t)(254 - ex) << 23), up = __uint_as_float((uint32_t)ex << 23);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        qb[nt][j][0] = f16x2(__uint_as_float(raw[j].x << 16) * down, __uint_as_float(raw[j].x & 0xffff0000u) * down);
        qb[nt][j][1] = f16x2(__uint_as_float(raw[j].y << 16) * down, __uint_as_float(raw[j].y & 0xffff0000u) * down);
      }
      const float mine = p.scale_log2 * up;
      qs[nt][0] = __shfl_sync(0xffffffffu, mine, 8 * q4);       // of head 2 q4 (held by lanes 4 * head ..)
      qs[nt][1] = __shfl_sync(0xffffffffu, mine, 8 * q4 + 4);
    }
    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2], M[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) o[nt][c][0] = o[nt][c][1] = o[nt][c][2] = o[nt][c][3] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[nt][j] = M[nt][j] = -INFINITY;
        l[nt][j] = 0.f;
      }
    }
    // The warp's tokens of the steps u0 .. u0 + N of stage s.  MASK: of those, tokens
    // from `left` on do not exist (token 64 u + i for step u0 + u, i < 16).
    const auto take = [&](auto steps, auto mask, uint32_t s, int u0, int left) {
      constexpr int N = decltype(steps)::value;
      constexpr bool MASK = decltype(mask)::value;
      const uint32_t kb = sbase + s * C::kStage + row_off + u0 * (kStep * D), vb = kb + C::kHalf;
      // S^T of the steps; one step: in two chains of products
      constexpr int kChains = N == 1 ? 2 : 1;
      float acc[N][NT][kChains][4];
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < kChains; ++i)
            acc[u][nt][i][0] = acc[u][nt][i][1] = acc[u][nt][i][2] = acc[u][nt][i][3] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; j += 2)
#pragma unroll
        for (int u = 0; u < N; ++u) {
          uint32_t r[4];
          ldsm_x4(kb + u * (kStep * D) + (((j + chunk0) ^ swz) << 4), r);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16x4(r[2 * i], a0, a2);
            e4m3x4_to_f16x4(r[2 * i + 1], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(acc[u][nt][i % kChains], a0, a1, a2, a3, qb[nt][j + i][0], qb[nt][j + i][1]);
          }
        }
      const uint8_t* sc = smem + C::kScales + s * 2 * kTile + u0 * kStep + warp * 16 + g;
      float ks[N][2], ev[N][2];   // of tokens g and g + 8
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ks[u][i] = __uint_as_float((uint32_t)sc[kStep * u + 8 * i] << 23);
          ev[u][i] = (float)((int)sc[kTile + kStep * u + 8 * i] - 127);
        }
      // V's bytes (t0 2g, t0 2g+1, t1 2g, t1 2g+1) -> (t0, t1) of 2g and of 2g + 1.  A token past the end is picked as
      // zero, whatever its codes are (a weight of 0 would not silence a NaN).
      uint32_t sel[N][2];
#pragma unroll
      for (int u = 0; u < N; ++u) sel[u][0] = sel[u][1] = 0x3120u;
      const bool some = MASK && left < (N - 1) * kStep + 16;
      if (some) {
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int tl = kStep * u + 8 * i + 2 * q4;
            sel[u][i] = (tl < left ? 0x0100u : 0x0404u) | (tl + 1 < left ? 0x3020u : 0x4040u);
          }
      }
      uint32_t pb[N][NT][2];
      float y[NT][2][2 * N];   // [head 2 q4 + j][step u, token 8 i + g]
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[2][2 * N];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2 * N; ++e) {
            const int u = e / 2, i = e % 2;
            float a = acc[u][nt][0][2 * i + j];
            if constexpr (kChains == 2) a += acc[u][nt][1][2 * i + j];
            // Key and query scales may be far out and make up for each other: a small qs goes to ks first, a
            // large one last (a third product an element: up to 1 % of the time).
            x[j][e] = a * (ks[u][i] * fminf(qs[nt][j], 1.f)) * fmaxf(qs[nt][j], 1.f);
          }
        if (some) {
#pragma unroll
          for (int e = 0; e < 2 * N; ++e)
            if (kStep * (e / 2) + 8 * (e % 2) + g >= left) x[0][e] = x[1][e] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(x[j][0], x[j][1]), my;
#pragma unroll
          for (int e = 2; e < 2 * N; ++e) mx = fmaxf(mx, x[j][e]);
          const bool up = mx > m[nt][j] + 8.f;
          l[nt][j] *= ex2f(up ? m[nt][j] - mx : 0.f);
          m[nt][j] = up ? mx : m[nt][j];
          const float sub = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
#pragma unroll
          for (int e = 0; e < 2 * N; ++e) {
            l[nt][j] += ex2f(x[j][e] - sub);
            y[nt][j][e] = x[j][e] + ev[e / 2][e % 2];
            my = e ? fmaxf(my, y[nt][j][e]) : y[nt][j][e];
          }
          moved |= my > M[nt][j] + 8.f;
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
        // A row of zeros (scale byte 127) adds nothing and must not raise M: the
        // rows that carry the output would fall below f16.  Its y goes to -inf.
        // Where M does not move its weight is at most 2^8 and its codes say the rest.
        bool at_127 = false;
#pragma unroll
        for (int u = 0; u < N; ++u) at_127 |= ev[u][0] == 0.f || ev[u][1] == 0.f;
        if (__any_sync(0xffffffffu, at_127)) {
          uint32_t some_code = 0;   // bit 2 u + i: token 8 i + g of step u has a code other than 0 and NaN
          const uint8_t* vrow = smem + s * C::kStage + C::kHalf + (u0 * kStep + warp * 16 + g) * D + q4 * (D / 4);
#pragma unroll 1
          for (int e = 0; e < 2 * N; ++e) {
            uint32_t any = 0;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              const uint4 w = reinterpret_cast<const uint4*>(vrow + ((e >> 1) * kStep + (e & 1) * 8) * D)[c];
              // a byte's magnitude + 1 has a bit of 0x7e unless it was 0 or 0x7f
              any |= ((w.x & 0x7f7f7f7fu) + 0x01010101u) | ((w.y & 0x7f7f7f7fu) + 0x01010101u) |
                     ((w.z & 0x7f7f7f7fu) + 0x01010101u) | ((w.w & 0x7f7f7f7fu) + 0x01010101u);
            }
            some_code |= (any & 0x7e7e7e7eu) ? 1u << e : 0u;
          }
          some_code |= __shfl_xor_sync(0xffffffffu, some_code, 1);
          some_code |= __shfl_xor_sync(0xffffffffu, some_code, 2);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 2 * N; ++e)
                if (!(some_code >> e & 1)) y[nt][j][e] = -INFINITY;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = M[nt][j];
#pragma unroll
            for (int e = 0; e < 2 * N; ++e) mx = fmaxf(mx, y[nt][j][e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float corr = mx == -INFINITY ? 1.f : ex2f(M[nt][j] - mx);
            M[nt][j] = mx;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              o[nt][c][j] *= corr;
              o[nt][c][2 + j] *= corr;
            }
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float M0 = M[nt][0] == -INFINITY ? 0.f : M[nt][0], M1 = M[nt][1] == -INFINITY ? 0.f : M[nt][1];
#pragma unroll
        for (int e = 0; e < 2 * N; ++e)
          pb[e / 2][nt][e % 2] = transpose8x8(f16x2(ex2f(y[nt][0][e] - M0), ex2f(y[nt][1][e] - M1)));
      }
#pragma unroll
      for (int c = 0; c < D / 16; c += 2)
#pragma unroll
        for (int u = 0; u < N; ++u) {
          uint32_t r[4];
          ldsm_x4_t(vb + u * (kStep * D) + (((c + chunk0) ^ swz) << 4), r);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16x4(__byte_perm(r[2 * i], 0, sel[u][0]), a0, a1);
            e4m3x4_to_f16x4(__byte_perm(r[2 * i + 1], 0, sel[u][1]), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][c + i], a0, a1, a2, a3, pb[u][nt][0], pb[u][nt][1]);
          }
        }
    };
    uint32_t s = 0;
    for (int t = sg.tok0; t < sg.tok1; t += kTile, ++n) {
      s = n % C::kStages;
      // On a timeout the warp still goes through the merge below, so that the
      // barriers stay matched.
      const bool got = wc.wait(&bars.full[s], (n / C::kStages) & 1);
      if (!__all_sync(0xffffffffu, got)) break;   // the warp decides as one
      const int left = sg.tok1 - (t + warp * 16);
      if constexpr (U <= 2) {
        if (left > 0) take(std::integral_constant<int, U>{}, std::true_type{}, s, 0, left);
      } else {
        // Four steps at once where they are there, else one by one: short sequences
        // and rests (48 sequences of 50 to 107 tokens: 8.9 -> 8.3 us).
        if (t + kTile <= sg.tok1) take(std::integral_constant<int, U>{}, std::false_type{}, s, 0, kTile);
        else
          for (int u = 0; u < U && left > u * kStep; ++u)
            take(std::integral_constant<int, 1>{}, std::true_type{}, s, u, left - u * kStep);
      }
      // the last stage of a segment is kept for the merge
      if (t + kTile < sg.tok1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.empty[s]);
      }
    }

    // ---- merge the warps: references and sums of every head, and the outputs,
    // through shared memory; the outputs through the last stage, [warp][NT * 8
    // heads][D] floats, columns permuted by 8 (h / 2 mod 4) so that the four lanes
    // of a g do not meet in a bank.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mm = m[nt][j];
        mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 4));
        mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 8));
        mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, 16));
        float ll = l[nt][j] * (m[nt][j] == -INFINITY ? 1.f : ex2f(m[nt][j] - mm));
        ll += __shfl_xor_sync(0xffffffffu, ll, 4);
        ll += __shfl_xor_sync(0xffffffffu, ll, 8);
        ll += __shfl_xor_sync(0xffffffffu, ll, 16);
        m[nt][j] = mm;
        l[nt][j] = ll;
      }
    float* part_o = reinterpret_cast<float*>(smem + s * C::kStage);
    static_assert(kWarps * NT * 8 * D * 4 <= C::kStage, "the outputs fit a stage");
    consumer_sync();   // the stage's codes, and the previous segment's sums, have been read
    if (g == 0)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int h = warp * 16 + nt * 8 + 2 * q4 + j;
          red_m[h] = m[nt][j];
          red_l[h] = l[nt][j];
          red_M[h] = M[nt][j];
        }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float2*>(part_o + ((warp * NT + nt) * 8 + 2 * q4 + j) * D + ((16 * c + 2 * g) ^ (8 * q4))) =
              make_float2(o[nt][c][j], o[nt][c][2 + j]);
    if (tid == 0) bars.stop = *wc.abort_flag;
    consumer_sync();
    constexpr int kPer = kWarps * 32 / (NT * 8);   // threads a head
    const int h = tid / kPer;
    if (h < p.G) {
      const bool whole = sg.tok0 == 0 && sg.tok1 == sg.len;
      const int64_t part = ((int64_t)(grp + sg.b) * p.Hkv + kvh) * p.G + h;
      const int64_t row = (int64_t)sg.b * p.Hq + kvh * p.G + h;
      float mx = -INFINITY, Mx = -INFINITY, sum = 0.f, f[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mx = fmaxf(mx, red_m[w * 16 + h]);
        Mx = fmaxf(Mx, red_M[w * 16 + h]);
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = red_m[w * 16 + h], Mw = red_M[w * 16 + h];
        sum += red_l[w * 16 + h] * (mw == -INFINITY ? 1.f : ex2f(mw - mx));
        f[w] = Mw == -INFINITY ? 1.f : ex2f(Mw - Mx);
      }
      // o = a 2^Mx / (sum 2^mx); both powers may be far out, their quotient is the values' scale, and up to 2^8
      // more (2^128 at the largest values) since mx lags: a part of a large one comes after the division.
      const float back = Mx - mx > 64.f ? 65536.f : 1.f;
      const float to = (Mx == -INFINITY ? 1.f : ex2f(Mx - mx - (back == 1.f ? 0.f : 16.f))) / sum;
#pragma unroll
      for (int d = (tid % kPer) * 4; d < D; d += kPer * 4) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(part_o + (w * NT * 8 + h) * D + (d ^ (8 * ((h >> 1) & 3))));
          a.x = fmaf(f[w], v.x, a.x);
          a.y = fmaf(f[w], v.y, a.y);
          a.z = fmaf(f[w], v.z, a.z);
          a.w = fmaf(f[w], v.w, a.w);
        }
        a.x *= to; a.y *= to; a.z *= to; a.w *= to;
        a.x *= back; a.y *= back; a.z *= back; a.w *= back;
        if (whole)
          *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.O) + row * D + d) =
              make_uint2(f32_to_bf16x2(a.x, a.y), f32_to_bf16x2(a.z, a.w));
        else
          *reinterpret_cast<float4*>(p.o_part + part * D + d) = a;
      }
      if (tid % kPer == 0) {
        const float lse = (mx + __log2f(sum)) * 0.69314718055994531f;
        if (!whole) p.lse_part[part] = lse;
        else if (p.LSE) p.LSE[row] = lse;
      }
    }
    // After a wait that ran out all warps stop at the same segment, so that none
    // waits at a barrier for one that has left, and no stage is given back any more.
    if (*(volatile int*)&bars.stop) break;
    fence_proxy_async_smem();   // the stage goes back to the copies
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars.empty[s]);
  }
}

// The joins sum their segments times 2^-10: up to 2^10 of them (kMaxDecodeBlocks)
// whose values are near fp32's largest have a mean in range and a sum beyond it.
constexpr float kJoinDown = 1.f / 1024.f, kJoinUp = 1024.f;

// One block of T threads per (sequence, query head): the segments of the sequence
// are the groups whose runs meet its tiles; kUnroll times the segments that fit
// side by side are in flight.
template <int D, int T, int kUnroll>
__global__ void __launch_bounds__(T) decode_fp8_join_kernel(const Fp8DecodeParams p) {
  constexpr int kLanes = D / 4;              // 4 columns a thread
  constexpr int kRows = T / kLanes;          // segments side by side
  __shared__ float4 part[kRows][kLanes];
  __shared__ float wsum_s[kRows], max_s[T / 32];
  after_previous_kernel();   // the segments are written
  const int hq = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int kvh = hq / p.G, g = hq - kvh * p.G;
  const int first = p.prefix[b], last = p.prefix[b + 1], per = tiles_per_group(p.prefix[p.B], p.groups);
  const int64_t row = (int64_t)b * p.Hq + hq;
  __nv_bfloat16* O = static_cast<__nv_bfloat16*>(p.O) + row * D;
  if (first == last) {                       // no tokens
    for (int d = tid; d < D; d += T) O[d] = __float2bfloat16(0.f);
    if (p.LSE && tid == 0) p.LSE[row] = -INFINITY;
    return;
  }
  const int g0 = first / per, n = (last - 1) / per - g0 + 1;
  if (n == 1) return;                        // written by its segment
  const int64_t base = ((int64_t)(g0 + b) * p.Hkv + kvh) * p.G + g, step = (int64_t)p.Hkv * p.G;
  float mx = -INFINITY;
  for (int i = tid; i < n; i += T) mx = fmaxf(mx, p.lse_part[base + i * step]);
#pragma unroll
  for (int off = 16; off; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
  if ((tid & 31) == 0) max_s[tid >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / 32; ++w) mx = fmaxf(mx, max_s[w]);
  const float sub = mx == -INFINITY ? 0.f : mx;
  const int lane = tid % kLanes, r = tid / kLanes;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float wsum = 0.f;
  for (int i0 = r; i0 < n; i0 += kRows * kUnroll) {
    float w[kUnroll];
    float4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * kRows;
      w[u] = -INFINITY;
      if (i < n) {
        w[u] = p.lse_part[base + i * step];
        v[u] = *reinterpret_cast<const float4*>(p.o_part + (base + i * step) * D + 4 * lane);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (i0 + u * kRows < n) {
        const float e = __expf(w[u] - sub), ed = e * kJoinDown;
        wsum += e;
        acc.x = fmaf(ed, v[u].x, acc.x);
        acc.y = fmaf(ed, v[u].y, acc.y);
        acc.z = fmaf(ed, v[u].z, acc.z);
        acc.w = fmaf(ed, v[u].w, acc.w);
      }
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
    *reinterpret_cast<uint2*>(O + 4 * lane) = make_uint2(f32_to_bf16x2(acc.x * inv * kJoinUp, acc.y * inv * kJoinUp),
                                                         f32_to_bf16x2(acc.z * inv * kJoinUp, acc.w * inv * kJoinUp));
    if (p.LSE && lane == 0) p.LSE[row] = sub + __logf(wsum);
  }
}

// The same for few segments: a warp per (sequence, query head), no barriers.
template <int D>
__global__ void __launch_bounds__(128) decode_fp8_join_few_kernel(const Fp8DecodeParams p) {
  constexpr int kLanes = D / 4, kSide = 32 / kLanes;   // 4 columns a lane; segments side by side
  after_previous_kernel();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)p.B * p.Hq) return;
  const int b = (int)(row / p.Hq), hq = (int)(row - (int64_t)b * p.Hq);
  const int kvh = hq / p.G, g = hq - kvh * p.G;
  const int first = p.prefix[b], last = p.prefix[b + 1], per = tiles_per_group(p.prefix[p.B], p.groups);
  const int col = lane % kLanes, side = lane / kLanes;
  __nv_bfloat16* O = static_cast<__nv_bfloat16*>(p.O) + row * D + 4 * col;
  if (first == last) {                       // no tokens
    if (side == 0) *reinterpret_cast<uint2*>(O) = make_uint2(0u, 0u);
    if (p.LSE && lane == 0) p.LSE[row] = -INFINITY;
    return;
  }
  const int g0 = first / per, n = (last - 1) / per - g0 + 1;
  if (n == 1) return;                        // written by its segment
  const int64_t base = ((int64_t)(g0 + b) * p.Hkv + kvh) * p.G + g, step = (int64_t)p.Hkv * p.G;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float mx = -INFINITY, sum = 0.f;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const float lse = i0 + lane < n ? p.lse_part[base + (i0 + lane) * step] : -INFINITY;
    float m = lse;
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    m = fmaxf(m, mx);
    const float sub = m == -INFINITY ? 0.f : m;
    const float corr = __expf(mx - sub), w = __expf(lse - sub);
    mx = m;
    sum *= corr;
    acc.x *= corr; acc.y *= corr; acc.z *= corr; acc.w *= corr;
    const int cnt = min(32, n - i0);
    for (int j0 = 0; j0 < cnt; j0 += 2 * kSide) {
      float4 v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = j0 + u * kSide + side;
        if (j < cnt) v[u] = *reinterpret_cast<const float4*>(p.o_part + (base + (i0 + j) * step) * D + 4 * col);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = j0 + u * kSide + side;
        const float e = __shfl_sync(0xffffffffu, w, j & 31);
        if (j < cnt) {
          const float ed = e * kJoinDown;
          sum += e;
          acc.x = fmaf(ed, v[u].x, acc.x);
          acc.y = fmaf(ed, v[u].y, acc.y);
          acc.z = fmaf(ed, v[u].z, acc.z);
          acc.w = fmaf(ed, v[u].w, acc.w);
        }
      }
    }
  }
  if constexpr (kSide == 2) {
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
  }
  if (side == 0) {
    const float inv = 1.f / sum;
    *reinterpret_cast<uint2*>(O) = make_uint2(f32_to_bf16x2(acc.x * inv * kJoinUp, acc.y * inv * kJoinUp),
                                              f32_to_bf16x2(acc.z * inv * kJoinUp, acc.w * inv * kJoinUp));
    if (p.LSE && lane == 0) p.LSE[row] = (mx == -INFINITY ? 0.f : mx) + __logf(sum);
  }
}

template <int D, int NT, bool WHOLE>
cudaError_t launch_main(const Fp8DecodeParams& p, const Fp8DecodeMaps& maps, cudaStream_t stream) {
  auto kern = decode_fp8_kernel<D, NT, WHOLE>;
  // Once per device; the limit, not what a launch takes, so it covers every B.
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(allowed.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kPrefix + (kMaxB + 1) * 4 + 1024);
    if (e != cudaSuccess) return e;
    if (dev < 64) allowed |= uint64_t(1) << dev;
  }
  return launch_early(kern, dim3(p.groups * p.Hkv), dim3(kThreads), Cfg<D>::kPrefix + (p.B + 1) * 4 + 1024, stream, p, maps);
}

template <int D, int NT>
cudaError_t launch(const Fp8DecodeParams& p, const Fp8DecodeMaps& maps, cudaStream_t stream) {
  // Sequences of a few tiles are not cut: the join and its launch would cost more
  // than a block's further tiles.  The table's width decides, which is all that the
  // host knows of the lengths: a table of fixed width gets the cut and the join for
  // the same sequences.  Up to two tiles always (48 sequences of up to 107 tokens, 4
  // KV heads, D = 64: 6.1 us; with a table for 131072 tokens 7.0), up to four where
  // sequences and heads occupy the GPU (16 of up to 500 tokens, 8 KV heads: 9.9, 10.8;
  // 116 of up to 246: 18.8, 20.4; but 2 of up to 1000, 2 KV heads, D = 64: 8.9 not cut,
  // 8.0 cut).  With up to eight it is slower or the same (16 of up to 1000: 13.5 not
  // cut, 12.0 cut).
  const int tiles = (p.max_tokens + Cfg<D>::kTile - 1) / Cfg<D>::kTile;
  if (tiles <= 2 || (tiles <= 4 && 4 * p.B >= p.groups)) return launch_main<D, NT, true>(p, maps, stream);
  const cudaError_t e = launch_main<D, NT, false>(p, maps, stream);
  if (e != cudaSuccess) return e;
  // A sequence has about groups / B segments, and no more than tiles.  Many (few KV
  // heads, few long sequences): wide blocks with 4 loads in flight a thread (131072
  // tokens, one KV head, 256 segments: 18.9 us for both kernels against 26).  Few:
  // the small kernel starts sooner (one sequence of 517 tokens: 7.6 against 8.0 us;
  // 32 of 500 to 2000: 24.3 against 25.4).
  if (p.groups > 32 * p.B && p.max_tokens > 32 * Cfg<D>::kTile)
    return launch_early(decode_fp8_join_kernel<D, 512, 4>, dim3(p.Hq, p.B), dim3(512), 0, stream, p);
  // Many rows (then their segments are few): a warp each, which fits in one wave
  // (73 sequences x 208 heads: 114 -> 106 us; 32 x 32: 23.3 -> 23.6).
  if ((int64_t)p.B * p.Hq >= 2048)
    return launch_early(decode_fp8_join_few_kernel<D>, dim3((unsigned)(((int64_t)p.B * p.Hq + 3) / 4)), dim3(128), 0,
                        stream, p);
  return launch_early(decode_fp8_join_kernel<D, 128, 1>, dim3(p.Hq, p.B), dim3(128), 0, stream, p);
}

}  // namespace

int decode_fp8_blocks(int num_sms) { return num_sms * kBlocksPerSm; }

cudaError_t launch_decode_fp8(const Fp8DecodeParams& p, const Fp8DecodeMaps& maps, cudaStream_t stream) {
  if (p.D == 128) return p.G <= 8 ? launch<128, 1>(p, maps, stream) : launch<128, 2>(p, maps, stream);
  return p.G <= 8 ? launch<64, 1>(p, maps, stream) : launch<64, 2>(p, maps, stream);
}

}  // namespace bw
