// INT8 quantisation of rows, alone and fused into the MoE dispatch.
//
// Signed 8-bit codes with one scale per row (token or output channel):
//
//   scale[r] = max|x[r, :]| / 127        q[r, c] = round_half_even(127 x[r, c] / max|x[r, :]|)
//
// (a zero row: scale 1, codes 0; a row with an infinity or NaN: scale NaN, codes 0, so everything
// computed from the row is NaN). The code is defined by the quotient of 127 x and the maximum, not by
// x / scale: with significands of at most 11 bits 127 x is exact in fp32, and a quotient in
// [2^m, 2^(m+1)) that is not exactly half-way between two integers is at least 2^(m-20) away from
// it, sixteen times fp32's half step there, so the fp32 quotient always rounds to the integer the
// exact one rounds to. x / scale would inherit the rounding of the scale and miss the tie at
// x = max / 2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ggo.h"
#include "ggo_internal.h"

namespace ggo {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kRouteTokens = 32;  // tokens per block of the router's offset table
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 16;

// Largest |x| of eight 16-bit floats as its bit pattern (for the sign-free patterns of one format
// the order of the integers is the order of the values, NaN above infinity above all finite ones),
// kept per 16-bit half.
__device__ __forceinline__ uint32_t abs_max8(uint32_t m, const uint4& v) {
  m = __vmaxu2(m, v.x & 0x7fff7fffu);
  m = __vmaxu2(m, v.y & 0x7fff7fffu);
  m = __vmaxu2(m, v.z & 0x7fff7fffu);
  return __vmaxu2(m, v.w & 0x7fff7fffu);
}

template <typename T16>
__device__ __forceinline__ float from_bits(uint32_t b) {
  const unsigned short h = static_cast<unsigned short>(b);
  return static_cast<float>(*reinterpret_cast<const T16*>(&h));
}

// What a row needs to turn its values into codes: q = round(x * mul / top), mul a power of two times
// 127 that brings the quotient's operands near 1 (no overflow, no underflow of anything that
// could round to a code other than 0), inv = 1 / top.
struct RowCode {
  float mul, top, inv, scale;
};

template <typename T16>
__device__ __forceinline__ RowCode row_code(uint32_t max2) {
  const uint32_t bits = max(max2 & 0xffffu, max2 >> 16);
  const float amax = from_bits<T16>(bits);
  RowCode c;
  const int field = static_cast<int>(__float_as_uint(amax) >> 23);  // biased exponent of the maximum
  if (bits == 0 || field == 255) {
    c.mul = 0.f;  // codes 0 (the quotient below is then 0 or, for x = inf or NaN, masked)
    c.top = c.inv = 1.f;
    c.scale = bits == 0 ? 1.f : __int_as_float(0x7fc00000);
    return c;
  }
  // 2^(127 - exponent field), between 2^-126 and 2^119 so that it and 127 times it are normal
  // numbers: top lands in [2^-14, 4)
  const int f = 254 - field;
  const float two = __uint_as_float(static_cast<uint32_t>(f < 1 ? 1 : (f > 246 ? 246 : f)) << 23);
  c.top = amax * two;
  c.mul = 127.f * two;
  c.inv = __frcp_rn(c.top);
  c.scale = __fdiv_rn(amax, 127.f);
  return c;
}

// Code of x as the low byte of the result. t = 127 x and top are exact, and one correction of
// q0 = t * (1 / top) with the exact remainder r = t - top q0 gives the correctly rounded quotient
// (Markstein, IBM J. Res. Dev. 34(1), 1990). Adding 1.5 * 2^23 rounds it to an integer, half to even, whose
// two's complement is the sum's low bits.
__device__ __forceinline__ uint32_t code_of(float x, const RowCode& c) {
  const float t = x * c.mul;
  const float q0 = t * c.inv;
  const float q = fmaf(fmaf(-c.top, q0, t), c.inv, q0);
  return __float_as_uint(q + 12582912.f);
}

// Eight values to eight codes (64 bits).
template <typename T16>
__device__ __forceinline__ uint2 code8(const uint4& v, const RowCode& c) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t a = code_of(from_bits<T16>(w[2 * h] & 0xffffu), c);
    const uint32_t b = code_of(from_bits<T16>(w[2 * h] >> 16), c);
    const uint32_t d = code_of(from_bits<T16>(w[2 * h + 1] & 0xffffu), c);
    const uint32_t e = code_of(from_bits<T16>(w[2 * h + 1] >> 16), c);
    o[h] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(d, e, 0x0040), 0x5410);
  }
  return c.mul == 0.f ? make_uint2(0u, 0u) : make_uint2(o[0], o[1]);
}

__device__ __forceinline__ uint32_t warp_max2(uint32_t m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(kAll, m, o));
  return m;
}

// Short rows: LPR neighbouring lanes per row, each holding up to P 16-byte pieces, so that a warp's
// loads stay contiguous and no lane idles on rows of a few hundred bytes. 65536 x 64: 3.4 us;
// 65536 x 2048: 60 us, where a block of 256 threads per row took 195 us for 65536 x 2064.
template <typename T16, int LPR, int P>
__global__ void __launch_bounds__(256)
    quantize_int8_short_kernel(const T16* __restrict__ x, int rows, int cols,
                               uint8_t* __restrict__ q, float* __restrict__ scale) {
  const int64_t r = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / LPR;
  const int l = threadIdx.x % LPR;
  const int vec = cols / 8;
  const bool row_ok = r < rows;
  const uint4* xr = reinterpret_cast<const uint4*>(x + r * cols);
  uint4 v[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = l + i * LPR;
    v[i] = row_ok && c < vec ? xr[c] : make_uint4(0, 0, 0, 0);
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) m = abs_max8(m, v[i]);
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(kAll, m, o));
  const RowCode rc = row_code<T16>(m);
  if (!row_ok) return;
  if (l == 0) scale[r] = rc.scale;
  uint2* qr = reinterpret_cast<uint2*>(q + r * cols);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = l + i * LPR;
    if (c < vec) qr[c] = code8<T16>(v[i], rc);
  }
}

// One block of TB threads per row, the row held in registers, up to P 16-byte pieces a thread.
// 32768 x 14336: 212 us at 1965 MHz (6.6 TB/s, the rate of a plain copy); 241 us (5.9 TB/s) in a stream
// of calls that the power limit holds at 1640 MHz. The sizes matter: 65536 x 4096 took 224 us
// with 256 threads and eight pieces, six of them idle, and takes 121 us.
constexpr int kRegCols = 16384;

template <typename T16, int TB, int P>
__global__ void __launch_bounds__(TB)
    quantize_int8_block_kernel(const T16* __restrict__ x, int cols, uint8_t* __restrict__ q,
                               float* __restrict__ scale) {
  __shared__ uint32_t s_max[TB / 32];
  const size_t r = blockIdx.x;
  const int vec = cols / 8;
  const uint4* xr = reinterpret_cast<const uint4*>(x + r * cols);
  uint4 v[P];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = threadIdx.x + i * TB;
    v[i] = c < vec ? xr[c] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < P; ++i) m = abs_max8(m, v[i]);
  m = warp_max2(m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < TB / 32; ++w) m = __vmaxu2(m, s_max[w]);
  const RowCode rc = row_code<T16>(m);
  if (threadIdx.x == 0) scale[r] = rc.scale;
  uint2* qr = reinterpret_cast<uint2*>(q + r * cols);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = threadIdx.x + i * TB;
    if (c < vec) qr[c] = code8<T16>(v[i], rc);
  }
}

// Rows longer than the block form holds: two passes, the second one out of L2.
template <typename T16>
__global__ void __launch_bounds__(256)
    quantize_int8_long_kernel(const T16* __restrict__ x, int cols, uint8_t* __restrict__ q,
                              float* __restrict__ scale) {
  __shared__ uint32_t s_max[8];
  const size_t r = blockIdx.x;
  const int vec = cols / 8;
  const uint4* xr = reinterpret_cast<const uint4*>(x + r * cols);
  uint32_t m = 0;
#pragma unroll 4
  for (int c = threadIdx.x; c < vec; c += 256) m = abs_max8(m, xr[c]);
  m = warp_max2(m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = __vmaxu2(m, s_max[w]);
  const RowCode rc = row_code<T16>(m);
  if (threadIdx.x == 0) scale[r] = rc.scale;
  uint2* qr = reinterpret_cast<uint2*>(q + r * cols);
#pragma unroll 4
  for (int c = threadIdx.x; c < vec; c += 256) qr[c] = code8<T16>(xr[c], rc);
}

// The dispatch's permutation with the quantisation on the way: every token's row is read, coded
// once and written to its top_k expert-sorted places as codes. grid = (ceil(T / 32), 4 WPT): block
// (b, s) finds the sorted positions of 32-token block b (one warp walks its (token, slot) entries
// in order, as the bf16 dispatch does) and moves tokens s, s + 4 WPT, ... of it, WPT warps each. A lane
// takes pairs of neighbouring 16-byte pieces, which make one 16-byte piece of codes, and holds up to
// 2 P of them in registers; what lies beyond is read a second time, out of L1 or L2.
template <typename T16, int WPT, int P>
__global__ void __launch_bounds__(256)
    permute_int8_kernel(const T16* __restrict__ x, int T, int H, int E, int K,
                        const int32_t* __restrict__ topk_ids, const int* __restrict__ block_offsets,
                        uint8_t* __restrict__ q_sorted, float* __restrict__ scale_sorted,
                        int32_t* __restrict__ slot_pos) {
  extern __shared__ int psm[];
  __shared__ uint32_t s_max[8];
  int* off = psm;      // [E] running sorted position per expert
  int* lim = off + E;  // [E] first sorted position behind this block's rows of the expert
  int* pos = lim + E;  // [kRouteTokens * K] sorted position per entry, -1 for a dropped one
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.x * kRouteTokens;
  const int ntok = min(kRouteTokens, T - t0);
  const int nent = ntok * K;
  const int pairs = H / 16;
  constexpr int kStep = 32 * WPT;  // pairs between a thread's pieces of a row
  const int at = threadIdx.x % kStep;
  const int tl = static_cast<int>(threadIdx.x / kStep) * 4 * WPT + blockIdx.y;
  const bool some = tl < ntok;
  const uint4* src = reinterpret_cast<const uint4*>(x + static_cast<size_t>(t0 + tl) * H);
  uint4 v[2 * P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int c = at + i * kStep;
    const bool ok = some && c < pairs;
    v[2 * i] = ok ? src[2 * c] : make_uint4(0, 0, 0, 0);
    v[2 * i + 1] = ok ? src[2 * c + 1] : make_uint4(0, 0, 0, 0);
  }
  const int* first = block_offsets + static_cast<size_t>(blockIdx.x) * E;
  const bool last = blockIdx.x + 1 == gridDim.x;
  for (int e = threadIdx.x; e < E; e += 256) {
    // the next block's first place or, behind the table's last block, the next expert's
    const int begin = first[e], next = first[E + (last ? min(e + 1, E - 1) : e)];
    off[e] = begin;
    lim[e] = last && e + 1 == E ? T * K : min(max(next, 0), T * K);
  }
  __syncthreads();
  if (warp == 0) {
    const int32_t* ids = topk_ids + static_cast<size_t>(t0) * K;
    for (int base = 0; base < nent; base += 32) {
      const int i = base + lane;
      const bool valid = i < nent;
      const unsigned vmask = __ballot_sync(kAll, valid);
      if (valid) {
        // a choice that the table has no place for is dropped, as in the dispatch of ggo_moe.cu
        const int id = ids[i];
        const bool known = id >= 0 && id < E;
        const unsigned peers = __match_any_sync(vmask, id);
        const unsigned b = known ? off[id] : 0;  // unsigned: a table may hold anything
        __syncwarp(vmask);
        if (known && lane == __ffs(peers) - 1) off[id] = static_cast<int>(b + __popc(peers));
        int ps = static_cast<int>(b + __popc(peers & ((1u << lane) - 1u)));
        if (!known || ps < 0 || ps >= lim[id]) ps = -1;
        pos[i] = ps;
        if (blockIdx.y == 0) slot_pos[static_cast<size_t>(t0) * K + i] = ps;
      }
      __syncwarp();
    }
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 2 * P; ++i) m = abs_max8(m, v[i]);
  if (some)
    for (int c = at + P * kStep; c < pairs; c += kStep)
      m = abs_max8(abs_max8(m, src[2 * c]), src[2 * c + 1]);
  m = warp_max2(m);
  if (WPT > 1 && lane == 0) s_max[warp] = m;
  __syncthreads();
  if (!some) return;
  if (WPT > 1) {
    const int first = warp / WPT * WPT;
#pragma unroll
    for (int w = 0; w < WPT; ++w) m = __vmaxu2(m, s_max[first + w]);
  }
  const RowCode rc = row_code<T16>(m);
  if (at < K && pos[tl * K + at] >= 0) scale_sorted[pos[tl * K + at]] = rc.scale;
  auto put = [&](int c, const uint4& a, const uint4& b) {
    const uint2 lo = code8<T16>(a, rc), hi = code8<T16>(b, rc);
    for (int j = 0; j < K; ++j) {
      const int ps = pos[tl * K + j];
      if (ps >= 0)
        reinterpret_cast<uint4*>(q_sorted + static_cast<size_t>(ps) * H)[c] =
            make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  };
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (at + i * kStep < pairs) put(at + i * kStep, v[2 * i], v[2 * i + 1]);
  for (int c = at + P * kStep; c < pairs; c += kStep) put(c, src[2 * c], src[2 * c + 1]);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T16, int LPR, int P>
int launch_quantize_short(const T16* x, int64_t rows, int cols, uint8_t* q, float* scale,
                          cudaStream_t stream) {
  const int64_t per_block = 256 / LPR;
  const unsigned grid = static_cast<unsigned>((rows + per_block - 1) / per_block);
  quantize_int8_short_kernel<T16, LPR, P><<<grid, 256, 0, stream>>>(x, static_cast<int>(rows), cols,
                                                                    q, scale);
  return check_launch();
}

template <typename T16>
int launch_quantize(const void* x, int64_t rows, int cols, uint8_t* q, float* scale,
                    cudaStream_t stream) {
  const T16* xp = static_cast<const T16*>(x);
  if (cols <= 16) return launch_quantize_short<T16, 2, 1>(xp, rows, cols, q, scale, stream);
  if (cols <= 64) return launch_quantize_short<T16, 4, 2>(xp, rows, cols, q, scale, stream);
  if (cols <= 256) return launch_quantize_short<T16, 8, 4>(xp, rows, cols, q, scale, stream);
  if (cols <= 512) return launch_quantize_short<T16, 16, 4>(xp, rows, cols, q, scale, stream);
  if (cols <= 1024) return launch_quantize_short<T16, 32, 4>(xp, rows, cols, q, scale, stream);
  if (cols <= 2048) return launch_quantize_short<T16, 32, 8>(xp, rows, cols, q, scale, stream);
  const unsigned grid = static_cast<unsigned>(rows);
  if (cols <= 4096)
    quantize_int8_block_kernel<T16, 128, 4><<<grid, 128, 0, stream>>>(xp, cols, q, scale);
  else if (cols <= 8192)
    quantize_int8_block_kernel<T16, 256, 4><<<grid, 256, 0, stream>>>(xp, cols, q, scale);
  else if (cols <= kRegCols)
    quantize_int8_block_kernel<T16, 256, 8><<<grid, 256, 0, stream>>>(xp, cols, q, scale);
  else
    quantize_int8_long_kernel<T16><<<grid, 256, 0, stream>>>(xp, cols, q, scale);
  return check_launch();
}

template <typename T16>
int launch_permute(const void* x, int T, int H, int E, int K, const int32_t* ids,
                   const int* offsets, uint8_t* q, float* scale, int32_t* slot_pos,
                   cudaStream_t stream) {
  const int nb = (T - 1) / kRouteTokens + 1;  // T > 0; T + 31 may pass 32 bits
  const size_t smem = (2 * static_cast<size_t>(E) + kRouteTokens * K) * 4;  // at most 10 KB
  const T16* xp = static_cast<const T16*>(x);
  // Few tokens: all eight warps on one, so that every SM has a row. Else as many as hold a row of that
  // length in their registers. 16384 tokens x 4096 columns, two choices: 48 us (5.6 TB/s); 67 us with
  // one warp per row that reads it twice and stores 8 bytes a lane.
  if (4 * nb <= 148)
    permute_int8_kernel<T16, 8, 2><<<dim3(nb, 32), 256, smem, stream>>>(
        xp, T, H, E, K, ids, offsets, q, scale, slot_pos);
  else if (H <= 2048)
    permute_int8_kernel<T16, 1, 4><<<dim3(nb, 4), 256, smem, stream>>>(
        xp, T, H, E, K, ids, offsets, q, scale, slot_pos);
  else if (H <= 4096)
    permute_int8_kernel<T16, 2, 4><<<dim3(nb, 8), 256, smem, stream>>>(
        xp, T, H, E, K, ids, offsets, q, scale, slot_pos);
  else
    permute_int8_kernel<T16, 4, 4><<<dim3(nb, 16), 256, smem, stream>>>(
        xp, T, H, E, K, ids, offsets, q, scale, slot_pos);
  return check_launch();
}

}  // namespace
}  // namespace ggo

extern "C" {

int ggo_quantize_int8_rows(const void* x_dev, int64_t rows, int64_t cols, int dtype, void* q_dev,
                           float* scale_dev, cudaStream_t stream) {
  if (rows < 0 || cols <= 0) return GGO_ERR_INVALID_ARG;
  if (dtype != GGO_DTYPE_BF16 && dtype != GGO_DTYPE_FP16) return GGO_ERR_DTYPE;
  if (rows == 0) return GGO_OK;
  if (!x_dev || !q_dev || !scale_dev) return GGO_ERR_INVALID_ARG;
  if (cols % 16 || !ggo::aligned16(x_dev) || !ggo::aligned16(q_dev)) return GGO_ERR_ALIGNMENT;
  if (rows > INT32_MAX || cols > INT32_MAX) return GGO_ERR_SHAPE;
  uint8_t* q = static_cast<uint8_t*>(q_dev);
  const int c = static_cast<int>(cols);
  return dtype == GGO_DTYPE_BF16
             ? ggo::launch_quantize<__nv_bfloat16>(x_dev, rows, c, q, scale_dev, stream)
             : ggo::launch_quantize<__half>(x_dev, rows, c, q, scale_dev, stream);
}

int ggo_moe_permute_int8(const void* x_dev, int64_t num_tokens, int64_t hidden, int num_experts,
                         int top_k, const int32_t* topk_ids_dev, void* q_sorted_dev,
                         float* scale_sorted_dev, int32_t* slot_pos_dev, const void* scratch_dev,
                         int dtype, cudaStream_t stream) {
  if (num_tokens < 0 || hidden <= 0 || num_experts <= 0 || num_experts > ggo::kMaxExperts ||
      top_k <= 0 || top_k > ggo::kMaxTopK || top_k > num_experts)
    return GGO_ERR_INVALID_ARG;
  if (dtype != GGO_DTYPE_BF16 && dtype != GGO_DTYPE_FP16) return GGO_ERR_DTYPE;
  if (num_tokens == 0) return GGO_OK;
  if (!x_dev || !topk_ids_dev || !q_sorted_dev || !scale_sorted_dev || !slot_pos_dev ||
      !scratch_dev)
    return GGO_ERR_INVALID_ARG;
  if (hidden % 16 || !ggo::aligned16(x_dev) || !ggo::aligned16(q_sorted_dev))
    return GGO_ERR_ALIGNMENT;
  if (num_tokens * top_k > INT32_MAX || hidden > INT32_MAX) return GGO_ERR_SHAPE;
  const int T = static_cast<int>(num_tokens), H = static_cast<int>(hidden);
  uint8_t* q = static_cast<uint8_t*>(q_sorted_dev);
  const int* off = static_cast<const int*>(scratch_dev);
  return dtype == GGO_DTYPE_BF16
             ? ggo::launch_permute<__nv_bfloat16>(x_dev, T, H, num_experts, top_k, topk_ids_dev, off,
                                                  q, scale_sorted_dev, slot_pos_dev, stream)
             : ggo::launch_permute<__half>(x_dev, T, H, num_experts, top_k, topk_ids_dev, off, q,
                                           scale_sorted_dev, slot_pos_dev, stream);
}

}  // extern "C"
