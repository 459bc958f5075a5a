// Scatter new K/V rows into the paged cache.
//
// Cache layout [num_blocks, Hkv, block_size, D]: each (block, head) tile is a
// contiguous block_size*D*2-byte region (4 KB at 16x128 bf16) — the unit the
// decode kernel stages through LDS.
#include "common.h"

namespace {

__global__ void reshape_and_cache_kernel(
    const short* __restrict__ k,  // [T, Hkv, D]
    const short* __restrict__ v,  // [T, Hkv, D]
    short* __restrict__ k_cache,  // [B, Hkv, bs, D]
    short* __restrict__ v_cache,
    const int* __restrict__ slot_mapping,  // [T]
    const int T, const int Hkv, const int D, const int block_size,
    const long sk, const long sv) {
  const int t = blockIdx.x;
  if (t >= T) return;
  const int slot = slot_mapping[t];
  if (slot < 0) return;  // padding slot
  const int blk = slot / block_size;
  const int off = slot % block_size;
  const int nvec = (Hkv * D) >> 3;
  const short8_t* k_src = reinterpret_cast<const short8_t*>(k + (long)t * sk);
  const short8_t* v_src = reinterpret_cast<const short8_t*>(v + (long)t * sv);
  const int dvec = D >> 3;
  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    const int h = i / dvec;
    const int dv = i % dvec;
    const long dst =
        (((long)blk * Hkv + h) * block_size + off) * dvec + dv;
    reinterpret_cast<short8_t*>(k_cache)[dst] = k_src[i];
    reinterpret_cast<short8_t*>(v_cache)[dst] = v_src[i];
  }
}

// fp8 (OCP E4M3) cache variant: bf16 rows are converted pairwise with
// v_cvt_pk_fp8_f32 at store time (scale 1.0; E4M3 range +-448 covers
// RMSNorm'd projections). Halves KV bytes -> ~2x decode-attention bandwidth
// for engines opting into kv_cache_dtype="fp8".
__global__ void reshape_and_cache_fp8_kernel(
    const short* __restrict__ k, const short* __restrict__ v,
    unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache,
    const int* __restrict__ slot_mapping, const int T, const int Hkv,
    const int D, const int block_size, const long sk, const long sv) {
  const int t = blockIdx.x;
  if (t >= T) return;
  const int slot = slot_mapping[t];
  if (slot < 0) return;
  const int blk = slot / block_size;
  const int off = slot % block_size;
  const int nvec = (Hkv * D) >> 3;  // 8 values -> 8 bytes out
  const short8_t* k_src = reinterpret_cast<const short8_t*>(k + (long)t * sk);
  const short8_t* v_src = reinterpret_cast<const short8_t*>(v + (long)t * sv);
  const int dvec = D >> 3;
  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    const int h = i / dvec;
    const int dv = i % dvec;
    const long dst = (((long)blk * Hkv + h) * block_size + off) * dvec + dv;
    short8_t kv = k_src[i];
    short8_t vv = v_src[i];
    // the builtin's word-select must be a literal; unroll by hand
#define CVT2(dst_, a, b, w) \
    dst_ = __builtin_amdgcn_cvt_pk_fp8_f32( \
        bf16_bits_to_float(a), bf16_bits_to_float(b), dst_, w)
    unsigned int kpk0 = 0, kpk1 = 0, vpk0 = 0, vpk1 = 0;
    CVT2(kpk0, kv[0], kv[1], false);
    CVT2(kpk0, kv[2], kv[3], true);
    CVT2(kpk1, kv[4], kv[5], false);
    CVT2(kpk1, kv[6], kv[7], true);
    CVT2(vpk0, vv[0], vv[1], false);
    CVT2(vpk0, vv[2], vv[3], true);
    CVT2(vpk1, vv[4], vv[5], false);
    CVT2(vpk1, vv[6], vv[7], true);
#undef CVT2
    reinterpret_cast<unsigned int*>(k_cache)[dst * 2] = kpk0;
    reinterpret_cast<unsigned int*>(k_cache)[dst * 2 + 1] = kpk1;
    reinterpret_cast<unsigned int*>(v_cache)[dst * 2] = vpk0;
    reinterpret_cast<unsigned int*>(v_cache)[dst * 2 + 1] = vpk1;
  }
}

// Block-scaled E4M3 cache: the bytes of a page of one KV head stand for code * 2^e, and
// e + 127 is the head's byte of the page's scales (E8M0). New rows ask for the least 2^e,
// 2^-100 at least, that brings the largest of their finite values to 448 or below. A call
// that writes a page's first row begins the page anew under that scale; otherwise the
// page keeps the larger of its own and the new one, and where that is the new one its
// other rows are rounded to it: a power of two leaves E4M3's normal numbers as they are.
// Infinities become +-448 * 2^e.
//
// A page's rows have to be known together, so the block of a page's first token in the
// call (`own`) finds all of them by reading the whole slot map, 4 bytes a token out of
// L2; the blocks of its other tokens end. Slots given twice take the later token's row.
// A wave then takes a page of one KV head, K or V: up to 16 rows in registers, their
// largest bits (bf16 magnitudes order as integers), and the bytes out.
struct ScaledWrite {
  const short* k;  // [T, Hkv, D], rows sk elements apart
  const short* v;
  unsigned char* k_cache;  // [pages, Hkv, 16, D]
  unsigned char* v_cache;
  unsigned char* k_scale;  // [pages, Hkv]
  unsigned char* v_scale;
  const int* slots;  // [T]
  int T, Hkv;
  unsigned int limit;  // slots of the cache
  long sk, sv;
  int vec;  // rows are 16-byte aligned
};

constexpr int ROWS = 16;          // of a page
constexpr int LEAST_SCALE = 27;   // 2^-100: far from what fp32 flushes
constexpr int NO_SCALE = 255;     // E8M0's not-a-number: a page that holds nothing

__device__ __forceinline__ float pow2(int e) {  // 2^e, 0 below 2^-126; e < 128
  return __uint_as_float(e < -126 ? 0u : (unsigned int)(e + 127) << 23);
}

__device__ __forceinline__ unsigned int to_fp8(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned int)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}

// eight bf16 numbers times inv (the largest of the finite ones 448 at most)
__device__ __forceinline__ uint2 encode8(short8_t x, float inv, bool special) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const short b = special && (x[i] & 0x7fff) >= 0x7f80 ? (short)0 : x[i];
    f[i] = bf16_bits_to_float(b) * inv;
  }
  unsigned int w[2] = {to_fp8(f[0], f[1], f[2], f[3]), to_fp8(f[4], f[5], f[6], f[7])};
  if (special) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned int m = x[i] & 0x7fff;
      const unsigned int code = (m > 0x7f80 ? 0x7fu : 0x7eu) | (x[i] < 0 ? 0x80u : 0u);
      if (m >= 0x7f80) w[i >> 2] = (w[i >> 2] & ~(0xffu << (i & 3) * 8)) | code << (i & 3) * 8;
    }
  }
  return uint2{w[0], w[1]};
}

// eight E4M3 numbers times ratio, at most 1
__device__ __forceinline__ uint2 rescale8(uint2 x, float ratio) {
  unsigned int w[2] = {x.x, x.y};
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const float2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[d], false);
    const float2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[d], true);
    w[d] = to_fp8(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
  }
  return uint2{w[0], w[1]};
}

// token_of: the call's token of each row of the page, -1 without
template <int D>
__device__ __forceinline__ void write_scaled_page(const ScaledWrite& p, const int* token_of,
                                                  long page, int task) {
  constexpr int LPR = D / 8, RPI = 64 / LPR, NI = ROWS / RPI;
  const bool is_v = task >= p.Hkv;
  const int head = is_v ? task - p.Hkv : task;
  const int lane = threadIdx.x & 63, lrow = lane / LPR, col = lane % LPR * 8;
  const long at = page * p.Hkv + head;
  unsigned char* scale = (is_v ? p.v_scale : p.k_scale) + at;
  unsigned char* rows = (is_v ? p.v_cache : p.k_cache) + at * (ROWS * D) + lrow * D + col;
  const short* src = (is_v ? p.v : p.k) + head * D + col;
  const long stride = is_v ? p.sv : p.sk;
  const int old_raw = *scale;
  short8_t x[NI];
  int token[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    token[i] = token_of[i * RPI + lrow];
    x[i] = short8_t{0, 0, 0, 0, 0, 0, 0, 0};
    if (token[i] >= 0) {
      const short* from = src + token[i] * stride;
      if (p.vec) {
        x[i] = *reinterpret_cast<const short8_t*>(from);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = from[e];
      }
    }
  }
  int top = 0;
  bool special = false;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int m = x[i][e] & 0x7fff;
      special |= m >= 0x7f80;
      top = max(top, m >= 0x7f80 ? 0 : m);
    }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
  special = __any(special);
  // 448 = 1.75 * 2^8
  const int need = max((top >> 7) - 8 + ((top & 0x7f) > 0x60 ? 1 : 0), LEAST_SCALE);
  const bool begun = token_of[0] >= 0;
  const int old = old_raw == NO_SCALE ? 0 : old_raw;
  const int now = begun ? need : max(old, need);
  const float inv = pow2(127 - now);
  const bool rescale = !begun && now != old_raw;
  const float ratio = old_raw == NO_SCALE ? 0.f : pow2(old - now);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    unsigned char* to = rows + i * RPI * D;
    if (token[i] >= 0)
      *reinterpret_cast<uint2*>(to) = encode8(x[i], inv, special);
    else if (rescale)
      *reinterpret_cast<uint2*>(to) = rescale8(*reinterpret_cast<const uint2*>(to), ratio);
  }
  if (lane == 0 && now != old_raw) *scale = (unsigned char)now;
}

// `per` consecutive tokens to a block
template <int D>
__global__ __launch_bounds__(1024) void write_scaled_kernel(const ScaledWrite p, const int per) {
  __shared__ int token_of[ROWS];
  __shared__ int taken;  // an earlier token's block writes this page
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  auto page_of = [&](int slot) { return (unsigned int)slot < p.limit ? slot >> 4 : -1; };
  const int end = min((int)blockIdx.x * per + per, p.T);
  for (int t = blockIdx.x * per; t < end; ++t) {
    const int page = page_of(p.slots[t]);
    if (page < 0 || (t > 0 && page_of(p.slots[t - 1]) == page)) continue;
    if (threadIdx.x < ROWS) token_of[threadIdx.x] = -1;
    if (threadIdx.x == ROWS) taken = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < p.T; j += blockDim.x) {
      const int slot = p.slots[j];
      if (page_of(slot) != page) continue;
      if (j < t) taken = 1;
      else atomicMax(&token_of[slot & (ROWS - 1)], j);
    }
    __syncthreads();
    if (!taken)
      for (int task = wave; task < 2 * p.Hkv; task += waves)
        write_scaled_page<D>(p, token_of, page, task);
    __syncthreads();
  }
}

}  // namespace

extern "C" hipError_t ks_write_scaled_pages(const void* k, const void* v, void* k_cache,
                                            void* v_cache, void* k_scale, void* v_scale,
                                            const void* slots, long T, long Hkv, int D,
                                            long pages, long sk, long sv,
                                            hipStream_t stream) {
  if (T < 0 || T > (1L << 30) || Hkv < 1 || Hkv > (1L << 20) || pages < 0 ||
      (D != 64 && D != 128))
    return hipErrorInvalidValue;
  if (T == 0 || pages == 0) return hipSuccess;
  const bool vec = ((((uintptr_t)k | (uintptr_t)v) & 15) | ((sk | sv) & 7)) == 0;
  const ScaledWrite p{(const short*)k,
                      (const short*)v,
                      (unsigned char*)k_cache,
                      (unsigned char*)v_cache,
                      (unsigned char*)k_scale,
                      (unsigned char*)v_scale,
                      (const int*)slots,
                      (int)T,
                      (int)Hkv,
                      (unsigned int)(pages < (1L << 27) ? pages * ROWS : 1L << 31),
                      sk,
                      sv,
                      vec};
  const int per = T <= 1024 ? 1 : 4;
  const dim3 grid((unsigned)((T + per - 1) / per));
  const dim3 block(64 * (unsigned)(2 * Hkv < 16 ? 2 * Hkv : 16));
  if (D == 128)
    hipLaunchKernelGGL((write_scaled_kernel<128>), grid, block, 0, stream, p, per);
  else
    hipLaunchKernelGGL((write_scaled_kernel<64>), grid, block, 0, stream, p, per);
  HIP_CHECK_KERNEL();
  return hipSuccess;
}

extern "C" hipError_t ks_reshape_and_cache_fp8(
    const void* k, const void* v, void* k_cache, void* v_cache,
    const void* slot_mapping, int T, int Hkv, int D, int block_size, long sk,
    long sv, hipStream_t stream) {
  if (D % 8 != 0 || T == 0) return T == 0 ? hipSuccess : hipErrorInvalidValue;
  int threads = (Hkv * D) >> 3;
  if (threads > 256) threads = 256;
  if (threads < 64) threads = 64;
  hipLaunchKernelGGL(reshape_and_cache_fp8_kernel, dim3(T), dim3(threads), 0,
                     stream, (const short*)k, (const short*)v,
                     (unsigned char*)k_cache, (unsigned char*)v_cache,
                     (const int*)slot_mapping, T, Hkv, D, block_size, sk, sv);
  HIP_CHECK_KERNEL();
  return hipSuccess;
}

extern "C" hipError_t ks_reshape_and_cache(const void* k, const void* v,
                                           void* k_cache, void* v_cache,
                                           const void* slot_mapping, int T,
                                           int Hkv, int D, int block_size,
                                           long sk, long sv,
                                           hipStream_t stream) {
  if (D % 8 != 0 || T == 0) return T == 0 ? hipSuccess : hipErrorInvalidValue;
  int threads = (Hkv * D) >> 3;
  if (threads > 256) threads = 256;
  if (threads < 64) threads = 64;
  hipLaunchKernelGGL(reshape_and_cache_kernel, dim3(T), dim3(threads), 0,
                     stream, (const short*)k, (const short*)v, (short*)k_cache,
                     (short*)v_cache, (const int*)slot_mapping, T, Hkv, D,
                     block_size, sk, sv);
  HIP_CHECK_KERNEL();
  return hipSuccess;
}
