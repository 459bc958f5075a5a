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
// call finds all of them by reading the whole slot map, 4 bytes a token out of L2; the
// blocks of its other tokens leave it alone. Slots given twice take the later token's row.
// A wave then takes a page of one KV head, K or V: up to 16 rows in registers, their
// largest bits (bf16 magnitudes order as integers), and the bytes out by the scaling
// conversions, two numbers at a time. Of a page with one new row (a decode step's) it takes
// four heads of 128 at once.
//
// Measured (8 KV heads of 128, us, the kernel's trace; K and V are read and written once at
// 4.9 TB/s in brackets): 1 token 2.4, 256 tokens of as many sequences 4.6 (0.3), 1536 6.2
// (2.0), 8 prompts of 1000 16.5 (10.3), 16 of 1000 26.7 (20.2), 32 of 1024 62 (41), 64 of 1024
// 147 (82). A few tokens are two memory accesses, a barrier and one more; prompts are bound by
// how few pages they are (500, 16 waves each), and past 16000 tokens by the map: each page, or
// each two that begin in one block, reads all of it, in every block of its heads.
// Before the one-row form, with a page's heads to a wave each, 1536 tokens took 15.4; with
// conversions through fp32 and the map read token by token, prompts of 8 x 1000 took 43.
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
};

constexpr int ROWS = 16;          // of a page
constexpr int LEAST_SCALE = 27;   // 2^-100: far from what fp32 flushes
constexpr int NO_SCALE = 255;     // E8M0's not-a-number: a page that holds nothing
constexpr int INF = 0x7f80;       // bf16

// 2^(e - 127) as the scaling conversions take it
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned int)e << 23); }

typedef short short2_t __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// eight numbers over 2^(e - 127), rounded to nearest even
__device__ __forceinline__ uint2 encode8(uint4 x, int e) {
  const unsigned int w[4] = {x.x, x.y, x.z, x.w};
  unsigned int o[2];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    short2_t two = short2_t{0, 0};
    two = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(
        two, __builtin_bit_cast(bf16x2_t, w[2 * d]), pow2(e), false);
    two = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(
        two, __builtin_bit_cast(bf16x2_t, w[2 * d + 1]), pow2(e), true);
    o[d] = __builtin_bit_cast(unsigned int, two);
  }
  return uint2{o[0], o[1]};
}

// the bytes of what is no finite number put in: 448 (all ones but the last bit) or none
__device__ __forceinline__ uint2 encode_special8(uint4 x, uint2 codes) {
  const unsigned int w[4] = {x.x, x.y, x.z, x.w};
  unsigned int o[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int b = (int)(w[i >> 1] >> (i & 1) * 16 & 0xffff), m = b & 0x7fff;
    const int at = (i & 3) * 8;
    const unsigned int code = (m > INF ? 0x7fu : 0x7eu) | (unsigned int)b >> 15 << 7;
    if (m >= INF) o[i >> 2] = (o[i >> 2] & ~(0xffu << at)) | code << at;
  }
  return uint2{o[0], o[1]};
}

// eight E4M3 numbers times 2^(from - to), at most 1
__device__ __forceinline__ uint2 rescale8(uint2 x, int from, int to) {
  auto two = [&](unsigned int w, bool high) {
    return __builtin_bit_cast(
        unsigned int, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, pow2(from), true)
                           : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, pow2(from), false));
  };
  return encode8(uint4{two(x.x, false), two(x.x, true), two(x.y, false), two(x.y, true)}, to);
}

// zeros with the signs of eight E4M3 numbers; what is no number stays none
__device__ __forceinline__ uint2 no_numbers8(uint2 x) {
  auto four = [](unsigned int w) {
    const unsigned int sign = w & 0x80808080u;
    // a carry into the top bit where the lower seven are all ones
    const unsigned int none = ((w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u) >> 7;
    return sign | none * 0x7f;
  };
  return uint2{four(x.x), four(x.y)};
}

// bf16 magnitudes of eight numbers, the largest of two at a time
__device__ __forceinline__ ushort2_t largest8(uint4 x) {
  auto two = [](unsigned int w) { return __builtin_bit_cast(ushort2_t, w & 0x7fff7fffu); };
  return __builtin_elementwise_max(__builtin_elementwise_max(two(x.x), two(x.y)),
                                   __builtin_elementwise_max(two(x.z), two(x.w)));
}

// token_of: the call's token of each row of the page, -1 without
template <int D, bool VEC>
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
  uint4 x[NI];
  int token[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    token[i] = token_of[i * RPI + lrow];
    x[i] = uint4{0, 0, 0, 0};
    if (token[i] >= 0) {
      const short* from = src + token[i] * stride;
      if constexpr (VEC) {
        x[i] = *reinterpret_cast<const uint4*>(from);
      } else {
        short8_t e;
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = from[j];
        x[i] = __builtin_bit_cast(uint4, e);
      }
    }
  }
  ushort2_t two = largest8(x[0]);
#pragma unroll
  for (int i = 1; i < NI; ++i) two = __builtin_elementwise_max(two, largest8(x[i]));
  int top = max((int)two[0], (int)two[1]);
  const bool special = __any(top >= INF);
  if (special) {  // the largest of the finite ones
    top = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const short8_t e = __builtin_bit_cast(short8_t, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, (e[j] & 0x7fff) >= INF ? 0 : e[j] & 0x7fff);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
  // 448 = 1.75 * 2^8
  const int need = max((top >> 7) - 8 + ((top & 0x7f) > 0x60 ? 1 : 0), LEAST_SCALE);
  const bool begun = token_of[0] >= 0;
  const int old = old_raw == NO_SCALE ? 0 : old_raw;
  const int now = begun ? need : max(old, need);
  const bool rescale = !begun && now != old_raw;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    unsigned char* to = rows + i * RPI * D;
    if (token[i] >= 0) {
      uint2 codes = encode8(x[i], now);
      if (special) codes = encode_special8(x[i], codes);
      *reinterpret_cast<uint2*>(to) = codes;
    } else if (rescale) {
      // from 2^-126 at least: what is smaller by 2^26 than the new scale is 0 in any case
      uint2 codes = rescale8(*reinterpret_cast<const uint2*>(to), max(old, 1), now);
      if (old_raw == NO_SCALE) codes = no_numbers8(*reinterpret_cast<const uint2*>(to));
      *reinterpret_cast<uint2*>(to) = codes;
    }
  }
  if (lane == 0 && now != old_raw) *scale = (unsigned char)now;
}

// The same where `token` alone is written, to row `off`: a wave takes 64 / (D / 8) heads.
template <int D, bool VEC>
__device__ __forceinline__ void write_scaled_row(const ScaledWrite& p, int token, int off,
                                                 long page, int task) {
  constexpr int LPR = D / 8, HEADS = 64 / LPR;
  const int lane = threadIdx.x & 63, col = lane % LPR * 8;
  const int item = task * HEADS + lane / LPR;
  const bool used = item < 2 * p.Hkv;
  const bool is_v = item >= p.Hkv;
  const int head = !used ? 0 : is_v ? item - p.Hkv : item;
  const long at = page * p.Hkv + head;
  unsigned char* scale = (is_v ? p.v_scale : p.k_scale) + at;
  unsigned char* rows = (is_v ? p.v_cache : p.k_cache) + at * (ROWS * D) + col;
  const short* from = (is_v ? p.v : p.k) + head * D + col + token * (is_v ? p.sv : p.sk);
  const int old_raw = *scale;
  uint4 x;
  if constexpr (VEC) {
    x = *reinterpret_cast<const uint4*>(from);
  } else {
    short8_t e;
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = from[j];
    x = __builtin_bit_cast(uint4, e);
  }
  const ushort2_t two = largest8(x);
  int top = max((int)two[0], (int)two[1]);
  const bool special = __any(top >= INF);
  if (special) {
    top = 0;
    const short8_t e = __builtin_bit_cast(short8_t, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, (e[j] & 0x7fff) >= INF ? 0 : e[j] & 0x7fff);
  }
#pragma unroll
  for (int step = LPR / 2; step > 0; step >>= 1) top = max(top, __shfl_xor(top, step, 64));
  const int need = max((top >> 7) - 8 + ((top & 0x7f) > 0x60 ? 1 : 0), LEAST_SCALE);
  const int old = old_raw == NO_SCALE ? 0 : old_raw;
  const int now = off == 0 ? need : max(old, need);
  if (!used) return;
  uint2 codes = encode8(x, now);
  if (special) codes = encode_special8(x, codes);
  if (off != 0 && now != old_raw) {
    constexpr int AHEAD = 4;
#pragma unroll 1
    for (int r = 0; r < ROWS; r += AHEAD) {
      uint2 kept[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        kept[i] = *reinterpret_cast<const uint2*>(rows + (r + i) * D);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        *reinterpret_cast<uint2*>(rows + (r + i) * D) =
            old_raw == NO_SCALE ? no_numbers8(kept[i]) : rescale8(kept[i], max(old, 1), now);
    }
  }
  *reinterpret_cast<uint2*>(rows + off * D) = codes;
  if (lane % LPR == 0 && now != old_raw) *scale = (unsigned char)now;
}

// `per` (64 at most) consecutive tokens to a block, the pages that begin among them two at a
// time; VEC: rows and the slot map are 16-byte aligned
template <int D, bool VEC>
__global__ __launch_bounds__(512, 6) void write_scaled_kernel(const ScaledWrite p, const int per) {
  constexpr int PAIR = 2;
  __shared__ int token_of[PAIR][ROWS];
  __shared__ int taken[PAIR];  // an earlier token's block writes this page
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  const int first = blockIdx.x * per;
  auto page_of = [&](int slot) { return (unsigned int)slot < p.limit ? slot >> 4 : -1; };
  // the first tokens of runs in one page: one to a lane
  const int mine = min(first + lane, p.T - 1);
  const int page_here = page_of(p.slots[mine]);
  const int page_before = mine > 0 ? page_of(p.slots[mine - 1]) : -1;
  unsigned long todo = __ballot(lane < per && first + lane < p.T && page_here >= 0 &&
                                page_here != page_before);
  while (todo) {
    int t[PAIR], page[PAIR];
#pragma unroll
    for (int b = 0; b < PAIR; ++b) {
      const int at = todo ? __builtin_ctzl(todo) : 0;
      t[b] = first + at;
      page[b] = todo ? __builtin_amdgcn_readlane(page_here, at) : -1;
      todo &= todo - (todo ? 1 : 0);
    }
    if (threadIdx.x < PAIR * ROWS) token_of[threadIdx.x / ROWS][threadIdx.x % ROWS] = -1;
    if (threadIdx.x < PAIR) taken[threadIdx.x] = 0;
    __syncthreads();
    auto here = [&](int slot) {
      const unsigned int at = (unsigned int)slot >> 4;  // (negative: no page's)
      return at == (unsigned int)page[0] || at == (unsigned int)page[1];
    };
    auto look = [&](int j) {
      const int slot = p.slots[j];
#pragma unroll
      for (int b = 0; b < PAIR; ++b) {
        if ((unsigned int)slot >> 4 != (unsigned int)page[b]) continue;
        if (j < t[b]) taken[b] = 1;
        else atomicMax(&token_of[b][slot & (ROWS - 1)], j);
      }
    };
    // eight tokens at a time, looked at singly only where one of them is of these pages
    const int whole = VEC ? p.T & ~7 : 0;
    for (int j = threadIdx.x * 8; j < whole; j += blockDim.x * 8) {
      const int4 a = *reinterpret_cast<const int4*>(p.slots + j);
      const int4 b = *reinterpret_cast<const int4*>(p.slots + j + 4);
      if (here(a.x) | here(a.y) | here(a.z) | here(a.w) | here(b.x) | here(b.y) | here(b.z) |
          here(b.w)) {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) look(j + i);
      }
    }
    for (int j = whole + threadIdx.x; j < p.T; j += blockDim.x) look(j);
    __syncthreads();
    // one row (a decode step's) or several: the pages' tasks one after the other
    unsigned int given[PAIR];
    int tasks[PAIR];
#pragma unroll
    for (int b = 0; b < PAIR; ++b) {
      given[b] = (unsigned int)__ballot(lane < ROWS && token_of[b][lane % ROWS] >= 0) & 0xffff;
      const bool one = (given[b] & (given[b] - 1)) == 0;
      tasks[b] = given[b] == 0 || taken[b] ? 0 : one ? (2 * p.Hkv * (D / 8) + 63) / 64 : 2 * p.Hkv;
    }
    for (int task = blockIdx.y * waves + wave; task < tasks[0] + tasks[1];
         task += gridDim.y * waves) {
      const int b = task >= tasks[0];
      const int of = b ? task - tasks[0] : task;
      const unsigned int rows = b ? given[1] : given[0];
      const int at = b ? page[1] : page[0];
      if ((rows & (rows - 1)) == 0) {
        const int off = __builtin_ctz(rows);
        write_scaled_row<D, VEC>(p, token_of[b][off], off, at, of);
      } else {
        write_scaled_page<D, VEC>(p, token_of[b], at, of);
      }
    }
    if (todo) __syncthreads();
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
  const bool vec =
      ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)slots) & 15) | ((sk | sv) & 7)) == 0;
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
                      sv};
  // Tokens to a block, and blocks to a page's heads. One of eight waves, for two tokens each,
  // up to what a decode step has (us, 1536 tokens of as many sequences / 2 prompts of 1000:
  // so 6.0 / 11.0, two blocks 8.5 / 8.3, one for four tokens 8.0 / 8.4: steps are the more
  // frequent); above, prompts (8 of 1000: about 1024 blocks 15.2, half as many 16.4, twice
  // 19.5).
  const int per = T <= 512 ? 1 : T <= 2048 ? 2 : T >= 65536 ? 64 : (int)((T + 1023) / 1024);
  // a page's heads, K and V, in blocks of up to eight waves
  const long tasks = 2 * Hkv;
  const long parts = T <= 2048 ? 1 : tasks <= 8 * 64 ? (tasks + 7) / 8 : 64;
  const dim3 grid((unsigned)((T + per - 1) / per), (unsigned)parts);
  const dim3 block(64 * (unsigned)(tasks < 8 ? tasks : 8));
#define GO(DD, VV) \
  hipLaunchKernelGGL((write_scaled_kernel<DD, VV>), grid, block, 0, stream, p, per)
  if (D == 128) {
    if (vec) GO(128, true);
    else GO(128, false);
  } else {
    if (vec) GO(64, true);
    else GO(64, false);
  }
#undef GO
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
