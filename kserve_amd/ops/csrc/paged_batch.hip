// What attention over a paged cache is told of a batch, from its requests' page lists
// and lengths: cu_seqlens are the exclusive sums of the new lengths; token t of request
// s stands at position computed_s + t - cu_s and in slot pages_s[pos / block] * block +
// pos % block; a row of the page tables holds the pages that the request's computed and
// new tokens fill, and zeros (the scratch page) behind them.
//
// One launch: the blocks of the first part take TOKENS tokens each and find their
// requests by the sums of the lengths, which every block forms by itself, 1024 at a time
// in LDS (cheaper than a launch that forms them once: 64 blocks of 1024 lengths read
// 256 KB out of L2); the blocks of the second part take TABLE table entries each.
#include "common.h"

namespace {

constexpr int TOKENS = 1024;  // of a block, 4 to a thread
constexpr int TABLE = 4096;   // entries of a block, in steps of 4 to a thread
constexpr int CHUNK = 1024;   // requests whose sums are in LDS at a time

struct BatchArgs {
  const int* pages;        // [P] requests' pages one after the other
  const int* page_starts;  // [S + 1] where each begins
  const int* computed;     // [S] tokens that are in pages already
  const int* fresh;        // [S] new tokens
  long* positions;         // [T]
  int* slots;              // [T]
  int* seqs;               // [T]
  int* cu;                 // [S + 1]
  int* tables;             // [S, width]
  int* ctx;                // [S]
  int P, S, T, width, block;
  int token_blocks;
};

// the request's pages inside the list: {first, count}
__device__ __forceinline__ int2 page_span(const BatchArgs& p, int s) {
  const int a = min(max(p.page_starts[s], 0), p.P);
  const int b = min(max(p.page_starts[s + 1], a), p.P);
  return int2{a, b - a};
}

__device__ void token_part(const BatchArgs& p) {
  // first token of each of a chunk's requests, and the end of the last
  __shared__ long sums[CHUNK + 1];
  __shared__ long part[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long t0 = (long)blockIdx.x * TOKENS + threadIdx.x * 4;
  long pos[4] = {0, 0, 0, 0};
  int slot[4] = {-1, -1, -1, -1}, seq[4] = {-1, -1, -1, -1};
  long base = 0;
  for (int s0 = 0; s0 < p.S; s0 += CHUNK) {
    long len[4], mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + threadIdx.x * 4 + i;
      len[i] = s < p.S ? max(p.fresh[s], 0) : 0;
      mine += len[i];
    }
    long up = mine;  // inclusive over the wave
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const long x = __shfl_up(up, off, 64);
      if (lane >= off) up += x;
    }
    if (lane == 63) part[wave] = up;
    __syncthreads();
    long at = base + up - mine;
    for (int w = 0; w < wave; ++w) at += part[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sums[threadIdx.x * 4 + i] = at;
      at += len[i];
    }
    if (threadIdx.x == 255) sums[CHUNK] = at;
    __syncthreads();
    const int n = min(CHUNK, p.S - s0);
    const long end = sums[n];
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i < n; i += 256)
        p.cu[s0 + i] = (int)min(sums[i], (long)p.T);
      if (s0 + n == p.S && threadIdx.x == 0) p.cu[p.S] = (int)min(end, (long)p.T);
    }
    if (t0 + 4 > base && t0 < end) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long t = t0 + i;
        if (t < base || t >= end || t >= p.T) continue;
        int lo = 0, hi = n;  // the last request that begins at or before t
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (sums[mid] <= t) lo = mid;
          else hi = mid;
        }
        const int s = s0 + lo;
        const unsigned int at_pos =
            (unsigned int)max(p.computed[s], 0) + (unsigned int)(t - sums[lo]);
        const unsigned int j = at_pos / (unsigned int)p.block;
        const int2 span = page_span(p, s);
        pos[i] = at_pos;
        seq[i] = s;
        if (j < (unsigned int)span.y) {
          const long at_slot =
              (long)p.pages[span.x + j] * p.block + (at_pos - j * (unsigned int)p.block);
          if (at_slot >= 0 && at_slot <= 0x7fffffffL) slot[i] = (int)at_slot;
        }
      }
    }
    base = sums[CHUNK];
    __syncthreads();  // before the next chunk's sums
    if (base > t0 - threadIdx.x * 4 + TOKENS && blockIdx.x != 0) break;
  }
  if (p.S == 0 && blockIdx.x == 0 && threadIdx.x == 0) p.cu[0] = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t0 + i < p.T) {
      p.positions[t0 + i] = pos[i];
      p.slots[t0 + i] = slot[i];
      p.seqs[t0 + i] = seq[i];
    }
}

__device__ void table_part(const BatchArgs& p) {
  const unsigned int total = (unsigned int)p.S * p.width;  // below 2^31
  const unsigned int first = (blockIdx.x - p.token_blocks) * (unsigned int)TABLE;
  for (int step = 0; step < TABLE; step += 1024) {
    const unsigned int at = first + step + threadIdx.x * 4;
    if (at >= total) break;
    int s = (int)(at / p.width), c = (int)(at - s * (unsigned int)p.width);
    auto held_of = [&](int2 span) {
      const long ctx = (long)max(p.computed[s], 0) + max(p.fresh[s], 0);
      return (int)min((ctx + p.block - 1) / p.block, (long)span.y);
    };
    int2 span = page_span(p, s);
    int held = held_of(span);
    int4 id{0, 0, 0, 0};
    if (c + 4 <= p.width) {  // of one row; at a multiple of 4 bytes only
      if (c + 4 <= held) __builtin_memcpy(&id, p.pages + span.x + c, 16);
      else if (c < held) {
        id.x = p.pages[span.x + c];
        if (c + 1 < held) id.y = p.pages[span.x + c + 1];
        if (c + 2 < held) id.z = p.pages[span.x + c + 2];
      }
    } else {
      int one[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (at + i >= total) continue;
        if (c < held) one[i] = p.pages[span.x + c];
        if (++c == p.width && ++s < p.S) {
          c = 0;
          span = page_span(p, s);
          held = held_of(span);
        }
      }
      id = int4{one[0], one[1], one[2], one[3]};
    }
    if (at + 4 <= total) {
      *reinterpret_cast<int4*>(p.tables + at) = id;
    } else {
      const int one[4] = {id.x, id.y, id.z, id.w};
      for (unsigned int i = 0; i < 3 && at + i < total; ++i) p.tables[at + i] = one[i];
    }
  }
}

__global__ __launch_bounds__(256) void paged_batch_kernel(const BatchArgs p) {
  const int s = blockIdx.x * 256 + threadIdx.x;
  for (int i = s; i < p.S; i += gridDim.x * 256)
    p.ctx[i] = (int)min((long)max(p.computed[i], 0) + max(p.fresh[i], 0), 0x7fffffffL);
  if ((int)blockIdx.x < p.token_blocks) token_part(p);
  else table_part(p);
}

}  // namespace

// `tables` is 16-byte aligned
extern "C" hipError_t ks_paged_batch(const void* pages, const void* page_starts,
                                     const void* computed, const void* fresh, long P, long S,
                                     long T, long width, long block, void* positions,
                                     void* slots, void* seqs, void* cu, void* tables,
                                     void* ctx, hipStream_t stream) {
  constexpr long MOST = 0x7fffffffL;
  if (P < 0 || S < 0 || T < 0 || width < 0 || block < 1 || P > MOST || S >= MOST / 4 ||
      T > MOST - TOKENS || block > MOST || S * width > MOST)
    return hipErrorInvalidValue;
  // one block of tokens at least: it writes cu_seqlens
  const int token_blocks = T > TOKENS ? (int)((T + TOKENS - 1) / TOKENS) : 1;
  const int table_blocks = (int)((S * width + TABLE - 1) / TABLE);
  const BatchArgs p{(const int*)pages, (const int*)page_starts, (const int*)computed,
                    (const int*)fresh, (long*)positions, (int*)slots, (int*)seqs, (int*)cu,
                    (int*)tables, (int*)ctx, (int)P, (int)S, (int)T, (int)width, (int)block,
                    token_blocks};
  hipLaunchKernelGGL(paged_batch_kernel, dim3(token_blocks + table_blocks), dim3(256), 0,
                     stream, p);
  HIP_CHECK_KERNEL();
  return hipSuccess;
}
