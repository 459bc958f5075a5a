// What attention over a paged cache is told of a batch, from its requests' page lists
// and lengths: cu_seqlens are the exclusive sums of the new lengths; token t of request
// s stands at position computed_s + t - cu_s and in slot pages_s[pos / block] * block +
// pos % block; a row of the page tables holds the pages that the request's computed and
// new tokens fill, and zeros (the scratch page) behind them.
//
// One launch: the blocks of the first part take TOKENS tokens each and find their
// requests by the sums of the lengths, which every block forms by itself, 1024 at a time
// (cheaper than a launch that forms them once: 64 blocks of 1024 lengths read 256 KB out
// of L2); the blocks of the second part take ENTRIES table entries each (four times as
// many one after the other: 96 requests' tables of 130 pages 5.2 to 9.2 us). What bounds
// it: the launch and three dependent reads (96 requests of 5 tokens 4.1 us), with 1024
// tables of 8101 pages the 55 MB (10.6 us, 5.2 TB/s).
#include "common.h"

namespace {

constexpr int TOKENS = 1024;   // of a block, 4 to a thread
constexpr int ENTRIES = 1024;  // of the tables, the same
constexpr int CHUNK = 1024;    // requests whose sums a block forms at a time

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

// Every request marks its first token among the block's in LDS; a scan over the marks then
// gives each token its request (a search for each among the sums: 96 requests 5.7 for 4.1
// us, 1024 of a token 8.8 for 6.1; one request 3.1 for 3.6).
__device__ void token_part(const BatchArgs& p) {
  __shared__ __attribute__((aligned(16))) int owner[TOKENS];  // request that begins here, or -1
  __shared__ unsigned int part[2][4], first_begin;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned int T = p.T, t_block = blockIdx.x * (unsigned int)TOKENS;
  const unsigned int t0 = t_block + threadIdx.x * 4;
  *reinterpret_cast<int4*>(owner + threadIdx.x * 4) = int4{-1, -1, -1, -1};
  // sums stop at 2^32 - 1: no token is behind them
  auto add = [](unsigned int a, unsigned int b) { return __builtin_elementwise_add_sat(a, b); };
  unsigned int base = 0;
  int turn = 0;
  for (int s0 = 0; s0 < p.S; s0 += CHUNK, turn ^= 1) {
    const int s = s0 + threadIdx.x * 4;
    unsigned int len[4], mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      len[i] = s + i < p.S ? max(p.fresh[s + i], 0) : 0;
      mine = add(mine, len[i]);
    }
    const unsigned int up = lanes_up_to(mine, 0, add);
    if (lane == 63) part[turn][wave] = up;
    __syncthreads();
    unsigned int at = base;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at = add(at, part[turn][w]);
      base = add(base, part[turn][w]);
    }
    const unsigned int before = __shfl_up(up, 1, 64);
    if (lane > 0) at = add(at, before);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned int end = add(at, len[i]);
      if (end > t_block && at < t_block + TOKENS && len[i] > 0) {
        owner[at > t_block ? at - t_block : 0] = s + i;
        if (at <= t_block) first_begin = at;
      }
      if (blockIdx.x == 0 && s + i < p.S) p.cu[s + i] = (int)min(at, T);
      at = end;
    }
    if (base >= t_block + TOKENS && blockIdx.x != 0) break;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.cu[p.S] = (int)min(base, T);
  __syncthreads();

  const int4 marks = *reinterpret_cast<const int4*>(owner + threadIdx.x * 4);
  const int mark[4] = {marks.x, marks.y, marks.z, marks.w};
  unsigned int from[4], run = 0;  // 1 + where the token's request is marked
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (mark[i] >= 0) run = threadIdx.x * 4 + i + 1;
    from[i] = run;
  }
  auto most = [](unsigned int a, unsigned int b) { return max(a, b); };
  const unsigned int up = lanes_up_to(run, 0, most);
  if (lane == 63) part[0][wave] = up;
  __syncthreads();
  const unsigned int left = __shfl_up(up, 1, 64);
  unsigned int carry = lane > 0 ? left : 0;
#pragma unroll
  for (int w = 0; w < 3; ++w)
    if (w < wave) carry = max(carry, part[0][w]);

  // four tokens in step, so that their reads are under way together
  int s[4], id[4];
  int2 span[4];
  unsigned int at_pos[4], page[4];
  bool in[4], held[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    from[i] = max(from[i], carry);
    in[i] = from[i] > 0 && t0 + i < min(base, T);
    s[i] = in[i] ? owner[from[i] - 1] : 0;
    const unsigned int begin = from[i] > 1 ? t_block + from[i] - 1 : first_begin;
    at_pos[i] = t0 + i - begin;
    span[i] = int2{0, 0};
    if (in[i]) {
      at_pos[i] += (unsigned int)max(p.computed[s[i]], 0);
      span[i] = page_span(p, s[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    page[i] = at_pos[i] / (unsigned int)p.block;
    held[i] = in[i] && page[i] < (unsigned int)span[i].y;
    id[i] = 0;
    if (held[i]) id[i] = p.pages[span[i].x + page[i]];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t0 + i < T) {
      const long slot = (long)id[i] * p.block + (at_pos[i] - page[i] * (unsigned int)p.block);
      p.positions[t0 + i] = in[i] ? at_pos[i] : 0;
      p.slots[t0 + i] = held[i] && slot >= 0 && slot <= 0x7fffffffL ? (int)slot : -1;
      p.seqs[t0 + i] = in[i] ? s[i] : -1;
    }
}

__device__ void table_part(const BatchArgs& p) {
  const unsigned int total = (unsigned int)p.S * p.width;  // below 2^31
  const unsigned int at =
      (blockIdx.x - p.token_blocks) * (unsigned int)ENTRIES + threadIdx.x * 4;
  if (at >= total) return;
  int s = (int)(at / p.width), c = (int)(at - s * (unsigned int)p.width);
  auto held_of = [&](int row, int2 span) {
    const long ctx = (long)max(p.computed[row], 0) + max(p.fresh[row], 0);
    return (int)min((ctx + p.block - 1) / p.block, (long)span.y);
  };
  int4 id{0, 0, 0, 0};
  if (c + 4 <= p.width) {  // of one row; at a multiple of 4 bytes only
    const int2 span = page_span(p, s);
    const int held = held_of(s, span);
    if (c + 4 <= held) __builtin_memcpy(&id, p.pages + span.x + c, 16);
    else if (c < held) {
      id.x = p.pages[span.x + c];
      if (c + 1 < held) id.y = p.pages[span.x + c + 1];
      if (c + 2 < held) id.z = p.pages[span.x + c + 2];
    }
  } else {
    int from[4], one[4];
    bool any[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int2 span = page_span(p, s);
      any[i] = c < held_of(s, span) && at + i < total;
      from[i] = span.x + c;
      if (++c == p.width && s + 1 < p.S) {
        c = 0;
        ++s;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      one[i] = 0;
      if (any[i]) one[i] = p.pages[from[i]];
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
  const int table_blocks = (int)((S * width + ENTRIES - 1) / ENTRIES);
  const BatchArgs p{(const int*)pages, (const int*)page_starts, (const int*)computed,
                    (const int*)fresh, (long*)positions, (int*)slots, (int*)seqs, (int*)cu,
                    (int*)tables, (int*)ctx, (int)P, (int)S, (int)T, (int)width, (int)block,
                    token_blocks};
  hipLaunchKernelGGL(paged_batch_kernel, dim3(token_blocks + table_blocks), dim3(256), 0,
                     stream, p);
  HIP_CHECK_KERNEL();
  return hipSuccess;
}
