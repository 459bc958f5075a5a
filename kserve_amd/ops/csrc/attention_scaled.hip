// Paged decode attention over the block-scaled E4M3 cache (bf16 queries, one per
// sequence): o = sum_j softmax_j(scale q k_j) v_j, where a page's bytes of one KV head
// stand for code * 2^e.
//
// A block takes the query heads of one KV head of one sequence (or of one of several
// splits of its context); its waves take pairs of pages in turn, each by itself until the
// sums are merged. Both products run transposed on v_mfma_f32_16x16x32_bf16: S^T = K Q^T
// has a query head per lane column, and its registers are the B operand of O^T += V^T P^T
// (contraction index 8 g + j: key 4 g + j of the first page for j < 4, of the second after
// that). Bytes become bf16 by the scaling conversions, which apply the page's power of two
// exactly and for nothing.
//
// K goes from memory into the product's registers: a contraction may take its columns in
// any order that both operands share, so a lane takes 16 consecutive bytes of its key's
// row for two products, and the query is laid out to match. V passes through LDS of the
// wave's own, to be read back by the transposing loads. Neither has addresses per lane:
// a page's rows of one head lie together, and whole pages are read. What lies outside the
// context or the window may be anything: scores there are replaced and rows of V zeroed.
// Page ids and scales are fetched for 32 pairs at once, a page to a lane.
//
// The weights keep 24 bits as three bf16 parts, as in attention_decode.hip: in the 16
// columns side by side for groups of up to five heads, by a second product for six to
// eight.
//
// What bounds it: the pages. 256 sequences of 2048 +- 60% (32 / 8 heads of 128) take 172 us,
// 6.3 TB/s, the longest first; the units' vector instructions are busy for a tenth of that
// and their matrix cores for a tenth. 1 of 131071 under groups of eight 50 with the launch
// that merges (5.3 TB/s); one of 560 8.1: four memory accesses one after the other, and the
// sums.
#include <type_traits>

#include "mfma_attention.h"

namespace {

using namespace mfma_attn;

struct ScaledDecode {
  void* out;                       // [S, H, D] bf16
  const short* q;                  // [S, H, D] bf16, row stride sq
  const unsigned char* k_cache;    // [pages, Hkv, 16, D]
  const unsigned char* v_cache;
  Scales s8;
  const int* block_tables;         // [S, max_blocks]
  const int* ctx_lens;             // [S]
  float scale;
  int H, Hkv, group, max_blocks;
  long sq;
  int n_splits, base;  // most, and those of any context that is long enough
  float* part_out;  // [S, H, n_splits, D]
  float* part_ml;   // [S, H, n_splits, 2]
  int window;
  int sorted;  // keys of a sequence from which on the longest go first, or 0
  int seqs;
  int help;    // rows of blocks ahead of the sequences' that help with long ones, or 0
};

// keys of sequence s: as many as its table row has at most
__device__ __forceinline__ int context_of(const ScaledDecode& p, int s) {
  return min(p.ctx_lens[s], p.max_blocks * PAGE);
}

// Splits of a context: p.base with a pair for every wave at least, or more of PART pairs
constexpr int PART = 128;
__device__ __forceinline__ Range decode_range(const ScaledDecode& p, int ctx, int waves) {
  Range r = page_range(ctx, p.window, 0, p.base, waves);
  const int more = min(r.pairs / PART, p.n_splits);
  if (more > r.splits) {
    r.splits = more;
    r.per = (r.pairs + more - 1) / more;
  }
  return r;
}

// The sequence, and its keys, that block row r of `seqs` takes: of the last LAST rows the
// longest first, to an eighth of its length, so that the launch does not end in one that
// begins late. Every wave finds it by itself, which takes a microsecond: lane l holds the
// lengths of rows l, l + 64, .., and each bit of them, from the highest on, leaves the rows
// that have it or the rest. Where no row reads p.sorted keys nothing is moved.
//
// us, in order / so: one query each, 64 of 2048 +- 60% 51.4 / 48.9, 96 of 3000 +- 60% 105 /
// 95, 160 of 2048 +- 60% 124 / 112, 256 of 2048 +- 60% 188 / 172 and all of 2048 170 / 171,
// 512 of 600 +- 60% 109 / 107, 1536 of 560 286 / 287, 256 of 100 in wide tables 17.8 / 18.4;
// five queries, 64 of 1500 +- 60% 41.4 / 41.0, 96 61 / 58 and all of 1500 58 / 60, 192 120 /
// 110, 256 of 800 +- 60% 78.5 / 81.
constexpr int LAST = 256;
__device__ __forceinline__ int2 longest_first(const ScaledDecode& p, int r, int seqs, int lane) {
  const int first = max(seqs - LAST, 0);
  if (r < first) return int2{r, context_of(p, r)};
  constexpr int N = LAST / 64;
  constexpr int LOW = 20, BITS = 6;  // of a float: exponent, 3 bits behind it
  constexpr int BASE = (127 + 9) << 3;  // 512's
  int len[N], key[N];
  bool some = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = first + i * 64 + lane;
    len[i] = context_of(p, min(s, seqs - 1));
    const int reads = p.window > 0 ? min(len[i], p.window) : len[i];
    some |= reads >= p.sorted;
    const int of = (__builtin_bit_cast(int, (float)max(reads, 1)) >> LOW) - BASE;
    key[i] = min(max(of, 0), (1 << BITS) - 1);
  }
  int at = r - first;
  if (__any(some)) {
    unsigned long long left[N];
#pragma unroll
    for (int i = 0; i < N; ++i) left[i] = __ballot(first + i * 64 + lane < seqs);
    int rank = at;
#pragma unroll
    for (int bit = BITS - 1; bit >= 0; --bit) {
      unsigned long long with[N];
      int n = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        with[i] = left[i] & __ballot(key[i] >> bit & 1);
        n += __popcll(with[i]);
      }
      const bool in = rank < n;
      rank -= in ? 0 : n;
#pragma unroll
      for (int i = 0; i < N; ++i) left[i] = in ? with[i] : left[i] & ~with[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int n = __popcll(left[i]);
      if (rank >= 0 && rank < n) {
        const int before = (int)__popcll(left[i] & ((1ull << lane) - 1));
        at = i * 64 + __ffsll(__ballot((left[i] >> lane & 1) && before == rank)) - 1;
      }
      rank -= n;
    }
  }
  at = __builtin_amdgcn_readfirstlane(at);
  int ctx = len[0];
#pragma unroll
  for (int i = 1; i < N; ++i) ctx = at >> 6 == i ? len[i] : ctx;
  return int2{first + at, __builtin_amdgcn_readlane(ctx, at & 63)};
}

// Rows of blocks that help sequences much longer than the rest of a batch: one for every
// 2^n pairs past the first 2^n, which are PART and twice the mean at least, given out
// in the order of the sequences for as long as there are any. Parts of a sequence lie at its
// helpers' rows, the first at p.help + its first helper's. Up to LAST sequences, and where
// the tables hold one that long: the launch that merges costs 3 us (us, without / with: 255
// of 500 and one of 32768 257 / 66, one of 8192 89 / 61, 99 and one of 32768 243 / 52, 31 and
// one 170 / 39; 256 of 500 in tables of 32768 48.0 / 50.8, 32 of 1500 19.8 / 22.6).
constexpr int HELP = 24;
struct Helpers {
  int first[LAST / 64], count[LAST / 64];  // of sequence 64 i + lane
  __device__ __forceinline__ Helpers(const ScaledDecode& p, int lane) {
    unsigned int pairs[LAST / 64], total = 0;
#pragma unroll
    for (int i = 0; i < LAST / 64; ++i) {
      const int s = i * 64 + lane;
      pairs[i] = page_range(context_of(p, min(s, p.seqs - 1)), p.window, 0, 1, 1).pairs;
      if (s >= p.seqs) pairs[i] = 0;
      total += pairs[i];
    }
    auto add = [](unsigned int a, unsigned int b) { return a + b; };
    auto last = [](unsigned int x) { return (unsigned int)__builtin_amdgcn_readlane(x, 63); };
    total = last(lanes_up_to(total, 0, add));
    const unsigned int cut = max((unsigned int)PART, 2 * (total / p.seqs));
    const int shift = 32 - __builtin_clz(cut - 1);
    unsigned int given = 0;
#pragma unroll
    for (int i = 0; i < LAST / 64; ++i) {
      const unsigned int n = pairs[i] > 0 ? min((pairs[i] - 1) >> shift, (unsigned int)HELP) : 0;
      const unsigned int up = lanes_up_to(n, 0, add);
      first[i] = given + up - n;
      count[i] = max(min((int)n, p.help - first[i]), 0);
      given += last(up);
    }
  }
  // the sequence for which `is` holds of its first helper and their number, or -1
  template <typename F>
  __device__ __forceinline__ int find(F is) const {
    int s = -1;
#pragma unroll
    for (int i = 0; i < LAST / 64; ++i) {
      const unsigned long long those = __ballot(is(first[i], count[i]));
      if (those) s = i * 64 + __ffsll(those) - 1;
    }
    return __builtin_amdgcn_readfirstlane(s);
  }
  // {first, count} of sequence s
  __device__ __forceinline__ int2 of(int s) const {
    int at = 0, n = 0;  // (each by itself: a choice among members would be in memory)
#pragma unroll
    for (int i = 0; i < LAST / 64; ++i) {
      const int a = __builtin_amdgcn_readlane(first[i], s & 63);
      const int b = __builtin_amdgcn_readlane(count[i], s & 63);
      at = s >> 6 == i ? a : at;
      n = s >> 6 == i ? b : n;
    }
    return int2{at, n};
  }
};

// 16-byte chunk that chunk c of staged row r is XORed with: the 16 rows of both pages
// that half a wave's transposing load brings lie in different banks
template <int D>
__device__ __forceinline__ int byte_swz(int r) {
  if constexpr (D == 128) return ((r >> 1) & 7) ^ (r >> 4 & 1) << 2;
  else return ((r >> 2) & 3) ^ (r >> 4 & 1) << 1;
}

// Adds to the first G columns of 16 the ones G and (PARTS 3) 2 G further on.
template <int G, int PARTS, int N>
__device__ __forceinline__ void add_parts(f32x4_t (&o)[N]) {
  auto from = [](float x, auto by) {  // the value `by` columns on
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x),
                                           0x120 + 16 - decltype(by)::value, 15, 15, true));
  };
#pragma unroll
  for (int b = 0; b < N; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = o[b][r];
      float sum = x + from(x, std::integral_constant<int, G>{});
      if constexpr (PARTS == 3) sum += from(x, std::integral_constant<int, 2 * G>{});
      o[b][r] = sum;
    }
}

// 16 bytes of K. With heads of 128 two loads take halves of the same lines, which have to
// stay in the cache between them; other lines pass once (us, K kept and V passing / both
// passing / both kept: 256 sequences of 2048 168 / 172 / 186, of 2048 +- 60% 186 / 195 / 203,
// 1536 of 560 286 / 312 / 312; with heads of 64, whose loads take whole lines, 64 of 601
// behind a window 7.4 / 7.1).
template <int D>
__device__ __forceinline__ uint4 load_k16(const char* from) {
  return D > 64 ? *reinterpret_cast<const uint4*>(from) : load16_nt(from);
}

constexpr int BATCH = 32;  // pairs whose page ids and scales a wave fetches at once

template <int D, int NW, bool WIDE>  // WIDE: groups of 6 to 8
__global__ __launch_bounds__(NW * 64, 4) void scaled_decode_kernel(const ScaledDecode p) {
  constexpr int KC = D / 32;       // contraction chunks of K Q^T
  constexpr int DB = D / 16;       // 16-column blocks of the output
  constexpr int ROWS = 2 * PAGE;   // keys of a pair
  constexpr int TILE = PAGE * D;   // bytes of a page of one head
  constexpr int NI = D / 64;       // wave-wide 16-byte loads of a page
  constexpr int LPR = D / 16;      // lanes per row of V as it is loaded
  constexpr int MERGE = 8 * (D + 4) + 16;  // floats: sums of 8 heads, their m and l
  constexpr int AREA = MERGE * 4 > 2 * TILE ? MERGE * 4 : 2 * TILE;

  const int kvh = blockIdx.x, row = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  int s = row - p.help, ctx = 0, split = blockIdx.z;
  if (s < 0) {
    const Helpers helpers(p, lane);
    s = helpers.find([&](int first, int n) { return first <= row && row < first + n; });
    if (s < 0) return;
    ctx = context_of(p, s);
  } else if (p.sorted) {
    const int2 of = longest_first(p, s, p.seqs, lane);
    s = of.x;
    ctx = of.y;
  } else {
    // (where few contexts have all splits, theirs are turned on to units of their own)
    if (p.n_splits > p.base) s = (s + 5 * split + split / 8) % p.seqs;
    ctx = context_of(p, s);
  }
  const int* bt = p.block_tables + (long)s * p.max_blocks;

  Range rg = decode_range(p, ctx, NW);
  long part_at = (long)s * p.H * p.n_splits + split, part_step = p.n_splits;  // by head
  if (p.help > 0) {
    const int2 helpers = Helpers(p, lane).of(s);
    if (helpers.y > 0) {
      split = row < p.help ? row - helpers.x + 1 : 0;
      rg.splits = 1 + helpers.y;
      rg.per = (rg.pairs + helpers.y) / rg.splits;
      part_at = (long)(split > 0 ? row : p.help + helpers.x) * p.H;
      part_step = 1;
    }
  }
  const int n_lo = split * rg.per + wave;
  const int n_hi = min((split + 1) * rg.per, rg.pairs);
  // waves with work, the first at least: the others end here and no barrier waits for them
  const int nw = min(max(n_hi - split * rg.per, 1), NW);
  if (split >= rg.splits || wave >= nw) return;
  const int col = lane & 15, g = lane >> 4;
  const int G = p.group;
  const int part = col / G;  // of the weights: high, middle, low
  const bool used = part < (WIDE ? 2 : 3);

  __shared__ __attribute__((aligned(16))) char lds[NW][AREA];

  // lane l of a batch from pair n on: page (l & 1) of pair n + l / 2 * NW
  int id = 0;
  unsigned int ks = 0, vs = 0;
  auto fetch = [&](int n) {
    id = bt[min(rg.first + 2 * (n + (lane >> 1) * NW) + (lane & 1), rg.last)];
    id = min(max(id, 0), p.s8.pages - 1);
    const long at = (long)id * p.Hkv + kvh;
    ks = p.s8.k[at];
    vs = p.s8.v[at];
  };
  uint4 kr[2][NI], vr[2][NI];
  const unsigned int klane = col * D + g * 16, vlane = lane * 16;
  auto tile = [&](const unsigned char* cache, int i, int h) {
    const int page = __builtin_amdgcn_readlane(id, (i % BATCH) * 2 + h);
    const char* at = reinterpret_cast<const char*>(cache) + ((long)page * p.Hkv + kvh) * TILE;
    // (kept apart from the lanes' 32-bit offsets: joined they are 64 bits of each lane)
    asm("" : "+s"(at));
    return at;
  };
  auto load_k = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* from = tile(p.k_cache, i, h);
#pragma unroll
      for (int j = 0; j < NI; ++j) kr[h][j] = load_k16<D>(from + klane + j * 64);
    }
  };
  auto load_v = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* from = tile(p.v_cache, i, h);
#pragma unroll
      for (int j = 0; j < NI; ++j) vr[h][j] = load16_nt(from + vlane + j * 1024);
    }
  };
  if (n_lo < n_hi) {
    fetch(n_lo);
    load_k(0);
    load_v(0);
  }

  bf16x8_t qf[KC];
  float c2 = p.scale * LOG2E;
  {
    const short flip = c2 < 0.f ? (short)0x8000 : (short)0;  // the scale's sign, exactly
    const short* qp = p.q + (long)s * p.sq + (long)(kvh * G + col % G) * D + g * 16;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      short8_t x = *reinterpret_cast<const short8_t*>(qp + (c >> 1) * 64 + (c & 1) * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = used ? (short)(x[j] ^ flip) : (short)0;
      qf[c] = __builtin_bit_cast(bf16x8_t, x);
    }
  }
  c2 = fabsf(c2);

  // Transposing load: lane i of 16 brings key i / 2, columns 8 (i % 2) .. + 7, and
  // receives column i of eight keys, four of each page.
  const int vrow = (col >> 3) * PAGE + g * 4 + ((col >> 1) & 3);
  unsigned int vaddr = vrow * D + byte_swz<D>(vrow) * 16 + (col & 1) * 8;
  // where a lane's bytes of V go: of the loads with odd h + j half a row of chunks off
  unsigned int to[2];
  to[0] = lane / LPR * D + ((lane % LPR) ^ byte_swz<D>(lane / LPR)) * 16;
  to[1] = to[0] ^ (D / 2);

  const int key_lo = ctx > 0 ? low_of(ctx - 1, p.window, 0) : 0;  // first visible key
  // Weights are 2^(score c2 - mc); mc follows the largest score once it is passed by 2^8
  constexpr float ROOM = 8.f;
  float mc = fmaxf(NO_MAX * c2, -3e38f), l = 0.f;
  f32x4_t o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b) o[b] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (int n = n_lo, i = 0; n < n_hi; n += NW, ++i) {
    float k2[2], v2[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      k2[h] = page_scale(__builtin_amdgcn_readlane(ks, (i % BATCH) * 2 + h));
      v2[h] = page_scale(__builtin_amdgcn_readlane(vs, (i % BATCH) * 2 + h));
    }
    const bool more = n + NW < n_hi;
    if (more && (i + 1) % BATCH == 0) fetch(n + NW);

    f32x4_t sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 x = kr[h][c >> 1];
        const uint2 half = c & 1 ? uint2{x.z, x.w} : uint2{x.x, x.y};
        sc[h] = mfma16x16x32(widen_fp8(half, k2[h]), qf[c], sc[h]);
      }
    }
    if (more) load_k(i + 1);
    const int key0 = (rg.first + 2 * n) * PAGE;
    const bool edge = key0 + ROWS > ctx || key0 < key_lo;
    if (edge) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = key0 + h * PAGE + g * 4 + r;
          sc[h][r] = key < ctx && key >= key_lo ? sc[h][r] : MASKED;
        }
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int key = key0 + h * PAGE + j * (64 / LPR) + lane / LPR;
          if (key >= ctx || key < key_lo) vr[h][j] = uint4{0, 0, 0, 0};
        }
      }
    }
    char* mine = lds[wave];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *reinterpret_cast<uint4*>(mine + to[(h + j) & 1] + (h * PAGE + j * (64 / LPR)) * D) =
            vr[h][j];
    if (more) load_v(i + 1);

    float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                     fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
    mx = column_max(mx) * c2;
    if (__any(mx > mc + ROOM)) {
      const float mn = fmaxf(mc, mx);
      const float f = __builtin_amdgcn_exp2f(mc - mn);
      mc = mn;
      l *= f;
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] *= f;
    }
    asm("" : "+v"(vaddr));  // (its eight forms are made here, not kept)
    bf16x8_t pf, pl;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[h][r], c2, -mc));
        l += w;
        const Split3 w3(w);
        if constexpr (WIDE) {
          pf[h * 4 + r] = part == 0 ? w3.hi : w3.mid;
          pl[h * 4 + r] = part == 0 ? w3.lo : (__bf16)0.f;
        } else {
          pf[h * 4 + r] = part == 0 ? w3.hi : part == 1 ? w3.mid : w3.lo;
        }
      }
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      typedef int i2_t __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) i2_t lds2_t;
      const char* a0 = mine + (vaddr ^ b * 16);
      const bf16x8_t a = widen_pages(
          __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds2_t*)a0)),
          v2[0], v2[1]);
      o[b] = mfma16x16x32(a, pf, o[b]);
      if constexpr (WIDE) o[b] = mfma16x16x32(a, pl, o[b]);
    }
  }

  // ---- merge: the parts of the weights, then the waves ----
  l = column_sum(l);
  float* mo = reinterpret_cast<float*>(lds[wave]);  // [8][D + 4], then m and l
  float* mm = mo + 8 * (D + 4);
  constexpr int PARTS = WIDE ? 2 : 3;
  if constexpr (WIDE) {
    if (G == 8) add_parts<8, PARTS>(o);
    else if (G == 7) add_parts<7, PARTS>(o);
    else add_parts<6, PARTS>(o);
  } else {
    if (G == 4) add_parts<4, PARTS>(o);
    else if (G == 1) add_parts<1, PARTS>(o);
    else if (G == 2) add_parts<2, PARTS>(o);
    else if (G == 3) add_parts<3, PARTS>(o);
    else add_parts<5, PARTS>(o);
  }
  if (col < G) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
      *reinterpret_cast<f32x4_t*>(mo + col * (D + 4) + b * 16 + g * 4) = o[b];
  }
  if (lane < G) {
    mm[lane] = mc;
    mm[8 + lane] = l;
  }
  __syncthreads();
  constexpr int WF = AREA / 4;  // floats between the waves' areas
  const float* all = reinterpret_cast<const float*>(lds);
  for (int i = threadIdx.x; i < G * (D / 4); i += nw * 64) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    float top = all[8 * (D + 4) + h];
#pragma unroll
    for (int w = 1; w < NW; ++w)
      if (w < nw) top = fmaxf(top, all[w * WF + 8 * (D + 4) + h]);
    float sum = 0.f;
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w >= nw) continue;
      const float* a = all + w * WF;
      const float f = __builtin_amdgcn_exp2f(a[8 * (D + 4) + h] - top);
      sum += f * a[8 * (D + 4) + 8 + h];
      acc += f * *reinterpret_cast<const f32x4_t*>(a + h * (D + 4) + d);
    }
    const int head = kvh * G + h;
    if (rg.splits == 1) {
      store4(p.out, ((long)s * p.H + head) * D + d, acc * (sum > 0.f ? 1.f / sum : 0.f), 0);
    } else {
      const long at = part_at + head * part_step;
      *reinterpret_cast<f32x4_t*>(p.part_out + at * D + d) = acc;
      if (d == 0) {
        p.part_ml[at * 2] = top;
        p.part_ml[at * 2 + 1] = sum;
      }
    }
  }
}

// Adds the splits of a (sequence, head), or of one with helpers: four waves take every
// fourth one, in order. Sequences that one split covers are done.
template <int D>
__global__ __launch_bounds__(256) void scaled_decode_reduce_kernel(const ScaledDecode p,
                                                                   const int waves) {
  constexpr int ACC = D / 64;
  const int h = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = blockIdx.y, splits;
  if (p.help > 0) {
    const Helpers helpers(p, lane);
    const int row = s;
    s = helpers.find([&](int first, int n) { return first == row && n > 0; });
    if (s < 0) return;
    splits = 1 + helpers.of(s).y;
  } else {
    splits = decode_range(p, context_of(p, s), waves).splits;
  }
  if (splits == 1) return;
  const long sh = (long)s * p.H + h;
  auto at = [&](int sp) {
    if (p.help == 0) return sh * p.n_splits + sp;
    return (long)(blockIdx.y + (sp > 0 ? sp - 1 : p.help)) * p.H + h;
  };
  float m = -3.4e38f;
  for (int sp = lane; sp < splits; sp += 64) m = fmaxf(m, p.part_ml[at(sp) * 2]);
  m = wave_reduce_max(m);
  float l = 0.f, acc[ACC];
#pragma unroll
  for (int a = 0; a < ACC; ++a) acc[a] = 0.f;
#pragma unroll 4
  for (int sp = wave; sp < splits; sp += 4) {
    const float w = __builtin_amdgcn_exp2f(p.part_ml[at(sp) * 2] - m);
    l += w * p.part_ml[at(sp) * 2 + 1];
    const float* po = p.part_out + at(sp) * D + lane * ACC;
#pragma unroll
    for (int a = 0; a < ACC; ++a) acc[a] += w * po[a];
  }
  __shared__ float sums[4][D + 1];
#pragma unroll
  for (int a = 0; a < ACC; ++a) sums[wave][lane * ACC + a] = acc[a];
  if (lane == 0) sums[wave][D] = l;
  __syncthreads();
  if (threadIdx.x >= D) return;
  const int d = threadIdx.x;
  const float all = sums[0][D] + sums[1][D] + sums[2][D] + sums[3][D];
  const float x = sums[0][d] + sums[1][d] + sums[2][d] + sums[3][d];
  reinterpret_cast<short*>(p.out)[sh * D + d] =
      float_to_bf16_bits(x * (all > 0.f ? 1.f / all : 0.f));
}

// Few queries per sequence behind their context (drafts under verification, short turns):
// decode's kernel with (query, head of the group) pairs of a sequence in 16 NB columns, each
// with a limit of its own; bytes are widened once for all of them. Block c Hkv + head takes
// the pairs from 16 NB c on. Weights are rounded to bf16, as in
// the chunk kernel (2^-9 of values that are summed and then rounded so themselves).
struct FewArgs {
  ScaledDecode d;      // out, q: [T, H, D]
  const int* cu_q;     // [S + 1]
  int tokens;          // T
  float* part_out;     // [n_splits, T, H, D]
  float* part_ml;      // [n_splits, T, H, 2]: exponent, sum of weights or NO_KEYS
};

template <int D, int NW, int NB>
__global__ __launch_bounds__(NW * 64, NB == 1 ? 3 : 2) void scaled_few_kernel(const FewArgs f) {
  constexpr int KC = D / 32, DB = D / 16, ROWS = 2 * PAGE, TILE = PAGE * D, NI = D / 64;
  constexpr int LPR = D / 16;
  constexpr int COLS = 16 * NB;
  constexpr int MERGE = COLS * (D + 4) + 2 * COLS;  // floats: the columns' sums, m and l
  constexpr int AREA = MERGE * 4 > 2 * TILE ? MERGE * 4 : 2 * TILE;
  const ScaledDecode& p = f.d;

  const int kvh = blockIdx.x % p.Hkv, first_col = blockIdx.x / p.Hkv * COLS;
  const int split = blockIdx.z;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int2 of = p.sorted ? longest_first(p, blockIdx.y, p.seqs, lane)
                           : int2{(int)blockIdx.y, context_of(p, blockIdx.y)};
  const int s = of.x, ctx = of.y;
  const int G = p.group;
  const int q_start = min(max(f.cu_q[s], 0), f.tokens);
  const int q_len = min(f.cu_q[s + 1], f.tokens) - q_start;
  const int cols = min(q_len * G - first_col, COLS);  // of the block
  if (cols <= 0) return;
  const int start = ctx - q_len;  // position of query 0
  auto low = [&](int pos) { return pos > 0 ? low_of(pos, p.window, 0) : 0; };
  // keys of the block's first and last query
  const int pos_lo = start + first_col / G, pos_hi = start + (first_col + cols - 1) / G;
  const int key_lo = low(pos_lo), low_hi = low(pos_hi);
  const int end = min(ctx, pos_hi + 1);  // keys
  const int first = key_lo / PAGE, last = (end - 1) / PAGE;
  const int pairs = end > 0 ? (last - first) / 2 + 1 : 0;
  const int splits = max(1, min(p.n_splits, (pairs + NW - 1) / NW));
  const int per = (pairs + splits - 1) / splits;
  const int n_lo = split * per + wave;
  const int n_hi = min((split + 1) * per, pairs);
  const long rows = (long)f.tokens * p.H;
  auto row_of = [&](int c) {  // (token, head) of the block's column c
    return (long)(q_start + (first_col + c) / G) * p.H + kvh * G + (first_col + c) % G;
  };
  if (split >= splits || pairs == 0) {
    for (int c = threadIdx.x; c < cols; c += NW * 64) {
      if (p.n_splits > 1) f.part_ml[(split * rows + row_of(c)) * 2 + 1] = NO_KEYS;
      else
        for (int d = 0; d < D; ++d) reinterpret_cast<short*>(p.out)[row_of(c) * D + d] = 0;
    }
    return;
  }
  const int nw = min(max(n_hi - split * per, 1), NW);
  if (wave >= nw) return;
  const int col = lane & 15, g = lane >> 4;

  __shared__ __attribute__((aligned(16))) char lds[NW][AREA];

  const int* bt = p.block_tables + (long)s * p.max_blocks;
  int id = 0;
  unsigned int ks = 0, vs = 0;
  auto fetch = [&](int n) {
    id = bt[min(first + 2 * (n + (lane >> 1) * NW) + (lane & 1), last)];
    id = min(max(id, 0), p.s8.pages - 1);
    const long at = (long)id * p.Hkv + kvh;
    ks = p.s8.k[at];
    vs = p.s8.v[at];
  };
  uint4 kr[2][NI], vr[2][NI];
  const unsigned int klane = col * D + g * 16, vlane = lane * 16;
  auto tile = [&](const unsigned char* cache, int i, int h) {
    const int page = __builtin_amdgcn_readlane(id, (i % BATCH) * 2 + h);
    const char* at = reinterpret_cast<const char*>(cache) + ((long)page * p.Hkv + kvh) * TILE;
    asm("" : "+s"(at));
    return at;
  };
  auto load_k = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* from = tile(p.k_cache, i, h);
#pragma unroll
      for (int j = 0; j < NI; ++j) kr[h][j] = load_k16<D>(from + klane + j * 64);
    }
  };
  auto load_v = [&](int i) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* from = tile(p.v_cache, i, h);
#pragma unroll
      for (int j = 0; j < NI; ++j)
        vr[h][j] = load16_nt(from + vlane + j * 1024);
    }
  };
  if (n_lo < n_hi) {
    fetch(n_lo);
    load_k(0);
    load_v(0);
  }

  bf16x8_t qf[NB][KC];
  int my_pos[NB];
  float c2 = p.scale * LOG2E;
  {
    const short flip = c2 < 0.f ? (short)0x8000 : (short)0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int c = first_col + min(b * 16 + col, cols - 1);
      my_pos[b] = start + c / G;
      const short* qp =
          p.q + (long)(q_start + c / G) * p.sq + (long)(kvh * G + c % G) * D + g * 16;
#pragma unroll
      for (int k = 0; k < KC; ++k) {
        short8_t x = *reinterpret_cast<const short8_t*>(qp + (k >> 1) * 64 + (k & 1) * 8);
        x ^= flip;
        qf[b][k] = __builtin_bit_cast(bf16x8_t, x);
      }
    }
  }
  c2 = fabsf(c2);

  const int vrow = (col >> 3) * PAGE + g * 4 + ((col >> 1) & 3);
  unsigned int vaddr = vrow * D + byte_swz<D>(vrow) * 16 + (col & 1) * 8;
  unsigned int to[2];
  to[0] = lane / LPR * D + ((lane % LPR) ^ byte_swz<D>(lane / LPR)) * 16;
  to[1] = to[0] ^ (D / 2);

  constexpr float ROOM = 8.f;
  float mc[NB], l[NB];
  f32x4_t o[NB][DB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    mc[b] = fmaxf(NO_MAX * c2, -3e38f);
    l[b] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[b][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  for (int n = n_lo, i = 0; n < n_hi; n += NW, ++i) {
    float k2[2], v2[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      k2[h] = page_scale(__builtin_amdgcn_readlane(ks, (i % BATCH) * 2 + h));
      v2[h] = page_scale(__builtin_amdgcn_readlane(vs, (i % BATCH) * 2 + h));
    }
    const bool more = n + NW < n_hi;
    if (more && (i + 1) % BATCH == 0) fetch(n + NW);

    f32x4_t sc[NB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int b = 0; b < NB; ++b) sc[b][h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint4 x = kr[h][c >> 1];
        const uint2 half = c & 1 ? uint2{x.z, x.w} : uint2{x.x, x.y};
        const bf16x8_t a = widen_fp8(half, k2[h]);
#pragma unroll
        for (int b = 0; b < NB; ++b) sc[b][h] = mfma16x16x32(a, qf[b][c], sc[b][h]);
      }
    }
    if (more) load_k(i + 1);
    const int key0 = (first + 2 * n) * PAGE;
    if (key0 + ROWS - 1 > pos_lo || key0 < low_hi) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = key0 + h * PAGE + g * 4 + r;
#pragma unroll
          for (int b = 0; b < NB; ++b)
            sc[b][h][r] = key < ctx && key <= my_pos[b] && key >= low(my_pos[b]) ? sc[b][h][r]
                                                                              : MASKED;
        }
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int key = key0 + h * PAGE + j * (64 / LPR) + lane / LPR;
          if (key >= ctx || key < key_lo) vr[h][j] = uint4{0, 0, 0, 0};
        }
      }
    }
    char* mine = lds[wave];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *reinterpret_cast<uint4*>(mine + to[(h + j) & 1] + (h * PAGE + j * (64 / LPR)) * D) =
            vr[h][j];
    if (more) load_v(i + 1);

    bf16x8_t pf[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float mx = fmaxf(fmaxf(fmaxf(sc[b][0][0], sc[b][0][1]), fmaxf(sc[b][0][2], sc[b][0][3])),
                       fmaxf(fmaxf(sc[b][1][0], sc[b][1][1]), fmaxf(sc[b][1][2], sc[b][1][3])));
      mx = column_max(mx) * c2;
      if (__any(mx > mc[b] + ROOM)) {
        const float mn = fmaxf(mc[b], mx);
        const float r = __builtin_amdgcn_exp2f(mc[b] - mn);
        mc[b] = mn;
        l[b] *= r;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[b][d] *= r;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][h][r], c2, -mc[b]));
          l[b] += w;
          pf[b][h * 4 + r] = (__bf16)w;
        }
    }
    asm("" : "+v"(vaddr));
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      typedef int i2_t __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) i2_t lds2_t;
      const char* a0 = mine + (vaddr ^ d * 16);
      const bf16x8_t a = widen_pages(
          __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds2_t*)a0)),
          v2[0], v2[1]);
#pragma unroll
      for (int b = 0; b < NB; ++b) o[b][d] = mfma16x16x32(a, pf[b], o[b][d]);
    }
  }

  float* mo = reinterpret_cast<float*>(lds[wave]);  // [COLS][D + 4], then m and l
  float* mm = mo + COLS * (D + 4);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float sum = column_sum(l[b]);
#pragma unroll
    for (int d = 0; d < DB; ++d)
      *reinterpret_cast<f32x4_t*>(mo + (b * 16 + col) * (D + 4) + d * 16 + g * 4) = o[b][d];
    if (lane < 16) {
      mm[b * 16 + col] = mc[b];
      mm[COLS + b * 16 + col] = sum;
    }
  }
  __syncthreads();
  constexpr int WF = AREA / 4;
  const float* all = reinterpret_cast<const float*>(lds);
  for (int i = threadIdx.x; i < cols * (D / 4); i += nw * 64) {
    const int c = i / (D / 4), d = i % (D / 4) * 4;
    float top = all[COLS * (D + 4) + c];
    for (int w = 1; w < nw; ++w) top = fmaxf(top, all[w * WF + COLS * (D + 4) + c]);
    float sum = 0.f;
    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < nw; ++w) {
      const float* a = all + w * WF;
      const float r = __builtin_amdgcn_exp2f(a[COLS * (D + 4) + c] - top);
      sum += r * a[COLS * (D + 4) + COLS + c];
      acc += r * *reinterpret_cast<const f32x4_t*>(a + c * (D + 4) + d);
    }
    if (p.n_splits == 1) {
      store4(p.out, row_of(c) * D + d, acc * (sum > 0.f ? 1.f / sum : 0.f), 0);
    } else {
      const long at = split * rows + row_of(c);
      *reinterpret_cast<f32x4_t*>(f.part_out + at * D + d) = acc;
      if (d == 0) *reinterpret_cast<float2_t*>(f.part_ml + at * 2) = float2_t{top, sum};
    }
  }
}

// Waves that share a context, 4 or 8, and its splits (us; 8 KV heads of 128).
//
// From TWO_BLOCKS blocks on, two to a compute unit, four waves and no splits (4 x 1 / 8 x 1 /
// 4 waves x 2 splits: 64 sequences of 600 +- 50% 18.5 / 19.7 / 23.6, 96 of 3000 +- 60% 95 /
// 95 / 108, 256 of 100 17.8 / 21.6 / 21.5, of 2048 +- 60% 172 / 172 / 205, 1000 of 16 21.8 / 34.8:
// waves without a pair end at once, but their block's LDS keeps others out); from UNIT_BLOCKS
// on eight (32 of 1500 +- 60% 24.6 / 21.5 / 27.1). Below, splits make up that many blocks (1
// of 131071 under groups of eight 83 / 53 / 53 with 16, 32 and 64, of 7000 18.0 / 15.0 / 16.0
// with 8, 16 and 32), unless eight waves take a table in SHORT pairs each, which spares the
// launch that merges (eight waves / splits: 1 of 1500 13.7 / 9.3, 8 of 1500 13.9 / 10.7, 20
// of 1000 12.0 / 15.1; 1 of 560 9.1 / 9.0 in a graph and 8.3 / 10.9 call by call). In wider
// tables it is a window that is short: in SHORT pairs from WINDOW_BLOCKS on, in half as many
// below, where a captured launch that merges costs less than the pairs (eight waves / splits
// in a graph, and call by call: 1 behind 255 7.2 / 7.7, 7.2 / 11.1, 8 behind 384 8.3 / 8.1, 8.3
// / 10.8, behind 1000 10.8 / 9.1, 10.7 / 10.9, 12 behind 1000 11.0 / 12.3, 16 behind 255 7.4 /
// 9.2, 20 behind 1000 11.5 / 14.6).
//
// Long contexts among short ones: without splits there are helpers; with them, up to
// WIDE_SPLITS for the contexts that have PART pairs for each (us, without / with: one of
// 32768 and 15 of 500 125 / 42, 23 170 / 38 with helpers, 7 67 / 40; 16 of 2048 in wide
// tables 18.0 / 18.2).
struct Shape {
  int waves, base, splits, help;
};
constexpr long UNIT_BLOCKS = 256, TWO_BLOCKS = 512, SHORT = 4, WINDOW_BLOCKS = 96;
constexpr long HELP_READS = 8192, WIDE_SPLITS = 16;

// From which length of a sequence on a launch takes the longest first: blocks that all
// begin at once are left in order, and tables that hold no such sequence.
constexpr int LONG = 512, FEW_LONG = 1536;
int sorted_from(int length, long blocks, int splits, int max_blocks, int window) {
  const long reads = (long)max_blocks * PAGE;
  const bool any = (window > 0 && window < reads ? window : reads) >= length;
  return splits == 1 && blocks >= TWO_BLOCKS && any ? length : 0;
}
Shape decode_shape(long seqs, long kv_heads, long max_blocks, int window) {
  const long blocks = seqs * kv_heads;
  const long reads = window > 0 && window < max_blocks * PAGE ? window : max_blocks * PAGE;
  const int help = seqs > 0 && seqs <= LAST && reads >= HELP_READS ? HELP : 0;
  if (blocks <= 0 || blocks >= TWO_BLOCKS) return {4, 1, 1, help};
  // pages that a query sees: of a window's first and last key, and between them
  const long seen = window > 0 ? (window + PAGE - 2L) / PAGE + 1 : max_blocks;
  const long pairs = ((seen < max_blocks ? seen : max_blocks) + 1) / 2;
  long splits = (UNIT_BLOCKS + blocks / 2) / blocks;
  if (splits <= 1) return {8, 1, 1, help};
  const bool narrow = max_blocks <= 2 * 8 * SHORT;
  if (narrow || pairs <= 8 * (blocks >= WINDOW_BLOCKS ? SHORT : SHORT / 2)) return {8, 1, 1, 0};
  const long most = (pairs + 3) / 4;  // a pair for every wave
  splits = splits < most ? splits : most;
  const long whole = reads / (2 * PAGE) / PART;
  const long parts = whole < WIDE_SPLITS ? whole : WIDE_SPLITS;
  return {4, (int)splits, (int)(splits < parts ? parts : splits), 0};
}

template <int D, int NW>
void launch_waves(const ScaledDecode& p, dim3 grid, hipStream_t stream) {
  if (3 * p.group <= 16)
    hipLaunchKernelGGL((scaled_decode_kernel<D, NW, false>), grid, dim3(NW * 64), 0, stream, p);
  else
    hipLaunchKernelGGL((scaled_decode_kernel<D, NW, true>), grid, dim3(NW * 64), 0, stream, p);
}

template <int D>
hipError_t launch_scaled(const ScaledDecode& p, int seqs, int waves, hipStream_t stream) {
  const dim3 grid(p.Hkv, p.help + seqs, p.n_splits);
  if (waves == 8) launch_waves<D, 8>(p, grid, stream);
  else launch_waves<D, 4>(p, grid, stream);
  HIP_CHECK_KERNEL();
  if (p.n_splits > 1 || p.help > 0) {
    hipLaunchKernelGGL((scaled_decode_reduce_kernel<D>),
                       dim3(p.H, p.help > 0 ? p.help : seqs), dim3(256), 0, stream, p, waves);
    HIP_CHECK_KERNEL();
  }
  return hipSuccess;
}

}  // namespace

// waves | splits << 8 | rows of helpers << 24 for such a call
extern "C" int ks_scaled_decode_shape(int num_seqs, int num_kv_heads, int max_blocks,
                                      int window) {
  const Shape s = decode_shape(num_seqs, num_kv_heads, max_blocks, window);
  return s.waves | s.splits << 8 | s.help << 24;
}

// part_out [S, H, splits, D] and part_ml [S, H, splits, 2] where the shape has several
// splits, [2 rows, H, D] and [2 rows, H, 2] where it has helpers
extern "C" hipError_t ks_paged_attention_decode_scaled(
    void* out, const void* q, const void* k_cache, const void* v_cache,
    const void* k_scale, const void* v_scale, const void* block_tables,
    const void* context_lens, float scale, int num_seqs, int num_heads, int num_kv_heads,
    int head_dim, int max_blocks, int pages, long q_row_stride, int shape,
    void* part_out, void* part_ml, int window, hipStream_t stream) {
  if (num_kv_heads < 1 || num_heads % num_kv_heads != 0 || pages < 1)
    return hipErrorInvalidValue;
  const int group = num_heads / num_kv_heads;
  const int waves = shape & 255;
  const bool parts = part_out && part_ml;
  const int base = decode_shape(num_seqs, num_kv_heads, max_blocks, window).base;
  const int splits = parts ? shape >> 8 & 0xffff : 1, help = parts ? shape >> 24 : 0;
  if (group < 1 || group > 8 || splits < 1 || (help > 0 && splits > 1) ||
      (help > 0 && num_seqs > LAST) || (waves != 4 && waves != 8))
    return hipErrorInvalidValue;
  if (num_seqs == 0) return hipSuccess;
  const ScaledDecode p{out,
                       (const short*)q,
                       (const unsigned char*)k_cache,
                       (const unsigned char*)v_cache,
                       Scales{(const unsigned char*)k_scale, (const unsigned char*)v_scale,
                              pages},
                       (const int*)block_tables,
                       (const int*)context_lens,
                       score_scale(scale),
                       num_heads,
                       num_kv_heads,
                       group,
                       max_blocks,
                       q_row_stride,
                       splits,
                       base < splits ? base : splits,
                       (float*)part_out,
                       (float*)part_ml,
                       window,
                       sorted_from(LONG, (long)num_seqs * num_kv_heads, splits, max_blocks,
                                   window),
                       num_seqs,
                       help};
  if (head_dim == 128) return launch_scaled<128>(p, num_seqs, waves, stream);
  if (head_dim == 64) return launch_scaled<64>(p, num_seqs, waves, stream);
  return hipErrorInvalidValue;
}

// (query, head of a group) pairs of a sequence that the kernel for few queries takes, 32 to a
// block. A chunk kernel's wave takes 32 queries of one head whatever there are, four such
// waves a group's (32 / 8 heads of 128, us, chunk / few: 96 sequences of 2 queries after 1500
// 110 / 53, of 5 115 / 66, of up to 10 116 / 94; 32 of 5 after 400 18.8 / 12.3; 4 of 5 after
// 12900 53 / 33, of up to 10 54 / 46). At 64 pairs they are level (96 of 16 after 1500 120 /
// 118, 4 of 16 after 12900 61 / 66), and beyond the chunk kernel is ahead (4 of 32 74 / 99).
constexpr int FEW_COLUMNS = 64;

// Column blocks of a launch over few queries (0: the chunk kernel's)
extern "C" int ks_scaled_few_columns(int max_q_len, int group) {
  const long cols = (long)max_q_len * group;
  return cols < 1 ? 0 : cols <= 16 ? 1 : cols <= FEW_COLUMNS ? 2 : 0;
}

// part_out [splits, T, H, D] and part_ml [splits, T, H, 2]: left to be merged
extern "C" hipError_t ks_scaled_few(
    void* out, const void* q, const void* k_cache, const void* v_cache,
    const void* k_scale, const void* v_scale, const void* block_tables,
    const void* ctx_lens, const void* cu_q, int num_seqs, int max_q_len, int Hq, int Hkv,
    int head_dim, int max_nb, int pages, float scale, long sq, int window, long rows,
    int n_splits, void* part_out, void* part_ml, hipStream_t stream) {
  const int nb = Hkv > 0 ? ks_scaled_few_columns(max_q_len, Hq / Hkv) : 0;
  if (nb == 0) return hipErrorInvalidValue;
  if (num_seqs == 0) return hipSuccess;
  const int groups = (max_q_len * (Hq / Hkv) + 16 * nb - 1) / (16 * nb);
  const ScaledDecode d{out,
                       (const short*)q,
                       (const unsigned char*)k_cache,
                       (const unsigned char*)v_cache,
                       Scales{(const unsigned char*)k_scale, (const unsigned char*)v_scale,
                              pages},
                       (const int*)block_tables,
                       (const int*)ctx_lens,
                       score_scale(scale),
                       Hq,
                       Hkv,
                       Hq / Hkv,
                       max_nb,
                       sq,
                       n_splits,
                       n_splits,
                       nullptr,
                       nullptr,
                       window,
                       sorted_from(FEW_LONG, (long)num_seqs * Hkv * groups, n_splits, max_nb,
                                   window),
                       num_seqs,
                       0};
  const FewArgs f{d, (const int*)cu_q, (int)(rows / Hq), (float*)part_out, (float*)part_ml};
  const dim3 grid(Hkv * groups, num_seqs, n_splits);
#define GO(DD, BB) \
  hipLaunchKernelGGL((scaled_few_kernel<DD, 4, BB>), grid, dim3(256), 0, stream, f)
  if (head_dim == 128) {
    if (nb == 1) GO(128, 1);
    else GO(128, 2);
  } else if (head_dim == 64) {
    if (nb == 1) GO(64, 1);
    else GO(64, 2);
  } else {
    return hipErrorInvalidValue;
  }
#undef GO
  HIP_CHECK_KERNEL();
  return hipSuccess;
}

// key parts of such a launch
extern "C" int ks_scaled_few_splits(int num_seqs, int max_q_len, int Hq, int Hkv, int max_nb) {
  const int groups = (int)(((long)max_q_len * (Hq / Hkv) + 31) / 32);
  const long blocks = (long)num_seqs * Hkv * groups, pairs = (max_nb + 1) / 2;
  // (as for decode: a launch that merges costs what eight pairs of a wave take)
  if (blocks <= 0 || blocks >= UNIT_BLOCKS || pairs <= 4 * 8) return 1;
  long splits = (UNIT_BLOCKS + blocks / 2) / blocks;
  const long most = (pairs + 7) / 8;  // two pairs for every wave
  if (splits > most) splits = most;
  return splits < 1 ? 1 : (int)splits;
}
