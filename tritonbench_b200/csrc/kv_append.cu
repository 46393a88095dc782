// Appending to a paged e4m3 cache, with the position rotation on the way: q and k are rotated at their sequence
// positions, q is written back in its own type, k and v are quantised and stored into the pages of their sequence.
//
//   cache page p, kv head h:  codes [page_size][dim] e4m3, one fp32 scale;  value = code * scale[p][h]
//   scale = the smallest power of two (>= 2^-126) with max |x| / scale <= 448 over the page's tokens of that head
//   code  = e4m3(x * (1 / scale)), to nearest even
//
// The scale is a power of two because a page fills over many calls: when a later token needs a larger one, the codes
// that are already there are multiplied by old / new, which is exact but for what falls below the format's smallest
// subnormal.  It costs nothing in precision - e4m3 is a floating format, a power of two only moves its range by less
// than one binade of its 15 - whereas an arbitrary scale would round the old codes anew each time it grows.
// Infinities and NaN do not enter the scale (one bad value would take the page's other tokens with it) and are stored
// as NaN.
//
// Bound by HBM for prompts (q in, q out, k and v in at 2 bytes, out at 1), by latency for single tokens.  One launch
// does it all.  Some blocks own pages: each group of threads has one (page, kv head, k or v), so that nothing but that
// group reads or writes the page's scale: no atomics and the same result every time.  The other blocks rotate q.  A
// group is a warp when few rows come to a page or it is small, else a block; its rows stay in registers between the
// maximum and the codes.
#include <cuda_fp8.h>

#include <type_traits>

#include "kernels.h"
#include "rotary.cuh"
#include "sequences.cuh"

namespace b200fp8 {
namespace {

constexpr int kThreads = 256;
constexpr int kN = 8;  // elements of a 16-byte vector of bf16 or fp16; a slot is two of them

__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.0f;  // false for NaN
}

__device__ __forceinline__ float pow2_scale(float amax) {
  // amax = m 2^(E - 127), m in [1, 2); 448 = 1.75 * 2^8
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);  // biased exponent 1: 2^-126
}

__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float nan_for_inf(float v) { return fabsf(v) <= 3.402823466e38f ? v : __int_as_float(0x7fffffff); }

__device__ __forceinline__ uint2 codes8(const float (&y)[kN], float inv, bool infinite) {
  float z[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) z[i] = y[i] * inv;
  if (infinite) {  // the conversion would saturate it; a NaN stays one by itself
#pragma unroll
    for (int i = 0; i < kN; ++i) z[i] = nan_for_inf(z[i]);
  }
  return make_uint2(codes2(z[0], z[1]) | (codes2(z[2], z[3]) << 16), codes2(z[4], z[5]) | (codes2(z[6], z[7]) << 16));
}

__device__ __forceinline__ uint32_t rescaled4(uint32_t w, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 h(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * i)), __NV_E4M3));
    const float2 f = __half22float2(h);
    out |= codes2(f.x * ratio, f.y * ratio) << (16 * i);
  }
  return out;
}

// Slot s of a head, at row x: vectors a and b at these elements.
struct SlotAt {
  int a, b;
  bool turns;
};
template <bool kInterleaved>
__device__ __forceinline__ SlotAt slot_at(int slot, int rot) {
  if (slot < rot / (2 * kN)) {
    if (kInterleaved) return {slot * 2 * kN, slot * 2 * kN + kN, true};
    return {slot * kN, rot / 2 + slot * kN, true};
  }
  return {slot * 2 * kN, slot * 2 * kN + kN, false};  // rot is a multiple of a slot
}

__device__ __forceinline__ void table_row(const KvAppendParams& p, long long pos, int slot, float (&c)[kN], float (&s)[kN]) {
  if (pos < p.max_pos) {
    const float* row = p.table + pos * p.rot + slot * kN;
    load_table<kN>(row, c);
    load_table<kN>(row + p.rot / 2, s);
  } else {  // the table ends before this position
#pragma unroll
    for (int i = 0; i < kN; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
  }
}

template <bool kInterleaved>
__device__ __forceinline__ void turn(const KvAppendParams& p, long long pos, int slot, float (&a)[kN], float (&b)[kN]) {
  float c[kN], s[kN];
  table_row(p, pos, slot, c, s);
  rotate_slot<kN, kInterleaved>(a, b, c, s);
}

// One page, one kv head, k or v: the rows that come to it.
struct PageRows {
  int which, head, page, held, rows;
  long long from, token0;  // position and token of the first row
};

// false: no row comes to this one
__device__ __forceinline__ bool find_rows(const KvAppendParams& p, long long work, PageRows& w) {
  w.which = static_cast<int>(work & 1);
  const long long rest = work >> 1;
  w.head = static_cast<int>(rest % p.kv_heads);
  const long long slot_no = rest / p.kv_heads;
  // slot_no -> sequence and page: sequence b owns the slots from cu[b] / page_size + 2 b on, at least as many as the
  // pages that its tokens can touch
  int b;
  long long first_token, count, page_no;
  if (p.cu_seqlens == nullptr) {
    b = static_cast<int>(slot_no);
    first_token = b;
    count = 1;
    page_no = 0;
  } else {
    const auto first_slot = [&](int i) { return static_cast<long long>(max(p.cu_seqlens[i], 0) >> p.page_shift) + 2ll * i; };
    b = search_sequence(p.batch, slot_no, first_slot);
    first_token = p.cu_seqlens[b];
    count = p.cu_seqlens[b + 1] - first_token;
    page_no = slot_no - first_slot(b);
  }
  const long long end = p.seq_lens[b];          // positions [begin, end) of the sequence are new
  const long long begin = end - count;          // negative: more tokens than the sequence has; those are left out
  if (count <= 0 || page_no < 0) return false;
  page_no += (begin > 0 ? begin : 0) >> p.page_shift;
  if (page_no >= p.table_width) return false;
  const long long lo = page_no << p.page_shift;
  w.from = lo > begin ? lo : begin;
  const long long to = lo + p.page_size < end ? lo + p.page_size : end;
  if (w.from >= to) return false;
  w.token0 = first_token + (w.from - begin);
  w.rows = static_cast<int>(to - w.from);
  if (w.token0 < 0 || w.token0 + w.rows > p.tokens) return false;  // lengths that do not belong to this q, k, v
  w.held = static_cast<int>(w.from - lo);
  w.page = p.block_table[b * p.bt_stride + page_no];  // on its way while the rows are read
  return true;
}

// kGroup threads: a warp or the block
template <typename T, bool kInterleaved, int kGroup, int kHold>
__device__ __forceinline__ void append_rows(const KvAppendParams& p, const PageRows& w) {
  const int in_group = static_cast<int>(threadIdx.x) % kGroup;
  const int which = w.which, head = w.head, page = w.page, held = w.held, rows = w.rows;
  const long long from = w.from, token0 = w.token0;
  const T* x = which ? static_cast<const T*>(p.v) + token0 * p.v_token + head * p.v_head
                     : static_cast<const T*>(p.k) + token0 * p.k_token + head * p.k_head;
  const long long x_token = which ? p.v_token : p.k_token;
  const int rot = which ? 0 : p.rot;
  const int slots = p.dim / (2 * kN);
  const int items = rows * slots;

  // the first kHold slots of a thread stay in registers, rotated; what is beyond them is read and rotated twice
  const auto load = [&](int item, float (&a)[kN], float (&c)[kN]) {
    const int row = item / slots, slot = item - row * slots;
    const SlotAt at = slot_at<kInterleaved>(slot, rot);
    const T* r = x + row * x_token;
    const uint4 ra = *reinterpret_cast<const uint4*>(r + at.a);
    const uint4 rb = *reinterpret_cast<const uint4*>(r + at.b);
    unpack16<T>(ra, a);
    unpack16<T>(rb, c);
    if (at.turns) turn<kInterleaved>(p, from + row, slot, a, c);
  };
  uint8_t* codes = nullptr;
  const long long code_row = p.cache_row[which];
  bool infinite = false;  // among the group's values
  const auto store = [&](int item, const float (&a)[kN], const float (&c)[kN], float inv) {
    const int row = item / slots;
    const SlotAt at = slot_at<kInterleaved>(item - row * slots, rot);
    uint8_t* r = codes + (held + row) * code_row;
    *reinterpret_cast<uint2*>(r + at.a) = codes8(a, inv, infinite);
    *reinterpret_cast<uint2*>(r + at.b) = codes8(c, inv, infinite);
  };

  float ka[kHold][kN], kb[kHold][kN];
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    if (in_group + i * kGroup < items) load(in_group + i * kGroup, ka[i], kb[i]);
  }
  if (page < 0 || page >= p.num_pages) return;
  codes = (which ? p.v_cache : p.k_cache) + page * p.cache_page[which] + head * p.cache_head[which];
  float* const scale_at = (which ? p.v_scale : p.k_scale) + page * p.scale_page[which] + head * p.scale_head[which];
  const float old_scale = held > 0 ? *scale_at : 0.0f;
  // largest magnitude; fmaxf passes over NaN, an infinity is looked for only when there is one
  const auto largest = [&](auto finite_only) {
    const auto take = [&](float v) { return finite_only.value ? finite_abs(v) : fabsf(v); };
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      if (in_group + i * kGroup < items) {
#pragma unroll
        for (int e = 0; e < kN; ++e) amax = fmaxf(amax, fmaxf(take(ka[i][e]), take(kb[i][e])));
      }
    }
    for (int item = in_group + kHold * kGroup; item < items; item += kGroup) {
      float a[kN], c[kN];
      load(item, a, c);
#pragma unroll
      for (int e = 0; e < kN; ++e) amax = fmaxf(amax, fmaxf(take(a[e]), take(c[e])));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if constexpr (kGroup > 32) {
      __shared__ float red[kThreads / 32];
      __syncthreads();  // red of a first pass has been read
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
      __syncthreads();
      amax = red[0];
#pragma unroll
      for (int w = 1; w < kGroup / 32; ++w) amax = fmaxf(amax, red[w]);
    } else {
      __syncwarp();  // every lane has read the old scale before lane 0 writes the new one
    }
    return amax;
  };
  float amax = largest(std::false_type{});
  infinite = !(amax <= 3.402823466e38f);  // the same for the whole group
  if (infinite) amax = largest(std::true_type{});
  const float need = pow2_scale(amax);
  const float scale = fmaxf(old_scale, need);
  const float inv = __fdiv_rn(1.0f, scale);
  if (held > 0 && scale > old_scale) {  // the tokens that are already there move to the larger scale
    const float ratio = __fdiv_rn(old_scale, scale);
    const int vecs = p.dim / 16;
    for (int i = in_group; i < held * vecs; i += kGroup) {
      const int row = i / vecs;
      uint4* at = reinterpret_cast<uint4*>(codes + row * code_row) + (i - row * vecs);
      uint4 w = *at;
      w.x = rescaled4(w.x, ratio);
      w.y = rescaled4(w.y, ratio);
      w.z = rescaled4(w.z, ratio);
      w.w = rescaled4(w.w, ratio);
      *at = w;
    }
  }
  if (in_group == 0) *scale_at = scale;
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    if (in_group + i * kGroup < items) store(in_group + i * kGroup, ka[i], kb[i], inv);
  }
  for (int item = in_group + kHold * kGroup; item < items; item += kGroup) {
    float a[kN], c[kN];
    load(item, a, c);
    store(item, a, c, inv);
  }
}

// q: a thread has one slot of kHeads neighbouring heads of a token, as in rotary.cu; the positions of the block's tokens
// are looked up once, in shared memory, while q is on its way.
constexpr int kMaxTokens = kThreads / 4 + 1;  // a head has at least four slots

template <typename T, bool kInterleaved, int kHeads>
__device__ __forceinline__ void rotate_q(const KvAppendParams& p, long long block) {
  __shared__ long long positions[kMaxTokens];
  const int slots = p.dim / (2 * kN);
  const unsigned per_token = static_cast<unsigned>((p.heads + kHeads - 1) / kHeads) * static_cast<unsigned>(slots);
  const long long first = block * kThreads;
  const long long items = static_cast<long long>(p.tokens) * per_token;
  const long long token0 = items <= 0xffffffffll ? static_cast<unsigned>(first) / per_token : first / per_token;
  const unsigned at = static_cast<unsigned>(first - token0 * per_token) + threadIdx.x;
  const int local = static_cast<int>(at / per_token);
  const unsigned in_token = at - local * per_token;
  const int group = static_cast<int>(in_token / static_cast<unsigned>(slots));
  const int slot = static_cast<int>(in_token - group * static_cast<unsigned>(slots));
  const int head0 = group * kHeads;
  const bool live = first + threadIdx.x < items;
  const SlotAt e = slot_at<kInterleaved>(slot, p.rot);
  uint4 ra[kHeads], rb[kHeads];
  if (live) {
    const T* x = static_cast<const T*>(p.q) + (token0 + local) * p.q_token + head0 * p.q_head;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (head0 + h < p.heads) {
        ra[h] = *reinterpret_cast<const uint4*>(x + h * p.q_head + e.a);
        rb[h] = *reinterpret_cast<const uint4*>(x + h * p.q_head + e.b);
      }
    }
  }
  // all warps look up the block's tokens, one token a warp at a time
  const long long last = min(static_cast<long long>(p.tokens) - 1, token0 + (static_cast<unsigned>(first - token0 * per_token) + kThreads - 1) / per_token);
  for (int i = threadIdx.x >> 5; i <= last - token0; i += kThreads / 32) {
    const long long t = token0 + i;
    long long pos;
    if (p.cu_seqlens == nullptr) {
      pos = max(p.seq_lens[t] - 1ll, -1ll);
    } else if (t < p.cu_seqlens[0] || t >= p.cu_seqlens[p.batch]) {
      pos = -2;  // no sequence's
    } else {
      const int b = search_sequence(p.batch, t, [&](int s) { return static_cast<long long>(p.cu_seqlens[s]); });
      pos = p.seq_lens[b] - static_cast<long long>(p.cu_seqlens[b + 1]) + t;
      if (pos < 0) pos = -1;
    }
    if ((threadIdx.x & 31) == 0) positions[i] = pos;
  }
  __syncthreads();
  if (!live) return;
  const long long pos = positions[local];
  if (pos == -2 && !p.fill_rest) return;
  T* y = static_cast<T*>(p.q_out) + (token0 + local) * p.qo_token + head0 * p.qo_head;
  float c[kN], s[kN];
  if (e.turns && pos >= 0) table_row(p, pos, slot, c, s);
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (head0 + h < p.heads) {
      if (pos < 0) {  // not a token of any sequence
        ra[h] = rb[h] = make_uint4(0u, 0u, 0u, 0u);
      } else if (e.turns) {
        float a[kN], b[kN];
        unpack16<T>(ra[h], a);
        unpack16<T>(rb[h], b);
        rotate_slot<kN, kInterleaved>(a, b, c, s);
        ra[h] = pack16<T>(a);
        rb[h] = pack16<T>(b);
      }
      *reinterpret_cast<uint4*>(y + h * p.qo_head + e.a) = ra[h];
      *reinterpret_cast<uint4*>(y + h * p.qo_head + e.b) = rb[h];
    }
  }
}

// Who appends: a warp a page, a block a page, or a warp each for pages that get a few rows and the block for the others.
enum { kWarps, kBlock, kEither };
// Rows x slots up to which a warp does a page by itself in kEither: 16 rows of 128 (64 sequences x 12 tokens 10.7 us, with a
// limit of 64 22.6; 63 x 1 and one of 400 the same with 32 to 192).
constexpr int kWarpItems = 128;

template <typename T, bool kInterleaved, int kWho, int kHold, int kHeads>
__global__ void __launch_bounds__(kThreads, 4) kv_append_kernel(const KvAppendParams p, long long works, unsigned page_blocks,
                                                                unsigned mix) {
  // Blocks that own pages are spread evenly among those that rotate q: the former wait for one load after another, the
  // latter for bandwidth, so they fill each other's gaps (17438 tokens: 132 us with the page blocks first, 115 us mixed).
  // With a token a sequence the pages take longest and go first (mix 0; 250 sequences: 6.3 us, mixed 7.2).  Four blocks an
  // SM (64 registers, a few spilled in the page part) hide more of the waiting than three.
  // mix is page_blocks / blocks in 32 fraction bits, rounded up: i * mix passes each whole number below page_blocks once.
  const unsigned i = blockIdx.x;
  const unsigned before = mix ? __umulhi(i, mix) : min(i, page_blocks);  // page blocks in front of this one
  if (mix ? __umulhi(i + 1, mix) > before : i < page_blocks) {
    PageRows w;
    if constexpr (kWho == kBlock) {
      if (find_rows(p, before, w)) append_rows<T, kInterleaved, kThreads, kHold>(p, w);
    } else if constexpr (kWho == kWarps) {
      const long long work = static_cast<long long>(before) * (kThreads / 32) + threadIdx.x / 32;
      if (work < works && find_rows(p, work, w)) append_rows<T, kInterleaved, 32, kHold>(p, w);
    } else {
      // a page's heads and a prompt's pages lie in different blocks, so that no block gets many that are large
      const auto work_of = [&](int warp) { return before + static_cast<long long>(page_blocks) * warp; };
      __shared__ bool large[kThreads / 32];
      const int warp = static_cast<int>(threadIdx.x / 32);
      const bool found = work_of(warp) < works && find_rows(p, work_of(warp), w);
      const bool by_warp = found && w.rows * (p.dim / (2 * kN)) <= kWarpItems;
      if (threadIdx.x % 32 == 0) large[warp] = found && !by_warp;
      const bool any = __syncthreads_or(found && !by_warp);
      if (by_warp) append_rows<T, kInterleaved, 32, kHold>(p, w);
      if (!any) return;
      for (int i = 0; i < kThreads / 32; ++i) {
        if (large[i] && find_rows(p, work_of(i), w)) append_rows<T, kInterleaved, kThreads, kHold>(p, w);
      }
    }
  } else {
    rotate_q<T, kInterleaved, kHeads>(p, static_cast<long long>(i - before));
  }
}

// (page, kv head, k or v) that tokens may come to
long long works_of(const KvAppendParams& p) {
  const long long page_slots = p.cu_seqlens == nullptr ? p.batch : (p.tokens >> p.page_shift) + 2ll * p.batch;
  return page_slots * p.kv_heads * 2;
}

template <typename T, bool kInterleaved, int kWho, int kHold, int kHeads>
cudaError_t launch_t(const KvAppendParams& p, cudaStream_t stream) {
  const long long works = works_of(p);
  constexpr int kPerBlock = kWho == kBlock ? 1 : kThreads / 32;
  const long long page_blocks = (works + kPerBlock - 1) / kPerBlock;
  const long long items = p.q == nullptr ? 0 : static_cast<long long>(p.tokens) * ((p.heads + kHeads - 1) / kHeads) * (p.dim / (2 * kN));
  const long long q_blocks = (items + kThreads - 1) / kThreads;
  if (page_blocks + q_blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  if (page_blocks + q_blocks == 0) return cudaSuccess;
  const long long blocks = page_blocks + q_blocks;
  const unsigned mix = kHold > 1 && q_blocks > 0 ? static_cast<unsigned>(((page_blocks << 32) + blocks - 1) / blocks) : 0u;
  kv_append_kernel<T, kInterleaved, kWho, kHold, kHeads>
      <<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p, works, static_cast<unsigned>(page_blocks), mix);
  return cudaGetLastError();
}

template <typename T, bool kInterleaved>
cudaError_t launch_i(const KvAppendParams& p, cudaStream_t stream) {
  // One token a sequence: a block for every page would leave nearly all of its threads idle.  Device us, warp / block a
  // page, 8 kv heads of 128: 250 sequences 6.3 / 18.6.
  if (p.cu_seqlens == nullptr) return launch_t<T, kInterleaved, kWarps, 1, 1>(p, stream);
  // More pages than a wave of blocks (148 SMs x 4) and few tokens a sequence, or a prompt among many single tokens.  Device
  // us, this / a block a page / a warp a page: 64 sequences x 1 token 4.4 / 9.5 / 4.1, x 12 10.2 / 13.1 / 10.0, x 16 12.7 /
  // 15.1, x 24 26.1 / 17.5 / 17.1; 63 x 1 and one of 400 9.3 / 12.9 / 22.6; 250 x 1 and one of 1500 24.5 / 38.7 / 33.6.  The
  // rule goes by the average: 63 x 1 and one of 2048 takes a block a page, 23.5.
  // Fewer pages: 16 x 12 6.6 / 5.4, 8 x 6 5.1 / 4.5 / 4.9.
  if (works_of(p) > 592 && p.tokens <= 16ll * p.batch) return launch_t<T, kInterleaved, kEither, 1, 1>(p, stream);
  // Two slots a thread: a warp for 16 tokens of 64 (5000 tokens in such pages 16.5 us, a block each 31.2), a block for 64
  // tokens of 128 (17438 tokens 115 us, a warp each 172).
  if (p.page_size * (p.dim / (2 * kN)) <= 64) return launch_t<T, kInterleaved, kWarps, 2, 4>(p, stream);
  return launch_t<T, kInterleaved, kBlock, 2, 4>(p, stream);
}

template <typename T>
cudaError_t launch_any(const KvAppendParams& p, cudaStream_t stream) {
  return p.interleaved ? launch_i<T, true>(p, stream) : launch_i<T, false>(p, stream);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, cudaStream_t stream) {
  return p.dtype == kQuantBf16 ? launch_any<__nv_bfloat16>(p, stream) : launch_any<__half>(p, stream);
}

}  // namespace b200fp8
