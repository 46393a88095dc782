// Attention of each sequence's newest tokens over a paged e4m3 cache (the layout that kv_append.cu writes).
//
//   s_ij = scale * k_scale[page(j)] * (q_i . code_j),   p_ij = exp(s_ij - max_j s_ij),
//   o_i  = sum_j p_ij * v_scale[page(j)] * code'_j / sum_j p_ij,      j = 0 .. position of query i
//
// Every cached byte is needed once per kv head and feeds 2 * group multiply-adds, so the floor is HBM: an SM has to take
// in 23 bytes of cache per clock.  What the kernel is built around:
//   * K is the A operand (16 tokens) and the queries are the B operand (8 columns) of mma.m16n8k16: the rows of queries
//     that share a kv head - group heads x new tokens, mostly 4 to 8 - fill a tile of 8 columns, where they would fill
//     half of a 16-row tile.  O^T = V^T P^T then has the head dimension as rows, and P^T goes from accumulator to
//     operand layout with one movmatrix per 8 tokens.
//   * e4m3 is exact in fp16, and so are queries once a row is scaled by a power of two, its largest element to [1, 2): of
//     those that fp16 holds in fewer bits then (bf16 below 2^-17 of the row's largest, fp16 below 2^-14) an element is off by
//     2^-25 of the largest at most.  p is rounded to fp16, to 2^-11 of itself, in units in which the largest is 2^11 to 2^15: what
//     is below 2^-25 of it is off by up to 2^-36 of it.  tcgen05 takes 8-bit operands only in pairs, which would round
//     queries and p to 3 bits of mantissa.  Sums, maxima and the output stay in fp32.
//   * The order of the contraction is free, so a thread's operand elements are 16 neighbouring bytes of a token:
//     whole 16-byte vectors are loaded, and the pairing of two tokens' V bytes costs one byte permute per 4 bytes.
//     A warp copies (cp.async, whole rows) and reads its own chunks, so the ring needs no barrier beyond the warp.
//   * v_scale differs by page: O is kept in units of the largest V scale of the chunk that was added last, so products
//     accumulate in place.
// Work is split over the context: all (sequence, kv head, row tile, unit of 4 chunks) units of the batch are one list,
// cut into equal runs for a grid that fills the GPU once; lengths are read on the device.  A run that ends inside a
// tile leaves its unnormalised sums in the workspace (at most two parts a CTA) and the second kernel joins them, in a
// fixed order.  The workspace needs no initialisation and nothing is kept in it between calls.
// Small calls (run_t) do without the list, the workspace and the second launch: a cluster of up to 8 CTAs takes a tile,
// divides its context evenly and joins through distributed shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "rotary.cuh"
#include "sequences.cuh"

namespace b200fp8 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kJoinThreads = 256;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMaxFloat = 3.402823466e38f;
constexpr float kMinusInf = -__builtin_inff();
constexpr uint32_t kNoPage = 0xffffffffu;  // in place of a chunk's k_scale: its page is not in the cache

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, bool take) {  // zeros where not taken
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// four e4m3 bytes -> bytes (0, 1) and bytes (2, 3) as fp16 pairs, exact
__device__ __forceinline__ void halves_of(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n"
      ".reg .b16 a, b;\n"
      "mov.b32 {a, b}, %2;\n"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n"
      "}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// the same, and 65504 for what is larger
__device__ __forceinline__ uint32_t finite_half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// lo += low half of h, hi += its high half, rounded once in fp32
__device__ __forceinline__ void add_halves(float& lo, float& hi, uint32_t h) {
  asm("{\n"
      ".reg .f16 a, b, one;\n"
      "mov.b32 {a, b}, %2;\n"
      "mov.b16 one, 0x3c00;\n"
      "fma.rn.f32.f16 %0, a, one, %0;\n"
      "fma.rn.f32.f16 %1, b, one, %1;\n"
      "}\n"
      : "+f"(lo), "+f"(hi)
      : "r"(h));
}
__device__ __forceinline__ void add_halves(float& lo, float& hi, uint32_t h, float times) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
  lo = fmaf(v.x, times, lo);
  hi = fmaf(v.y, times, hi);
}
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 2^(v f - ref), the product rounded as it was for the largest one that ref comes from: however large the scores are, the
// largest p is 2^kBelow, or what ref's own rounding makes of it (in a fused multiply-add the product's rounding error, 64 at
// 2^30, is left over in the argument)
__device__ __forceinline__ float exp2_of(float v, float f, float ref) { return exp2_approx(__fsub_rn(__fmul_rn(v, f), ref)); }
__device__ __forceinline__ bool has_nan_code(uint32_t w) {  // any byte 0x7f or 0xff
  const uint32_t m = (w & 0x7f7f7f7fu) + 0x01010101u;
  return (m & 0x80808080u) != 0;
}

// ------------------------------------------------------------------ the list of units
struct Seq {
  int n;          // new tokens
  int begin;      // position of the first new token; negative: more of them than the sequence has tokens
  int len;        // context, the new tokens included, as far as the block table goes
  int row_tiles;  // tiles of query rows
  int units;      // units of a tile, at least one (a tile without context still has an output)
  int q_base;     // first row of q
};

template <int kRows, int kUnit>
__device__ __forceinline__ Seq seq_of(const KvAttentionParams& p, int b) {
  Seq s;
  int first = b, last = b + 1;
  if (p.cu_seqlens != nullptr) {  // lengths that do not fit q are cut to it
    first = min(max(p.cu_seqlens[b], 0), p.tokens);
    last = min(max(p.cu_seqlens[b + 1], first), p.tokens);
  }
  s.q_base = first;
  s.n = last - first;
  const int len = max(p.seq_lens[b], 0);
  s.begin = len - s.n;
  s.len = min(len, p.max_len);
  s.row_tiles = static_cast<int>((static_cast<long long>(s.n) * p.group + kRows - 1) / kRows);
  s.units = max((s.len + kUnit - 1) / kUnit, 1);
  return s;
}
// Cost of a tile besides its units, in units: loading the queries, joining the warps and storing what they found takes a
// block 2 to 3 us, a unit takes it 2.0 us (three blocks an SM, the memory busy).  Shares of equal units without it ended
// between 67 and 98 us (64 sequences of 1 to 8192 tokens), those with eleven tiles last.  Device us for a cost of 1 / 2 / 3:
// those 95.1 / 93.5 / 94.5, drafted tokens 102.5 / 95.7 / 96.6; 48 sequences with heads of 64, whose tiles are half as
// large, 67.0 / 68.1 / 71.8.
template <int kUnit>
__host__ __device__ constexpr int tile_cost() { return kUnit >= 256 ? 1 : 2; }

template <int kRows, int kUnit>
__device__ __forceinline__ int cost_of(const KvAttentionParams& p, int b) {  // all sequences together: below 2^31
  const Seq s = seq_of<kRows, kUnit>(p, b);
  return s.row_tiles * p.kv_heads * (s.units + tile_cost<kUnit>());
}

// Equal shares of `total`: CTA c has [begin(c), begin(c + 1)).
struct Shares {
  int each, rest;  // the first `rest` shares are one larger
  __device__ __forceinline__ Shares(int total, int ctas) : each(total / ctas) { rest = total - each * ctas; }
  __device__ __forceinline__ int begin(int c) const { return c * each + min(c, rest); }
  // CTA whose share `at` is in.  Bounds that run backwards claim rows more than once: a sum of them that wraps can end inside a
  // tile, whose end is then no CTA's.  The join must not look for its part behind the workspace.
  __device__ __forceinline__ int holder(int at) const {
    const int large = rest * (each + 1);
    return min(at < large ? at / (each + 1) : rest + (at - large) / each, static_cast<int>(gridDim.x) - 1);
  }
};

// A place in the list: unit `unit` of tile `tile` (kv head, row tile) of sequence b.  The cost of a tile lies in front of
// its units: a share that begins or ends there begins or ends with the tile's first unit.
template <int kRows, int kUnit>
struct Cursor {
  Seq s;
  int b, tile, unit;
  // of the tile
  int kv_head, row0;
  int min_end, max_end;  // tokens that the tile's first and last query see: [0, end)

  // new token i sees the tokens up to its own position that the block table has room for: [0, end_of(i))
  __device__ __forceinline__ int end_of(int i) const { return min(max(s.begin + i + 1, 0), s.len); }
  __device__ __forceinline__ void enter_tile(const KvAttentionParams& p) {
    kv_head = tile / s.row_tiles;
    row0 = (tile - kv_head * s.row_tiles) * kRows;
    const int last_row = min(row0 + kRows, s.n * p.group) - 1;
    min_end = end_of(row0 / p.group);
    max_end = end_of(last_row / p.group);
  }
  __device__ __forceinline__ void enter_sequence(const KvAttentionParams& p) {
    s = seq_of<kRows, kUnit>(p, b);
  }
  // To the next unit, `left` being the rest of the share behind the present one, which becomes what is left behind the
  // cost of a tile that is entered.
  __device__ __forceinline__ void advance(const KvAttentionParams& p, int& left) {
    if (++unit < s.units || left <= 0) return;
    left -= tile_cost<kUnit>();
    if (left <= 0) return;  // the share ends in front of the tile's first unit
    unit = 0;
    if (++tile == s.row_tiles * p.kv_heads) {
      tile = 0;
      do {
        ++b;
        enter_sequence(p);
      } while (s.n == 0);  // units are left, so a sequence with rows follows
    }
    enter_tile(p);
  }
};

// A warp takes kChunk tokens a step, 8 KB of codes, in parts of kSub tokens that lie in one page each.
template <int kD, int kNT, int kSub>
struct Shape {
  static constexpr int kStages = 2;
  static constexpr int kRows = 8 * kNT;
  static constexpr int kChunk = 4096 / kD;
  static constexpr int kSubs = kChunk / kSub;
  static constexpr int kUnit = kWarps * kChunk;
  static constexpr int kMT = kChunk / 16;
  static constexpr int kTileBytes = kChunk * kD;               // codes of K or of V of a chunk
  static constexpr int kStageBytes = 2 * kTileBytes + 32;      // and the scales of its parts
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kVW = kD >= 128 ? 4 : 2;                // words of V a lane has of a token and 128 elements
  static constexpr int kVH = kD >= 128 ? kD / 128 : 1;
  static constexpr int kOT = 2 * kVW;                          // 16-row tiles of O^T per vector of V
  static constexpr int kQBytes = kRows * kD * 2;               // queries in fp16
  // the warps of a block join their O, 8 KB of rows at a time, where the chunk lay that each multiplied last
  static constexpr int kJoinNT = kNT < 256 / kD ? kNT : 256 / kD;
  static constexpr int kSmemBytes = kRingBytes + kQBytes;
  static constexpr int kClusteredSmemBytes = kSmemBytes + kRows * kD * 4;  // and what a CTA found
  static_assert(kJoinNT * 8 * kD * 4 <= 2 * kTileBytes && kSubs <= 4 && kSub % 16 == 0 && kNT % kJoinNT == 0, "");
};

// Where row and 16-byte vector c of a chunk's K or V lie in shared memory, in bytes.  A copy instruction writes whole
// rows (full lines in global memory: 6.8 TB/s of random 4 KB pieces, where a lane that fetched the vectors it reads
// itself, 64 bytes of 8 rows an instruction, got 5.1).  Operands are read from 8 (K) or 4 (V) rows at a time; the
// exclusive-or, together with the order in which tokens are assigned to operand rows (token_of), lets the eight (K,
// V) or sixteen (V, 8 bytes) lanes of a phase hit different banks.
template <int kD, int kChunk>
__device__ __forceinline__ uint32_t place(int row, int c) {
  if constexpr (kD == 64) return row * 64 + ((c ^ ((row >> 1) & 2)) << 4);
  return (c >> 3) * (kChunk * 128) + row * 128 + (((c ^ row) & 7) << 4);
}
// token (of 8) at operand row i: any bijection is right, as P and V are permuted alike
template <int kD>
__device__ __forceinline__ int token_of(int i) {
  if constexpr (kD == 64) return (i & 4) | ((0x2130 >> (4 * (i & 3))) & 3);  // 0 3 1 2, 4 7 5 6
  return i ^ ((i & 1) << 2);                                                  // 0 5 2 7, 4 1 6 3
}

// part of a tile in the workspace: O [kRows][kD], then (reference, sum) [kRows][2], then the sum for the log-sum-exp [kRows]
template <int kRows, int kD>
__host__ __device__ constexpr size_t part_floats() { return static_cast<size_t>(kRows) * (kD + 3); }

// A tile that CTAs first_cta to last_cta share (first_cta -1: none).
struct SharedTile {
  int first_cta, last_cta;
  int q_base, kv_head, row0, rows;
};
struct alignas(16) Split {
  SharedTile role[2];  // the tile inside which a CTA's share begins, the tile that it begins and does not finish
};

// q and out are bf16 or fp16: 16 bits an element either way
__device__ __forceinline__ void unpack_q(const uint4& raw, bool fp16, float (&v)[8]) {
  if (fp16) {
    unpack16<__half>(raw, v);
  } else {
    unpack16<__nv_bfloat16>(raw, v);
  }
}
__device__ __forceinline__ uint32_t pack_out2(float lo, float hi, bool fp16) {
  if (fp16) return half2_of(lo, hi);
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Four elements of an output row from its sums, and the row's log-sum-exp from the sum of p before its rounding (once, with
// the row's first elements).
__device__ __forceinline__ void store_row(const KvAttentionParams& p, int q_base, int kv_head, int row, int d, float4 acc,
                                          float top, float sum, float exact) {
  const int token = row / p.group;
  const int head = kv_head * p.group + row - token * p.group;
  const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);  // no token seen: zeros
  uint16_t* at = static_cast<uint16_t*>(p.out) + (q_base + static_cast<long long>(token)) * p.o_token + head * p.o_head + d;
  *reinterpret_cast<uint2*>(at) = make_uint2(pack_out2(acc.x * inv, acc.y * inv, p.fp16), pack_out2(acc.z * inv, acc.w * inv, p.fp16));
  if (p.lse != nullptr && d == 0) {
    p.lse[(q_base + static_cast<long long>(token)) * p.heads + head] = (top + log2f(exact)) * kLn2;
  }
}

// Rows in front of the first sequence and behind the last one: zeros (where asked for), and nothing to see.
template <int kD>
__device__ __forceinline__ void fill_rest(const KvAttentionParams& p, int threads) {
  if (p.cu_seqlens == nullptr || (!p.fill_rest && p.lse == nullptr)) return;
  const int first = min(max(p.cu_seqlens[0], 0), p.tokens), end = min(max(p.cu_seqlens[p.batch], first), p.tokens);
  const long long n = static_cast<long long>(first + p.tokens - end) * p.heads;
  for (long long r = blockIdx.x; r < n; r += gridDim.x) {
    const long long at = r / p.heads, token = at < first ? at : at - first + end;
    const int head = static_cast<int>(r % p.heads);
    uint16_t* o = static_cast<uint16_t*>(p.out) + token * p.o_token + head * p.o_head;
    if (p.fill_rest) {
      for (int d = threadIdx.x; d < kD; d += threads) o[d] = 0;
    }
    if (p.lse != nullptr && threadIdx.x == 0) p.lse[token * p.heads + head] = kMinusInf;
  }
}

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();  // the aligned forms want whole warps
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {  // the same shared memory of another CTA of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float load_cluster1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 load_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// kClustered: a cluster per tile (see run_t), else the shared list.  kLse: the log-sum-exp is asked for.  The output divides
// by the sum of p as it was rounded to fp16 (what a row's largest p is off by then cancels); the log-sum-exp is that of p in
// fp32, a second sum.  Device us without / with it: 64 requests 95.9 / 95.9, 48 requests with heads of 64 66.2 / 67.9, drafted
// tokens (16 rows a tile, no register to spare) 94.0 / 100.2, so the other calls do without.
template <int kD, int kNT, int kSub, bool kClustered, bool kLse>
__global__ void __launch_bounds__(kThreads, kNT * kD <= 256 ? 3 : 2) kv_attention_kernel(const KvAttentionParams p) {
  using S = Shape<kD, kNT, kSub>;
  using C = Cursor<S::kRows, S::kUnit>;
  constexpr int kChunk = S::kChunk, kStages = S::kStages;
  extern __shared__ __align__(128) char smem[];
  __shared__ int sums[kWarps], found_b, found_before;
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int g = lane >> 2, t = lane & 3;
  const int cta = static_cast<int>(blockIdx.x);
  Split* splits = static_cast<Split*>(p.workspace);
  float* parts = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + p.parts_offset);

  // ---- what this CTA has to do
  C cur;
  int left;                      // units of this CTA, from cur's on
  Shares shares(0, 1);
  int run_end = 0;
  if constexpr (kClustered) {
    fill_rest<kD>(p, kThreads);
    const int slot = cta / p.cluster;  // (row tile, kv head)
    const int row_slot = slot / p.kv_heads, kv_head = slot - row_slot * p.kv_heads;
    int row_tile;
    if (p.cu_seqlens == nullptr) {
      const int tiles = (p.group + S::kRows - 1) / S::kRows;
      cur.b = row_slot / tiles;
      row_tile = row_slot - cur.b * tiles;
    } else {  // sequence b owns the slots from cu[b] * group / kRows + b on, at least as many as it has row tiles
      const auto first_slot = [&](int i) {
        return static_cast<long long>(min(max(p.cu_seqlens[i], 0), p.tokens)) * p.group / S::kRows + i;
      };
      cur.b = search_sequence(p.batch, row_slot, first_slot);
      row_tile = static_cast<int>(row_slot - first_slot(cur.b));
    }
    if (cur.b >= p.batch) return;
    cur.enter_sequence(p);
    if (row_tile < 0 || row_tile >= cur.s.row_tiles) return;  // a slot without a tile, for the whole cluster
    cur.tile = kv_head * cur.s.row_tiles + row_tile;
    cur.enter_tile(p);
    const int rank = cta % p.cluster;
    cur.unit = cur.s.units * rank / p.cluster;
    left = cur.s.units * (rank + 1) / p.cluster - cur.unit;
  } else {
    if (threadIdx.x == 0) splits[cta].role[0].first_cta = splits[cta].role[1].first_cta = found_b = -1;
    int total = 0, own = 0;
    for (int b = threadIdx.x; b < p.batch; b += kThreads) own = cost_of<S::kRows, S::kUnit>(p, b), total += own;
    int upto = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += sums[w];
      total += sums[w];
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join waits for this grid to complete
    const int ctas = min(total, static_cast<int>(gridDim.x));
    if (cta >= ctas) return;
    shares = Shares(total, ctas);
    const int run_begin = shares.begin(cta);
    run_end = shares.begin(cta + 1);
    if (p.batch <= kThreads) {  // a thread has one sequence, and what lies in front of it
      if (run_begin >= upto - own && run_begin < upto) {
        found_b = threadIdx.x;
        found_before = upto - own;
      }
    } else {
      int before = 0;  // in front of b0
      for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
        const int b = b0 + static_cast<int>(threadIdx.x);
        own = b < p.batch ? cost_of<S::kRows, S::kUnit>(p, b) : 0;
        upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        __syncthreads();  // sums of the step before have been read
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        int step = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) upto += sums[w];
          step += sums[w];
        }
        upto += before;
        if (run_begin >= upto - own && run_begin < upto) {  // one thread of one step
          found_b = b;
          found_before = upto - own;
        }
        before += step;
        if (before > run_begin) break;
      }
    }
    __syncthreads();

    if (found_b < 0) return;  // bounds that run backwards and count rows more than once: the sum may have wrapped
    cur.b = found_b;
    cur.enter_sequence(p);
    left = run_end - run_begin;
    {
      constexpr int kCost = tile_cost<S::kUnit>();
      const int in_seq = run_begin - found_before, of_tile = cur.s.units + kCost;
      cur.tile = in_seq / of_tile;
      const int in_tile = in_seq - cur.tile * of_tile;
      cur.unit = max(in_tile - kCost, 0);
      left -= max(kCost - in_tile, 0);
    }
    if (left <= 0) return;  // nothing but the cost of a tile
    cur.enter_tile(p);
    if (threadIdx.x == 0 && cur.unit > 0) {
      const int tile_begin = run_begin - cur.unit;
      splits[cta].role[0] = {shares.holder(tile_begin), shares.holder(tile_begin + cur.s.units - 1), cur.s.q_base, cur.kv_head,
                             cur.row0, min(S::kRows, cur.s.n * p.group - cur.row0)};
    }
  }
  C ahead = cur;
  int ahead_left = left;

  // ---- the ring of a warp: it copies and reads its own chunks, in step
  char* const ring = smem + warp * kStages * S::kStageBytes;
  constexpr int kRowVecs = kD / 16;         // 16-byte vectors of a row
  constexpr int kCopyRows = 32 / kRowVecs;  // rows that one copy instruction of the warp covers
  const int copy_row = lane / kRowVecs, copy_vec = lane % kRowVecs;
  constexpr int kPlaces = 8 / kCopyRows > 0 ? 8 / kCopyRows : 1;  // the placement repeats after 8 rows
  uint32_t copy_at[kPlaces];
#pragma unroll
  for (int i = 0; i < kPlaces; ++i) copy_at[i] = place<kD, kChunk>(i * kCopyRows + copy_row, copy_vec);
  constexpr int k8Rows = 8 * (kD == 64 ? 64 : 128);  // bytes from a row to the one 8 further
  const bool dense = p.k_row == kD && p.v_row == kD;
  // operand rows: K tokens g and g + 8 of 16; V tokens 2t, 2t + 1 and those + 8 (the placement repeats after 8 rows)
  int k_at[kD / 64], v_at[2][S::kVH];
#pragma unroll
  for (int j = 0; j < kD / 64; ++j) k_at[j] = place<kD, kChunk>(token_of<kD>(g), 4 * j + t);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < S::kVH; ++h) {
      const int row = token_of<kD>(2 * t + i);
      v_at[i][h] = S::kTileBytes + (kD == 64 ? place<kD, kChunk>(row, g >> 1) + 8 * (g & 1) : place<kD, kChunk>(row, 8 * h + g));
    }
  __shared__ float join_ml[kWarps][S::kRows][2];
  __shared__ __align__(8) float row_scale[S::kRows];  // of a query row: what its scores are multiplied by, in units of log2
  __shared__ __align__(8) int row_end[S::kRows];      // the tokens it sees: [0, end)
  char* const queries = smem + S::kRingBytes;
  float4* const own_rows = reinterpret_cast<float4*>(queries + S::kQBytes);  // clustered: what this CTA found, unnormalised
  __shared__ float2 own_ml[S::kRows];
  __shared__ float join_exact[kWarps][kLse ? S::kRows : 1], own_exact[kLse ? S::kRows : 1];

  int next_page = -1;  // lane i: page of part i of the chunk that is requested next, loaded one step early
  const auto look_up = [&]() {
    next_page = -1;
    if (ahead_left > 0 && lane < S::kSubs) {
      const int token = ahead.unit * S::kUnit + warp * kChunk + lane * kSub;
      if (token < ahead.max_end) next_page = p.block_table[ahead.b * p.bt_stride + (token >> p.page_shift)];
    }
  };
  const auto request = [&](int stage) {  // one group a call, also when there is nothing to request
    if (ahead_left > 0) {
      const int token0 = ahead.unit * S::kUnit + warp * kChunk;
      if (token0 < ahead.max_end) {
        char* const at = ring + stage * S::kStageBytes;
        const uint32_t base = smem_addr(at);
        const int mine = next_page >= 0 && next_page < p.num_pages ? next_page : -1;
        const bool whole_chunk = token0 + kChunk <= ahead.max_end && __all_sync(0xffffffffu, mine >= 0 || lane >= S::kSubs);
        const uint8_t* const k_head = p.k_cache + static_cast<long long>(ahead.kv_head) * p.k_head;
        const uint8_t* const v_head = p.v_cache + static_cast<long long>(ahead.kv_head) * p.v_head;
        const auto copy_chunk = [&](auto whole, int k_row, int v_row) {
#pragma unroll
          for (int sub = 0; sub < S::kSubs; ++sub) {
            const int page = __shfl_sync(0xffffffffu, mine, sub);
            const long long at_page = whole.value ? page : max(page, 0);
            const int row0 = ((token0 + sub * kSub) & (p.page_size - 1)) + copy_row;
            const uint8_t* k = k_head + at_page * p.k_page + (row0 * k_row + 16 * copy_vec);
            const uint8_t* v = v_head + at_page * p.v_page + (row0 * v_row + 16 * copy_vec);
            const int left = page < 0 ? 0 : ahead.max_end - token0 - sub * kSub;  // tokens of the part that there are
#pragma unroll
            for (int n = 0; n < kSub / kCopyRows; ++n) {
              const int row = sub * kSub + n * kCopyRows;
              const uint32_t to = base + copy_at[n % kPlaces] + row / 8 * k8Rows;
              if constexpr (whole.value) {
                copy_async16(to, k + n * kCopyRows * k_row);
                copy_async16(to + S::kTileBytes, v + n * kCopyRows * v_row);
              } else {  // (q: an address that is not read, and there even when the cache has no page)
                const bool take = n * kCopyRows + copy_row < left;
                copy_async16(to, take ? static_cast<const void*>(k + n * kCopyRows * k_row) : p.q, take);
                copy_async16(to + S::kTileBytes, take ? static_cast<const void*>(v + n * kCopyRows * v_row) : p.q, take);
              }
            }
          }
        };
        if (!whole_chunk) {  // zeros in place of the others: zero times NaN is NaN
          copy_chunk(std::false_type{}, p.k_row, p.v_row);
        } else if (dense) {  // offsets that are known
          copy_chunk(std::true_type{}, kD, kD);
        } else {
          copy_chunk(std::true_type{}, p.k_row, p.v_row);
        }
        const int page = __shfl_sync(0xffffffffu, mine, lane >> 1);
        if (lane < 2 * S::kSubs) {
          if (page < 0) {
            *reinterpret_cast<uint32_t*>(at + 2 * S::kTileBytes + 4 * lane) = kNoPage;
          } else {
            copy_async4(base + 2 * S::kTileBytes + 4 * lane,
                          (lane & 1) ? p.v_scale + static_cast<long long>(page) * p.vs_page + static_cast<long long>(ahead.kv_head) * p.vs_head
                                     : p.k_scale + static_cast<long long>(page) * p.ks_page + static_cast<long long>(ahead.kv_head) * p.ks_head);
          }
        }
      }
      --ahead_left;
      ahead.advance(p, ahead_left);
    }
    copy_commit();
    look_up();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) request(s);

  int stage = 0;
  while (left > 0) {
    // ---- a segment: the units of this run that belong to one tile
    const int unit0 = cur.unit;
    const int unit_end = min(cur.s.units, unit0 + left);
    const int rows = min(S::kRows, cur.s.n * p.group - cur.row0);
    // queries to fp16, each row scaled by a power of two to a largest element in [1, 2); 16 elements a thread
    for (int i = threadIdx.x; i < S::kRows * (kD / 16); i += kThreads) {
      const int r = i / (kD / 16), piece = i % (kD / 16);
      const int row = cur.row0 + min(r, rows - 1);
      const int token = row / p.group;
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + (cur.s.q_base + static_cast<long long>(token)) * p.q_token +
                                                      (cur.kv_head * p.group + row - token * p.group) * p.q_head + 16 * piece);
      float x[16], big = 0.0f;
      {
        float a[8], b[8];
        unpack_q(q[0], p.fp16, a);
        unpack_q(q[1], p.fp16, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = a[e];
          x[8 + e] = b[e];
          big = fmaxf(big, fmaxf(fabsf(a[e]), fabsf(b[e])));
        }
      }
#pragma unroll
      for (int o = 1; o < kD / 16; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
      // rows of zeros, and with infinities, as they are
      int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
      e = big > 0.0f && e < 128 ? max(min(e, 126), -126) : 0;
      float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      if (p.softmax_scale < 0.0f) down = -down;  // the factor on the scores stays positive: their maximum is found first
      uint32_t h[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) h[c] = half2_of(x[2 * c] * down, x[2 * c + 1] * down);
      uint4* to = reinterpret_cast<uint4*>(queries + r * kD * 2);
      to[(2 * piece) ^ (r & 1)] = make_uint4(h[0], h[1], h[2], h[3]);  // neighbouring rows in different banks
      to[(2 * piece + 1) ^ (r & 1)] = make_uint4(h[4], h[5], h[6], h[7]);
      if (piece == 0) {
        row_scale[r] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * (fabsf(p.softmax_scale) * kLog2e);
        row_end[r] = r < rows ? cur.end_of(token) : 0;
      }
    }
    __syncthreads();
    float o[S::kVH][S::kOT][kNT][4];
#pragma unroll
    for (int h = 0; h < S::kVH; ++h)
#pragma unroll
      for (int i = 0; i < S::kOT; ++i)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) o[h][i][nt][0] = o[h][i][nt][1] = o[h][i][nt][2] = o[h][i][nt][3] = 0.0f;
    float v_unit = 1.0f, v_top = 1.0f;  // unit of o, the largest so far
    float m[kNT][2], l[kNT][2], exact[kNT][2];  // reference, sum of p as it was rounded, sum of p
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      m[nt][0] = m[nt][1] = kMinusInf;
      l[nt][0] = l[nt][1] = exact[nt][0] = exact[nt][1] = 0.0f;
    }

    for (int unit = unit0; unit < unit_end; ++unit) {
      __syncwarp();                                   // all lanes have read the stage that was emptied one step ago
      request(stage == 0 ? kStages - 1 : stage - 1);  // and is filled again
      copy_wait<kStages - 1>();
      __syncwarp();  // what the other lanes copied is there too
      const char* const base = ring + stage * S::kStageBytes;
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const int token0 = unit * S::kUnit + warp * kChunk;
      if (token0 >= cur.max_end) continue;
      float k_scale[S::kSubs], v_scale[S::kSubs];
      bool there[S::kSubs];
      bool partial = token0 + kChunk > cur.min_end;  // some column does not see all of the chunk
#pragma unroll
      for (int sub = 0; sub < S::kSubs; ++sub) {
        const uint2 sc = *reinterpret_cast<const uint2*>(base + 2 * S::kTileBytes + 8 * sub);
        there[sub] = sc.x != kNoPage;
        k_scale[sub] = __uint_as_float(sc.x);
        v_scale[sub] = __uint_as_float(sc.y);
        partial = partial || !there[sub];
      }

      // ---- S^T = K Q^T
      float s[S::kMT][kNT][4];
#pragma unroll
      for (int mt = 0; mt < S::kMT; ++mt)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < kD / 64; ++j) {
        uint32_t qf[kNT][8];  // elements 64 j + 16 t .. + 15 of column 8 nt + g
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const uint4* q = reinterpret_cast<const uint4*>(queries + (8 * nt + g) * kD * 2) + 8 * j;
          const uint4 lo = q[(2 * t) ^ (g & 1)], hi = q[(2 * t + 1) ^ (g & 1)];
          qf[nt][0] = lo.x, qf[nt][1] = lo.y, qf[nt][2] = lo.z, qf[nt][3] = lo.w;
          qf[nt][4] = hi.x, qf[nt][5] = hi.y, qf[nt][6] = hi.z, qf[nt][7] = hi.w;
        }
        uint32_t w[S::kMT][2][4];
#pragma unroll
        for (int mt = 0; mt < S::kMT; ++mt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(base + k_at[j] + (2 * mt + i) * k8Rows);
            w[mt][i][0] = v.x, w[mt][i][1] = v.y, w[mt][i][2] = v.z, w[mt][i][3] = v.w;
          }
#pragma unroll
        for (int i = 0; i < 4; ++i)  // neighbouring products do not wait for one another's sums
#pragma unroll
          for (int mt = 0; mt < S::kMT; ++mt) {
            uint32_t a0, a1, a2, a3;
            halves_of(w[mt][0][i], a0, a2);
            halves_of(w[mt][1][i], a1, a3);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) mma16816(s[mt][nt], a0, a1, a2, a3, qf[nt][2 * i], qf[nt][2 * i + 1]);
          }
      }
      // ---- softmax over the tokens, column by column.  The reference m is kBelow below a column's largest score when it is
      // set, so that fp16's range lies where the weights are (without it, first tokens that take nearly all of the weight
      // would leave the others, 17 and more below in units of e, to subnormals and zero).  It follows the largest score only
      // when that has grown by more than kSlack: p is at most 2^(kBelow + kSlack), and O and l are hardly ever rescaled
      // after a few chunks.
      constexpr float kBelow = 11.0f, kSlack = 4.0f;
      uint32_t pf[S::kMT][kNT][2];
      // The factor of a page's scores goes into the exponent's argument (it is not negative, so the largest product is the
      // largest score); masked scores are multiplied first.
      float2 col[kNT];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) col[nt] = *reinterpret_cast<const float2*>(&row_scale[8 * nt + 2 * t]);
      if (partial) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          const int2 end = *reinterpret_cast<const int2*>(&row_end[8 * nt + 2 * t]);
#pragma unroll
          for (int mt = 0; mt < S::kMT; ++mt) {
            const float f0 = col[nt].x * k_scale[mt * 16 / kSub], f1 = col[nt].y * k_scale[mt * 16 / kSub];
            const int token = there[mt * 16 / kSub] ? token0 + 16 * mt + token_of<kD>(g) : 0x7ffffff0;
            s[mt][nt][0] = token < end.x ? s[mt][nt][0] * f0 : kMinusInf;
            s[mt][nt][1] = token < end.y ? s[mt][nt][1] * f1 : kMinusInf;
            s[mt][nt][2] = token + 8 < end.x ? s[mt][nt][2] * f0 : kMinusInf;
            s[mt][nt][3] = token + 8 < end.y ? s[mt][nt][3] * f1 : kMinusInf;
          }
          col[nt] = make_float2(1.0f, 1.0f);  // what is left to multiply by
        }
#pragma unroll
        for (int sub = 0; sub < S::kSubs; ++sub) k_scale[sub] = 1.0f;
      }
      float top[kNT][2];
      bool passed = false;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        float top0 = kMinusInf, top1 = kMinusInf;
        constexpr int kSteps = kSub / 16;
#pragma unroll
        for (int sub = 0; sub < S::kSubs; ++sub) {
          float in0 = fmaxf(s[sub * kSteps][nt][0], s[sub * kSteps][nt][2]), in1 = fmaxf(s[sub * kSteps][nt][1], s[sub * kSteps][nt][3]);
#pragma unroll
          for (int mt = sub * kSteps + 1; mt < (sub + 1) * kSteps; ++mt) {
            in0 = fmaxf(in0, fmaxf(s[mt][nt][0], s[mt][nt][2]));
            in1 = fmaxf(in1, fmaxf(s[mt][nt][1], s[mt][nt][3]));
          }
          top0 = S::kSubs == 1 ? in0 : fmaxf(top0, in0 * (col[nt].x * k_scale[sub]));
          top1 = S::kSubs == 1 ? in1 : fmaxf(top1, in1 * (col[nt].y * k_scale[sub]));
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
          top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
        }
        top[nt][0] = S::kSubs == 1 ? top0 * (col[nt].x * k_scale[0]) : top0;
        top[nt][1] = S::kSubs == 1 ? top1 * (col[nt].y * k_scale[0]) : top1;
        passed = passed || top[nt][0] > m[nt][0] + (kBelow + kSlack) || top[nt][1] > m[nt][1] + (kBelow + kSlack);
      }
      if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          float f[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            f[c] = 1.0f;
            if (top[nt][c] > m[nt][c] + (kBelow + kSlack)) {
              const float to = top[nt][c] - kBelow;
              f[c] = exp2_approx(m[nt][c] - to);
              m[nt][c] = to;
              l[nt][c] *= f[c];
              if constexpr (kLse) exact[nt][c] *= f[c];
            }
          }
#pragma unroll
          for (int h = 0; h < S::kVH; ++h)
#pragma unroll
            for (int i = 0; i < S::kOT; ++i) {
              o[h][i][nt][0] *= f[0];
              o[h][i][nt][1] *= f[1];
              o[h][i][nt][2] *= f[0];
              o[h][i][nt][3] *= f[1];
            }
        }
      }
      // V scales: O is kept in units of the chunk's largest one, so that products can be added to it where they are; p is
      // multiplied by what a page's scale is of that, down to an eighth: in fp16 where the scales are powers of two (as the
      // append makes them; exact down to subnormals), else in fp32 before the one rounding to fp16 (48 requests with heads of
      // 64 and pages of 16, a call: 74 us when all chunks with different scales did that, 69.7 so, 68.7 with fp16 for all).
      float v_max = 0.0f;
#pragma unroll
      for (int sub = 0; sub < S::kSubs; ++sub) v_max = there[sub] ? fmaxf(v_max, v_scale[sub]) : v_max;
      bool plain = v_max <= kMaxFloat && v_max >= v_top * 0x1p-72f;
      bool mixed = false;
#pragma unroll
      for (int sub = 0; sub < S::kSubs; ++sub) {
        if (S::kSubs > 1) {
          plain = plain && (!there[sub] || v_scale[sub] >= v_max * 0.125f);
          mixed = mixed || (there[sub] && v_scale[sub] != v_max);
        }
      }
      mixed = mixed && plain;
      float share[S::kSubs];  // of the largest scale
      bool odd = false;       // some share is no power of two
      if (S::kSubs > 1 && mixed) {
        const float inv = 1.0f / v_max;
#pragma unroll
        for (int sub = 0; sub < S::kSubs; ++sub) {
          share[sub] = there[sub] ? v_scale[sub] * inv : 1.0f;
          odd = odd || (__float_as_uint(share[sub]) & 0x7fffffu) != 0;
        }
      }
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        // a column without a token so far: any finite reference will do
        const float ref0 = m[nt][0] == kMinusInf ? 0.0f : m[nt][0], ref1 = m[nt][1] == kMinusInf ? 0.0f : m[nt][1];
        // l sums p as it was rounded: what a row's largest p is off by cancels in the quotient.  Behind scores of 2^24 and more
        // the reference is rounded to several units, so that p may pass 2^(kBelow + kSlack) and fp16's largest.
        const auto weights = [&](auto by_share) {
#pragma unroll
          for (int mt = 0; mt < S::kMT; ++mt) {
            const float e0 = col[nt].x * k_scale[mt * 16 / kSub], e1 = col[nt].y * k_scale[mt * 16 / kSub];
            const float p0 = exp2_of(s[mt][nt][0], e0, ref0), p1 = exp2_of(s[mt][nt][1], e1, ref1);
            const float p2 = exp2_of(s[mt][nt][2], e0, ref0), p3 = exp2_of(s[mt][nt][3], e1, ref1);
            if constexpr (by_share.value) {
              const float f = share[mt * 16 / kSub], back = 1.0f / f;
              pf[mt][nt][0] = finite_half2_of(p0 * f, p1 * f);
              pf[mt][nt][1] = finite_half2_of(p2 * f, p3 * f);
              add_halves(l[nt][0], l[nt][1], pf[mt][nt][0], back);
              add_halves(l[nt][0], l[nt][1], pf[mt][nt][1], back);
            } else {
              pf[mt][nt][0] = finite_half2_of(p0, p1);
              pf[mt][nt][1] = finite_half2_of(p2, p3);
              add_halves(l[nt][0], l[nt][1], pf[mt][nt][0]);
              add_halves(l[nt][0], l[nt][1], pf[mt][nt][1]);
            }
            if constexpr (kLse) {
              exact[nt][0] += p0 + p2;
              exact[nt][1] += p1 + p3;
            }
          }
        };
        if (S::kSubs > 1 && odd) {
          weights(std::true_type{});
        } else {
          weights(std::false_type{});
          if (S::kSubs > 1 && mixed) {
#pragma unroll
            for (int mt = 0; mt < S::kMT; ++mt) {
              const uint32_t f = half2_of(share[mt * 16 / kSub], share[mt * 16 / kSub]);
#pragma unroll
              for (int i = 0; i < 2; ++i) asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(pf[mt][nt][i]) : "r"(f));
            }
          }
        }
#pragma unroll
        for (int mt = 0; mt < S::kMT; ++mt) {
          pf[mt][nt][0] = transpose8x8(pf[mt][nt][0]);
          pf[mt][nt][1] = transpose8x8(pf[mt][nt][1]);
        }
      }
      bool strange = false;
      if (partial && cur.min_end < cur.max_end) {
        // Tokens of this chunk that some columns see and others do not: their p is zero there, but zero times NaN is
        // NaN.  Look whether such a token has a NaN (or its page a scale that is not finite).
        bool bad = false;
#pragma unroll
        for (int sub = 0; sub < S::kSubs; ++sub) bad = bad || (there[sub] && !(fabsf(v_scale[sub]) <= kMaxFloat));
#pragma unroll 1
        for (int i = lane * 16; i < S::kTileBytes; i += 512) {
          const uint4 v = *reinterpret_cast<const uint4*>(base + S::kTileBytes + i);
          bad = bad || has_nan_code(v.x) || has_nan_code(v.y) || has_nan_code(v.z) || has_nan_code(v.w);
        }
        strange = __any_sync(0xffffffffu, bad);
      }
      // ---- O^T += V^T P^T.  Plain: the whole chunk, products added to O as they are.  cut: one part of it, V counts as zero
      // from token `end` of the chunk on, and the columns that `takes` names get f * product.
      const auto product = [&](auto cut, int sub, int end, float f, auto takes) {
#pragma unroll
        for (int h = 0; h < S::kVH; ++h) {
          constexpr int kW = S::kVW, kSteps = cut.value ? kSub / 16 : S::kMT;
          uint32_t w[kSteps][4][kW];
#pragma unroll
          for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int mt = sub * kSteps + ks;
              const char* from = base + v_at[i & 1][h] + (2 * mt + (i >> 1)) * k8Rows;
              if constexpr (kW == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(from);
                w[ks][i][0] = v.x, w[ks][i][1] = v.y, w[ks][i][2] = v.z, w[ks][i][3] = v.w;
              } else {
                const uint2 v = *reinterpret_cast<const uint2*>(from);
                w[ks][i][0] = v.x, w[ks][i][1] = v.y;
              }
              if constexpr (cut.value) {
                if (16 * mt + token_of<kD>(2 * t + (i & 1)) + 8 * (i >> 1) >= end) {
#pragma unroll
                  for (int c = 0; c < kW; ++c) w[ks][i][c] = 0u;
                }
              }
            }
          float d[kW][2][kNT][4];
          if constexpr (cut.value) {
#pragma unroll
            for (int c = 0; c < kW; ++c)
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) d[c][0][nt][e] = d[c][1][nt][e] = 0.0f;
          }
#pragma unroll
          for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
            for (int c = 0; c < kW; ++c)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const uint32_t pick = half == 0 ? 0x5140u : 0x7362u;  // bytes 2 half, 2 half + 1 of two tokens, interleaved
                const int mt = sub * kSteps + ks;
                uint32_t a0, a1, a2, a3;
                halves_of(__byte_perm(w[ks][0][c], w[ks][1][c], pick), a0, a1);
                halves_of(__byte_perm(w[ks][2][c], w[ks][3][c], pick), a2, a3);
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt) {
                  mma16816(cut.value ? d[c][half][nt] : o[h][2 * c + half][nt], a0, a1, a2, a3, pf[mt][nt][0], pf[mt][nt][1]);
                }
              }
          if constexpr (cut.value) {
#pragma unroll
            for (int c = 0; c < kW; ++c)
#pragma unroll
              for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    if (takes(nt, e & 1)) o[h][2 * c + half][nt][e] = fmaf(d[c][half][nt][e], f, o[h][2 * c + half][nt][e]);
                  }
          }
        }
      };
      if (!strange && plain) {
        if (v_max != v_unit) {
          const float ratio = v_unit / v_max;
          v_unit = v_max;
          v_top = fmaxf(v_top, v_max);
#pragma unroll
          for (int h = 0; h < S::kVH; ++h)
#pragma unroll
            for (int i = 0; i < S::kOT; ++i)
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[h][i][nt][e] *= ratio;
        }
        product(std::false_type{}, 0, 0, 1.0f, [](int, int) { return true; });
      } else {
        // Something that is not finite, or scales too far apart (zero, or 2^72 below the largest so far, would take O out
        // of fp32's range): every part on its own, added with its factor, once for every place where a column's context
        // can end in the part or behind it, with V cut there; columns that see nothing of the part take nothing from it.
        const int lo = min(max(cur.min_end - token0, 0), kChunk), hi = min(cur.max_end - token0, kChunk);
#pragma unroll
        for (int sub = 0; sub < S::kSubs; ++sub) {
          if (!there[sub]) continue;
          const float f = (mixed ? v_max : v_scale[sub]) / v_unit;  // p may have its share of the largest already
          for (int end = max(lo, sub * kSub + 1); end <= hi; ++end) {
            product(std::true_type{}, sub, end, f, [&](int nt, int c) {
              return min(row_end[8 * nt + 2 * t + c] - token0, kChunk) == end;
            });
          }
        }
      }
    }

    // ---- join the warps: O in the stage that was emptied last (no copy into it is on its way), 16-byte vectors of a
    // row exchanged so that the lanes of a phase write to different banks
    const bool begins = unit0 == 0, ends = unit_end == cur.s.units;
    float* const part = parts + (2ll * cta + (begins ? 1 : 0)) * part_floats<S::kRows, kD>();
    const int last = stage == 0 ? kStages - 1 : stage - 1;  // the warps of a block are at the same stage
    const auto join_row = [&](int w, int r) {
      return reinterpret_cast<float4*>(smem + (w * kStages + last) * S::kStageBytes) + r * (kD / 4);
    };
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
          if constexpr (kLse) exact[nt][c] += __shfl_xor_sync(0xffffffffu, exact[nt][c], x);
        }
        if (g == 0) {
          join_ml[warp][8 * nt + 2 * t + c][0] = m[nt][c];
          join_ml[warp][8 * nt + 2 * t + c][1] = l[nt][c];
          if constexpr (kLse) join_exact[warp][8 * nt + 2 * t + c] = exact[nt][c];
        }
      }
#pragma unroll
    for (int nt0 = 0; nt0 < kNT; nt0 += S::kJoinNT) {
      if (nt0 > 0) __syncthreads();  // the rows before have been read
      __syncwarp();                  // all lanes have read the stage
#pragma unroll
      for (int nt = nt0; nt < nt0 + S::kJoinNT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float4* row = join_row(warp, 8 * (nt - nt0) + 2 * t + c);
#pragma unroll
          for (int h = 0; h < S::kVH; ++h)
#pragma unroll
            for (int i = 0; i < S::kOT; i += 2) {
              row[(32 * h + S::kVW * g + i / 2) ^ t] =
                  make_float4(o[h][i][nt][c] * v_unit, o[h][i][nt][2 + c] * v_unit, o[h][i + 1][nt][c] * v_unit,
                              o[h][i + 1][nt][2 + c] * v_unit);
            }
        }
      __syncthreads();
      const int first_row = 8 * nt0, row_count = min(rows - first_row, 8 * S::kJoinNT);
      for (int i = threadIdx.x; i < row_count * (kD / 4); i += kThreads) {
        const int in = i / (kD / 4), d = i % (kD / 4), r = first_row + in;
        float top = join_ml[0][r][0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, join_ml[w][r][0]);
        const float ref = top == kMinusInf ? 0.0f : top;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f, all = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = exp2_approx(join_ml[w][r][0] - ref);
          const float4 v = join_row(w, in)[d ^ ((r >> 1) & 3)];
          sum = fmaf(join_ml[w][r][1], f, sum);
          if constexpr (kLse) all = fmaf(join_exact[w][r], f, all);
          acc.x = fmaf(v.x, f, acc.x);
          acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z);
          acc.w = fmaf(v.w, f, acc.w);
        }
        if constexpr (kClustered) {
          own_rows[r * (kD / 4) + d] = acc;
          if (d == 0) {
            own_ml[r] = make_float2(top, sum);
            if constexpr (kLse) own_exact[r] = all;
          }
        } else if (begins && ends) {
          store_row(p, cur.s.q_base, cur.kv_head, cur.row0 + r, 4 * d, acc, top, sum, all);
        } else {
          reinterpret_cast<float4*>(part)[r * (kD / 4) + d] = acc;
          if (d == 0) {
            part[S::kRows * kD + 2 * r] = top;
            part[S::kRows * kD + 2 * r + 1] = sum;
            if constexpr (kLse) part[S::kRows * (kD + 2) + r] = all;
          }
        }
      }
    }
    if (!kClustered && begins && !ends && threadIdx.x == 0) {
      // the share ends with this segment, so the tile's last unit is as far behind the share's end as behind the segment's
      splits[cta].role[1] = {cta, shares.holder(run_end + (cur.s.units - unit_end) - 1), cur.s.q_base, cur.kv_head, cur.row0, rows};
    }
    __syncthreads();  // the warps' sums and the queries have been read
    left -= unit_end - unit0;
    cur.unit = unit_end - 1;
    cur.advance(p, left);
  }
  copy_wait<0>();
  if constexpr (kClustered) {
    const int rows = min(S::kRows, cur.s.n * p.group - cur.row0), rank = cta % p.cluster;
    if (cur.s.units * rank / p.cluster == cur.s.units * (rank + 1) / p.cluster) {  // more CTAs than units
      for (int r = threadIdx.x; r < rows; r += kThreads) own_ml[r] = make_float2(kMinusInf, 0.0f);
    }
    cluster_sync();
    const int vecs = rows * (kD / 4), end = vecs * (rank + 1) / p.cluster;
    const uint32_t rows_at = smem_addr(own_rows), ml_at = smem_addr(own_ml), exact_at = smem_addr(own_exact);
    for (int i = vecs * rank / p.cluster + static_cast<int>(threadIdx.x); i < end; i += kThreads) {
      const int r = i / (kD / 4), d = i % (kD / 4);
      float2 ml[kMaxCluster];
      float top = kMinusInf;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        ml[c] = c < p.cluster ? load_cluster2(in_cta(ml_at + 8 * r, c)) : make_float2(kMinusInf, 0.0f);
        top = fmaxf(top, ml[c].x);
      }
      const float ref = top == kMinusInf ? 0.0f : top;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float sum = 0.0f, all = 0.0f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        if (!(ml[c].y == 0.0f)) {  // a CTA that saw nothing may have left its rows unwritten (NaN: it saw something)
          const float f = exp2_approx(ml[c].x - ref);
          const float4 v = load_cluster4(in_cta(rows_at + 16 * i, c));
          sum = fmaf(ml[c].y, f, sum);
          if constexpr (kLse) all = fmaf(load_cluster1(in_cta(exact_at + 4 * r, c)), f, all);
          acc.x = fmaf(v.x, f, acc.x);
          acc.y = fmaf(v.y, f, acc.y);
          acc.z = fmaf(v.z, f, acc.z);
          acc.w = fmaf(v.w, f, acc.w);
        }
      }
      store_row(p, cur.s.q_base, cur.kv_head, cur.row0 + r, 4 * d, acc, top, sum, all);
    }
    cluster_sync();  // nobody leaves while others read its memory
  }
}

// Joins the parts of the tiles that several CTAs of the first kernel shared.  The blocks of the CTAs that shared a tile
// share its join too (one long sequence leaves a few tiles of many parts each): each takes some of the output's 16-byte
// vectors, with up to kGroups groups of threads that take every kGroups-th part, kAhead loads in flight.
constexpr int kGroups = 8, kAhead = 4;

struct RunningSum {
  float top, sum, exact;
  float4 acc;
  __device__ __forceinline__ void move_to(float ref) {  // ref not below top
    const float f = exp2_approx(top - (ref == kMinusInf ? 0.0f : ref));
    top = ref;
    sum *= f;
    exact *= f;
    acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
  }
  __device__ __forceinline__ void add(float m, float l, float all, float4 v) {  // m not above top
    const float f = exp2_approx(m - (top == kMinusInf ? 0.0f : top));
    sum = fmaf(l, f, sum);
    exact = fmaf(all, f, exact);
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
  }
};

template <int kD, int kNT>
__global__ void __launch_bounds__(kJoinThreads) kv_attention_join_kernel(const KvAttentionParams p) {
  constexpr int kRows = 8 * kNT, kVecs = kD / 4;
  __shared__ float4 group_acc[kJoinThreads];
  __shared__ float2 group_ml[kJoinThreads];
  __shared__ float group_exact[kJoinThreads];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Split* splits = static_cast<const Split*>(p.workspace);
  const float* parts = reinterpret_cast<const float*>(static_cast<const char*>(p.workspace) + p.parts_offset);
  const int cta = static_cast<int>(blockIdx.x);
  fill_rest<kD>(p, kJoinThreads);
  // half of the threads take the tile that this CTA continued, half the one that it began
  constexpr int kThreadsOfRole = kJoinThreads / 2;
  const int role = static_cast<int>(threadIdx.x) / kThreadsOfRole, thread = static_cast<int>(threadIdx.x) % kThreadsOfRole;
  float4* const role_acc = group_acc + role * kThreadsOfRole;
  float2* const role_ml = group_ml + role * kThreadsOfRole;
  float* const role_exact = group_exact + role * kThreadsOfRole;
  const auto sync = [&]() {
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(1 + role), "n"(kThreadsOfRole) : "memory");
  };
  const SharedTile sp = splits[cta].role[role];
  if (sp.first_cta >= 0) {
    const int first = sp.first_cta;
    const int count = sp.last_cta - first + 1;
    // the beginning of the tile is part 1 of its CTA, what follows is part 0 of the next ones
    const auto part = [&](int i) { return parts + (2ll * (first + i) + (i == 0 ? 1 : 0)) * part_floats<kRows, kD>(); };
    const int vecs = sp.rows * kVecs;  // of the tile; this block's:
    const int begin = static_cast<int>(static_cast<long long>(vecs) * (cta - first) / count);
    const int end = static_cast<int>(static_cast<long long>(vecs) * (cta - first + 1) / count);
    for (int at = begin; at < end; at += kThreadsOfRole) {
      const int n = min(end - at, kThreadsOfRole);
      const int groups = min(min(kThreadsOfRole / n, kGroups), count);
      const int group = thread / n, vec = at + thread % n;
      const int r = vec / kVecs, d = vec % kVecs;
      RunningSum run = {kMinusInf, 0.0f, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
      if (group < groups) {
        for (int c0 = group; c0 < count; c0 += groups * kAhead) {
          float2 ml[kAhead];
          float all[kAhead];
          float4 v[kAhead];
#pragma unroll
          for (int x = 0; x < kAhead; ++x) {
            const int c = c0 + x * groups;
            ml[x] = make_float2(kMinusInf, 0.0f);
            v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            all[x] = 0.0f;
            if (c < count) {
              ml[x] = *reinterpret_cast<const float2*>(part(c) + kRows * kD + 2 * r);
              if (p.lse != nullptr) all[x] = part(c)[kRows * (kD + 2) + r];
              v[x] = reinterpret_cast<const float4*>(part(c))[vec];
            }
          }
          float ref = run.top;
#pragma unroll
          for (int x = 0; x < kAhead; ++x) ref = fmaxf(ref, ml[x].x);
          run.move_to(ref);
#pragma unroll
          for (int x = 0; x < kAhead; ++x) run.add(ml[x].x, ml[x].y, all[x], v[x]);
        }
      }
      if (groups > 1) {
        role_acc[thread] = run.acc;
        role_ml[thread] = make_float2(run.top, run.sum);
        role_exact[thread] = run.exact;
        sync();
      }
      if (group == 0) {
        float ref = run.top;
        for (int x = 1; x < groups; ++x) ref = fmaxf(ref, role_ml[thread + x * n].x);
        run.move_to(ref);
        for (int x = 1; x < groups; ++x) {
          const float2 ml = role_ml[thread + x * n];
          run.add(ml.x, ml.y, role_exact[thread + x * n], role_acc[thread + x * n]);
        }
        store_row(p, sp.q_base, sp.kv_head, sp.row0 + r, 4 * d, run.acc, run.top, run.sum, run.exact);
      }
      if (groups > 1) sync();
    }
  }
}

constexpr int kSmallUnits = 4;
constexpr int kClusterSizes = 4;  // 1, 2, 4, 8

// What the current device holds at once, per device (the same whoever asks first): CTAs of the list's kernel, and of the
// other one in clusters of 1 << i.
struct Residency {
  std::atomic<int> ctas{0}, clustered[kClusterSizes] = {};
};
struct Plan {
  int ctas;
  int clustered[kClusterSizes];
  size_t parts_offset, bytes;
};

cudaLaunchConfig_t cluster_config(cudaLaunchAttribute* attr, long long ctas, int cluster, int smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  *attr = {};
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = static_cast<unsigned>(cluster);
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

template <int kD, int kNT, int kSub>
cudaError_t make_plan(Plan* plan) {
  using S = Shape<kD, kNT, kSub>;
  static Residency per_device[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  Residency& known = per_device[dev];
  int ctas = known.ctas.load();
  if (ctas == 0) {
    const auto kernel = kv_attention_kernel<kD, kNT, kSub, false, false>;
    int sms = 0, per_sm = 0;
    err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (err != cudaSuccess) return err;
    const auto allow = [](const void* f, int smem) { return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); };
    const auto address = [](auto f) { return reinterpret_cast<const void*>(f); };
    if ((err = allow(address(kernel), S::kSmemBytes)) != cudaSuccess) return err;
    if ((err = allow(address(kv_attention_kernel<kD, kNT, kSub, false, true>), S::kSmemBytes)) != cudaSuccess) return err;
    if ((err = allow(address(kv_attention_kernel<kD, kNT, kSub, true, false>), S::kClusteredSmemBytes)) != cudaSuccess) return err;
    if ((err = allow(address(kv_attention_kernel<kD, kNT, kSub, true, true>), S::kClusteredSmemBytes)) != cudaSuccess) return err;
    err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, S::kSmemBytes);
    if (err != cudaSuccess) return err;
    if (per_sm < 1) return cudaErrorInvalidConfiguration;
    for (int i = 0; i < kClusterSizes; ++i) {
      int clusters = 0;
      cudaLaunchAttribute attr;
      const cudaLaunchConfig_t cfg = cluster_config(&attr, 1 << i, 1 << i, S::kClusteredSmemBytes, nullptr);
      err = cudaOccupancyMaxActiveClusters(&clusters, kv_attention_kernel<kD, kNT, kSub, true, false>, &cfg);
      if (err != cudaSuccess) return err;
      known.clustered[i] = clusters << i;
    }
    ctas = sms * per_sm;
    known.ctas = ctas;
  }
  plan->ctas = ctas;
  for (int i = 0; i < kClusterSizes; ++i) plan->clustered[i] = known.clustered[i].load();
  plan->parts_offset = (static_cast<size_t>(ctas) * sizeof(Split) + 255) / 256 * 256;
  plan->bytes = plan->parts_offset + 2 * static_cast<size_t>(ctas) * part_floats<S::kRows, kD>() * sizeof(float);
  return cudaSuccess;
}

template <int kD, int kNT, int kSub>
cudaError_t run_t(const KvAttentionParams& params, size_t* bytes, cudaStream_t stream) {
  using S = Shape<kD, kNT, kSub>;
  Plan plan;
  cudaError_t err = make_plan<kD, kNT, kSub>(&plan);
  if (err != cudaSuccess) return err;
  KvAttentionParams p = params;
  // A cluster per tile when all of them are resident at once and the largest context that the block table allows leaves a
  // CTA at most kSmallUnits units, up to 8 CTAs a tile.  It saves the second launch, the workspace and the list, about 2 us
  // on the device and 5 on the host, but shares nothing between tiles.  Device us, list / clusters: 1 sequence of 1024
  // tokens, 8 kv heads 8.0 / 5.9, of 4096 9.3 / 10.0 (4 units a CTA; the host takes 15.9 / 10.6), of 8192 11.1 / 14.8;
  // 16 of 1024 13.6 / 12.4, of 2048 18.4 / 17.8 (ragged 14.3 / 17.5); 64 of 256, two waves, 14.7 / 17.8.  What is resident
  // is asked of the clusters' own kernel, which needs more shared memory: 16 rows of 128 or 8 of 256 leave room for two of its
  // blocks an SM where the list's has three.  5 sequences of 1024 tokens, 8 kv heads with 16 query heads each: clusters of 4,
  // 10.8 us; clusters of 8 in two waves, by the list's figure, 16.6.
  const long long row_slots = p.cu_seqlens == nullptr ? static_cast<long long>(p.batch) * ((p.group + S::kRows - 1) / S::kRows)
                                                      : static_cast<long long>(p.tokens) * p.group / S::kRows + p.batch;
  const long long tiles = row_slots * p.kv_heads, units = p.max_len > S::kUnit ? (p.max_len + S::kUnit - 1) / S::kUnit : 1;
  int size = kClusterSizes - 1;
  while (size > 0 && (tiles << size > plan.clustered[size] || (1 << size) / 2 >= units)) --size;
  p.cluster = 1 << size;
  const bool clustered = tiles << size <= plan.clustered[size] && units <= kSmallUnits * p.cluster;
  if (bytes != nullptr) {  // only asked for the size
    *bytes = clustered ? 0 : plan.bytes;
    return cudaSuccess;
  }
  if (clustered) {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = cluster_config(&attr, tiles * p.cluster, p.cluster, S::kClusteredSmemBytes, stream);
    return cudaLaunchKernelEx(&cfg, p.lse != nullptr ? kv_attention_kernel<kD, kNT, kSub, true, true> : kv_attention_kernel<kD, kNT, kSub, true, false>, p);
  }
  if (params.workspace_bytes < plan.bytes) return cudaErrorMemoryAllocation;
  p.parts_offset = plan.parts_offset;
  if (p.lse != nullptr) {
    kv_attention_kernel<kD, kNT, kSub, false, true><<<plan.ctas, kThreads, S::kSmemBytes, stream>>>(p);
  } else {
    kv_attention_kernel<kD, kNT, kSub, false, false><<<plan.ctas, kThreads, S::kSmemBytes, stream>>>(p);
  }
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  // may be resident before the first kernel has ended; it waits for it (griddepcontrol.wait)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan.ctas));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_attention_join_kernel<kD, kNT>, p);
}

template <int kD, int kSub>
cudaError_t run_rows(const KvAttentionParams& p, size_t* bytes, cudaStream_t stream) {
  // query rows that share a kv head, in an average sequence
  const long long rows = p.cu_seqlens == nullptr ? p.group : (static_cast<long long>(p.tokens) * p.group + p.batch - 1) / (p.batch > 0 ? p.batch : 1);
  // 16 rows a tile (168 registers, three blocks an SM) beat 32 rows, which convert the codes half as often but leave room
  // for two blocks: 32 requests of 1 to 6 tokens, 8 heads a kv head, 103 us against 119 (8 rows: 124).
  return rows <= 8 ? run_t<kD, 1, kSub>(p, bytes, stream) : run_t<kD, 2, kSub>(p, bytes, stream);
}

}  // namespace

cudaError_t launch_kv_attention(const KvAttentionParams& p, size_t* bytes, cudaStream_t stream) {
  if (p.dim == 64) return p.page_size >= 32 ? run_rows<64, 32>(p, bytes, stream) : run_rows<64, 16>(p, bytes, stream);
  if (p.dim == 128) return p.page_size >= 32 ? run_rows<128, 32>(p, bytes, stream) : run_rows<128, 16>(p, bytes, stream);
  return run_rows<256, 16>(p, bytes, stream);
}

}  // namespace b200fp8
