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
//   * e4m3 is exact in fp16, and so are bf16 queries once a row is scaled by a power of two (what falls below fp16's
//     range then is under 2^-24 of the row's largest element); p <= 1 rounded to fp16 is off by 2^-12.  tcgen05 takes
//     8-bit operands only in pairs, which would round queries and p to 3 bits of mantissa.  Sums, maxima and the
//     output stay in fp32.
//   * The order of the contraction is free, so a thread's operand elements are 16 neighbouring bytes of a token:
//     whole 16-byte vectors are loaded, and the pairing of two tokens' V bytes costs one byte permute per 4 bytes.
//     Nothing is transposed through shared memory, and a thread reads only vectors that it copied itself (cp.async,
//     [stage][vector][lane]): the ring needs no barrier and has no bank conflict.
//   * v_scale differs by page and is applied in fp32 when a chunk's product is added to O, together with the
//     rescaling that a new maximum asks for.
// Work is split over the context: all (sequence, kv head, row tile, unit of 4 chunks) units of the batch are one list,
// cut into equal runs for a grid that fills the GPU once; lengths are read on the device.  A run that ends inside a
// tile leaves its unnormalised sums in the workspace (at most two parts a CTA) and the second kernel joins them, in a
// fixed order.  The workspace needs no initialisation and nothing is kept in it between calls.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "rotary.cuh"

namespace b200fp8 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kJoinThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kNoPage = 0xffffffffu;  // in place of a chunk's k_scale: its page is not in the cache

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool take) {  // zeros where not taken
  const int n = take ? kBytes : 0;
  if constexpr (kBytes == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes), "r"(n) : "memory");
  }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
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
__device__ __forceinline__ float exp2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ bool has_nan_code(uint32_t w) {  // any byte 0x7f or 0xff
  const uint32_t m = (w & 0x7f7f7f7fu) + 0x01010101u;
  return (m & 0x80808080u) != 0;
}

// ------------------------------------------------------------------ the list of units
struct Seq {
  int n;          // new tokens
  int len;        // context, the new tokens included
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
  s.len = min(max(p.seq_lens[b], 0), p.max_len);
  s.row_tiles = static_cast<int>((static_cast<long long>(s.n) * p.group + kRows - 1) / kRows);
  s.units = max((s.len + kUnit - 1) / kUnit, 1);
  return s;
}
template <int kRows, int kUnit>
__device__ __forceinline__ long long units_of(const KvAttentionParams& p, int b) {
  const Seq s = seq_of<kRows, kUnit>(p, b);
  return static_cast<long long>(s.row_tiles) * p.kv_heads * s.units;
}

// A place in the list: unit `unit` of tile `tile` (kv head, row tile) of sequence b.
template <int kRows, int kUnit>
struct Cursor {
  Seq s;
  int b, tile, unit;
  // of the tile
  int kv_head, row0;
  int min_end, max_end;  // tokens that the tile's first and last query see: [0, end)

  __device__ __forceinline__ void enter_tile(const KvAttentionParams& p) {
    kv_head = tile / s.row_tiles;
    row0 = (tile - kv_head * s.row_tiles) * kRows;
    const int last_row = min(row0 + kRows, s.n * p.group) - 1;
    const int begin = s.len - s.n;
    min_end = max(begin + row0 / p.group + 1, 0);
    max_end = max(begin + last_row / p.group + 1, 0);
  }
  __device__ __forceinline__ void enter_sequence(const KvAttentionParams& p) {
    s = seq_of<kRows, kUnit>(p, b);
  }
  __device__ __forceinline__ void advance(const KvAttentionParams& p, long long left) {
    if (++unit < s.units) return;
    if (left <= 0) return;  // the run ends here
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

template <int kD, int kNT, int kChunk, int kStages>
struct Shape {
  static constexpr int kRows = 8 * kNT;
  static constexpr int kUnit = kWarps * kChunk;
  static constexpr int kMT = kChunk / 16;
  static constexpr int kKVecs = (kChunk / 8) * (kD / 64);  // 16-byte vectors of K a lane has of a chunk
  static constexpr int kVBytes = kD >= 128 ? 16 : 8;       // a lane's vector of V
  static constexpr int kVH = kD >= 128 ? kD / 128 : 1;     // vectors of V per token
  static constexpr int kVVecs = (kChunk / 4) * kVH;
  static constexpr int kStageBytes = 32 * (16 * kKVecs + kVBytes * kVVecs + 8);
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kPitch = kD + 4;  // floats of a row of the warps' partial O
  static constexpr int kMergeBytes = kWarps * kRows * kPitch * 4 + kWarps * kRows * 2 * 4;
  static constexpr int kSmemBytes = kRingBytes + kMergeBytes;
};

// part of a tile in the workspace: O [kRows][kD], then (max, sum) [kRows][2]
template <int kRows, int kD>
__host__ __device__ constexpr size_t part_floats() { return static_cast<size_t>(kRows) * (kD + 2); }

struct Split {  // a tile that CTA c began and did not finish
  int last_cta;  // the CTA that finishes it; -1: none
  int b, tile;
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

// Four elements of an output row from its sums, and the row's log-sum-exp (once, with the row's first elements).
__device__ __forceinline__ void store_row(const KvAttentionParams& p, const Seq& s, int kv_head, int row, int d, float4 acc,
                                          float top, float sum) {
  const int token = row / p.group;
  const int head = kv_head * p.group + row - token * p.group;
  const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);  // no token seen: zeros
  uint16_t* at = static_cast<uint16_t*>(p.out) + (s.q_base + static_cast<long long>(token)) * p.o_token + head * p.o_head + d;
  *reinterpret_cast<uint2*>(at) = make_uint2(pack_out2(acc.x * inv, acc.y * inv, p.fp16), pack_out2(acc.z * inv, acc.w * inv, p.fp16));
  if (p.lse != nullptr && d == 0) {
    p.lse[(s.q_base + static_cast<long long>(token)) * p.heads + head] = (top + log2f(sum)) * kLn2;
  }
}

template <int kD, int kNT, int kChunk, int kStages>
__global__ void __launch_bounds__(kThreads) kv_attention_kernel(const KvAttentionParams p) {
  using S = Shape<kD, kNT, kChunk, kStages>;
  using C = Cursor<S::kRows, S::kUnit>;
  extern __shared__ uint4 smem[];
  __shared__ long long sums[kWarps];
  __shared__ long long found_before;
  __shared__ int found_b;
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int g = lane >> 2, t = lane & 3;
  const int cta = static_cast<int>(blockIdx.x);
  Split* splits = static_cast<Split*>(p.workspace);
  float* parts = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + p.parts_offset);

  // ---- this CTA's run of units
  long long mine = 0;
  for (int b = threadIdx.x; b < p.batch; b += kThreads) mine += units_of<S::kRows, S::kUnit>(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += sums[w];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join waits for this grid to complete
  // no more CTAs than units: every one of them then has a part in what it touches, which the join relies on
  const int ctas = static_cast<int>(min(total, static_cast<long long>(gridDim.x)));
  const long long run_begin = cta < ctas ? total * cta / ctas : total;
  const long long run_end = cta < ctas ? total * (cta + 1) / ctas : total;
  if (run_begin >= run_end) {
    if (threadIdx.x == 0) splits[cta].last_cta = -1;
    return;
  }
  long long before = 0;  // units of the sequences in front of b0
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    const long long own = b < p.batch ? units_of<S::kRows, S::kUnit>(p, b) : 0;
    long long upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();  // sums of the step before have been read
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long step = 0;
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
  __syncthreads();

  C cur;
  cur.b = found_b;
  cur.enter_sequence(p);
  {
    const long long in_seq = run_begin - found_before;
    cur.tile = static_cast<int>(in_seq / cur.s.units);
    cur.unit = static_cast<int>(in_seq - static_cast<long long>(cur.tile) * cur.s.units);
  }
  cur.enter_tile(p);
  C ahead = cur;
  long long ahead_at = run_begin;

  // ---- the ring: each lane copies what it will read
  const uint32_t ring = smem_addr(smem) + static_cast<uint32_t>(warp * kStages * S::kStageBytes);
  const uint32_t k_off = lane * 16;
  const uint32_t v_off = 32 * 16 * S::kKVecs + lane * S::kVBytes;
  const uint32_t s_off = 32 * (16 * S::kKVecs + S::kVBytes * S::kVVecs) + lane * 8;
  float* merge = reinterpret_cast<float*>(reinterpret_cast<char*>(smem) + S::kRingBytes);
  float* merge_ml = merge + kWarps * S::kRows * S::kPitch;

  int next_page = -1;  // page of the chunk that is requested next, loaded one step early
  const auto look_up = [&]() {
    next_page = -1;
    if (ahead_at < run_end) {
      const int token0 = ahead.unit * S::kUnit + warp * kChunk;
      if (token0 < ahead.max_end) next_page = p.block_table[ahead.b * p.bt_stride + (token0 >> p.page_shift)];
    }
  };
  const auto request = [&](int stage) {  // one group a call, also when there is nothing to request
    if (ahead_at < run_end) {
      const int token0 = ahead.unit * S::kUnit + warp * kChunk;
      if (token0 < ahead.max_end) {
        const uint32_t base = ring + stage * S::kStageBytes;
        const bool there = next_page >= 0 && next_page < p.num_pages;
        const long long page = there ? next_page : 0;
        const int row0 = token0 & (p.page_size - 1);
        const uint8_t* k = p.k_cache + page * p.k_page + ahead.kv_head * p.k_head + row0 * p.k_row;
        const uint8_t* v = p.v_cache + page * p.v_page + ahead.kv_head * p.v_head + row0 * p.v_row;
#pragma unroll
        for (int i = 0; i < kChunk / 8; ++i) {
          const bool take = there && token0 + 8 * i + g < ahead.max_end;
          const uint8_t* row = k + (8 * i + g) * p.k_row + 16 * t;
#pragma unroll
          for (int j = 0; j < kD / 64; ++j) {
            copy_async<16>(base + k_off + (i * (kD / 64) + j) * 512, take ? row + 64 * j : p.k_cache, take);
          }
        }
#pragma unroll
        for (int i = 0; i < kChunk / 4; ++i) {  // tokens 2t, 2t + 1, 2t + 8, 2t + 9 of every 16
          const int token = 16 * (i / 4) + 2 * t + (i & 1) + 8 * ((i >> 1) & 1);
          const bool take = there && token0 + token < ahead.max_end;
          const uint8_t* row = v + token * p.v_row + S::kVBytes * g;
#pragma unroll
          for (int h = 0; h < S::kVH; ++h) {
            copy_async<S::kVBytes>(base + v_off + (i * S::kVH + h) * 32 * S::kVBytes, take ? row + 128 * h : p.v_cache, take);
          }
        }
        if (there) {
          copy_async<4>(base + s_off, p.k_scale + page * p.ks_page + ahead.kv_head * p.ks_head, true);
          copy_async<4>(base + s_off + 4, p.v_scale + page * p.vs_page + ahead.kv_head * p.vs_head, true);
        } else {
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(base + s_off), "r"(kNoPage) : "memory");
        }
      }
      ++ahead_at;
      ahead.advance(p, run_end - ahead_at);
    }
    copy_commit();
    look_up();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) request(s);

  int stage = 0;
  long long at = run_begin;
  if (threadIdx.x == 0) splits[cta].last_cta = -1;
  while (at < run_end) {
    // ---- a segment: the units of this run that belong to one tile
    const int unit0 = cur.unit;
    const int unit_end = static_cast<int>(min(static_cast<long long>(cur.s.units), unit0 + (run_end - at)));
    const int rows = min(S::kRows, cur.s.n * p.group - cur.row0);
    // queries: column 8 nt + g, elements 64 j + 16 t .. + 15
    uint32_t qf[kNT][kD / 64][8];
    float col_scale[kNT][2];
    int col_end[kNT][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const int r = 8 * nt + g;
      float x[kD / 64][16];
      float big = 0.0f;
      const bool real = r < rows;
      const int row = cur.row0 + (real ? r : 0);
      const int token = row / p.group;
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + (cur.s.q_base + static_cast<long long>(token)) * p.q_token +
                          (cur.kv_head * p.group + row - token * p.group) * p.q_head + 16 * t;
#pragma unroll
      for (int j = 0; j < kD / 64; ++j) {
        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
        if (real) {
          lo = *reinterpret_cast<const uint4*>(q + 64 * j);
          hi = *reinterpret_cast<const uint4*>(q + 64 * j + 8);
        }
        float a[8], b[8];
        unpack_q(lo, p.fp16, a);
        unpack_q(hi, p.fp16, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[j][i] = a[i];
          x[j][8 + i] = b[i];
          big = fmaxf(big, fmaxf(fabsf(a[i]), fabsf(b[i])));
        }
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // 2^-e with the row's largest element in [1, 2); rows of zeros, and with infinities, as they are
      int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
      e = big > 0.0f && e < 128 ? max(min(e, 126), -126) : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int j = 0; j < kD / 64; ++j) {
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[nt][j][i] = half2_of(x[j][2 * i] * down, x[j][2 * i + 1] * down);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        col_scale[nt][c] = __shfl_sync(0xffffffffu, up, (2 * t + c) * 4) * (p.softmax_scale * kLog2e);
        const int rc = 8 * nt + 2 * t + c;
        col_end[nt][c] = rc < rows ? cur.s.len - cur.s.n + (cur.row0 + rc) / p.group + 1 : 0;
      }
    }
    float o[S::kVH][kD >= 128 ? 8 : 4][kNT][4];
    constexpr int kOT = kD >= 128 ? 8 : 4;  // 16-row tiles of O^T per vector of V
#pragma unroll
    for (int h = 0; h < S::kVH; ++h)
#pragma unroll
      for (int i = 0; i < kOT; ++i)
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[h][i][nt][c] = 0.0f;
    float m[kNT][2], l[kNT][2];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      m[nt][0] = m[nt][1] = __int_as_float(0xff800000);
      l[nt][0] = l[nt][1] = 0.0f;
    }

    for (int unit = unit0; unit < unit_end; ++unit) {
      request(stage == 0 ? kStages - 1 : stage - 1);  // into the stage that was emptied one step ago
      copy_wait<kStages - 1>();
      const uint32_t base = ring + stage * S::kStageBytes;
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const int token0 = unit * S::kUnit + warp * kChunk;
      if (token0 >= cur.max_end) continue;
      const uint2 sc = lds8(base + s_off);
      if (sc.x == kNoPage) continue;
      const float k_scale = __uint_as_float(sc.x), v_scale = __uint_as_float(sc.y);

      // ---- S^T = K Q^T
      float s[S::kMT][kNT][4];
#pragma unroll
      for (int mt = 0; mt < S::kMT; ++mt) {
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < kD / 64; ++j) {
          const uint4 ka = lds16(base + k_off + ((2 * mt) * (kD / 64) + j) * 512);
          const uint4 kb = lds16(base + k_off + ((2 * mt + 1) * (kD / 64) + j) * 512);
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            halves_of(wa[i], a0, a2);
            halves_of(wb[i], a1, a3);
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt) mma16816(s[mt][nt], a0, a1, a2, a3, qf[nt][j][2 * i], qf[nt][j][2 * i + 1]);
          }
        }
      }
      // ---- softmax over the tokens, column by column
      const bool partial = token0 + kChunk > cur.min_end;
      float alpha[kNT][2];
      uint32_t pf[S::kMT][kNT][2];
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        const float f0 = col_scale[nt][0] * k_scale, f1 = col_scale[nt][1] * k_scale;
        float top0 = m[nt][0], top1 = m[nt][1];
#pragma unroll
        for (int mt = 0; mt < S::kMT; ++mt) {
          s[mt][nt][0] *= f0;
          s[mt][nt][1] *= f1;
          s[mt][nt][2] *= f0;
          s[mt][nt][3] *= f1;
          if (partial) {
            const int token = token0 + 16 * mt + g;
            if (token >= col_end[nt][0]) s[mt][nt][0] = __int_as_float(0xff800000);
            if (token >= col_end[nt][1]) s[mt][nt][1] = __int_as_float(0xff800000);
            if (token + 8 >= col_end[nt][0]) s[mt][nt][2] = __int_as_float(0xff800000);
            if (token + 8 >= col_end[nt][1]) s[mt][nt][3] = __int_as_float(0xff800000);
          }
          top0 = fmaxf(top0, fmaxf(s[mt][nt][0], s[mt][nt][2]));
          top1 = fmaxf(top1, fmaxf(s[mt][nt][1], s[mt][nt][3]));
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, x));
          top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, x));
        }
        // a column without a token so far: any finite reference will do
        const float ref0 = top0 == __int_as_float(0xff800000) ? 0.0f : top0;
        const float ref1 = top1 == __int_as_float(0xff800000) ? 0.0f : top1;
        alpha[nt][0] = exp2_approx(m[nt][0] - ref0);
        alpha[nt][1] = exp2_approx(m[nt][1] - ref1);
        m[nt][0] = top0;
        m[nt][1] = top1;
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int mt = 0; mt < S::kMT; ++mt) {
          const float p0 = exp2_approx(s[mt][nt][0] - ref0), p1 = exp2_approx(s[mt][nt][1] - ref1);
          const float p2 = exp2_approx(s[mt][nt][2] - ref0), p3 = exp2_approx(s[mt][nt][3] - ref1);
          sum0 += p0 + p2;
          sum1 += p1 + p3;
          pf[mt][nt][0] = transpose8x8(half2_of(p0, p1));
          pf[mt][nt][1] = transpose8x8(half2_of(p2, p3));
        }
        l[nt][0] = l[nt][0] * alpha[nt][0] + sum0;
        l[nt][1] = l[nt][1] * alpha[nt][1] + sum1;
      }
      // ---- O^T += V^T P^T.  `end`: V counts as zero from this token on (kChunk and more: all of it counts)
      const auto product = [&](auto cut, int end, auto takes) {
#pragma unroll
        for (int h = 0; h < S::kVH; ++h) {
          constexpr int kW = S::kVBytes / 4;
          uint32_t w[S::kMT][4][kW];
#pragma unroll
          for (int mt = 0; mt < S::kMT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a = base + v_off + ((4 * mt + i) * S::kVH + h) * 32 * S::kVBytes;
              if constexpr (kW == 4) {
                const uint4 v = lds16(a);
                w[mt][i][0] = v.x, w[mt][i][1] = v.y, w[mt][i][2] = v.z, w[mt][i][3] = v.w;
              } else {
                const uint2 v = lds8(a);
                w[mt][i][0] = v.x, w[mt][i][1] = v.y;
              }
              if constexpr (decltype(cut)::value) {
                if (16 * mt + 2 * t + (i & 1) + 8 * (i >> 1) >= end) {
#pragma unroll
                  for (int c = 0; c < kW; ++c) w[mt][i][c] = 0u;
                }
              }
            }
#pragma unroll
          for (int c = 0; c < kW; ++c) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float d[kNT][4];
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt) d[nt][0] = d[nt][1] = d[nt][2] = d[nt][3] = 0.0f;
#pragma unroll
              for (int mt = 0; mt < S::kMT; ++mt) {
                const uint32_t pick = half == 0 ? 0x5140u : 0x7362u;  // bytes 2 half, 2 half + 1 of two tokens, interleaved
                uint32_t a0, a1, a2, a3;
                halves_of(__byte_perm(w[mt][0][c], w[mt][1][c], pick), a0, a1);
                halves_of(__byte_perm(w[mt][2][c], w[mt][3][c], pick), a2, a3);
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt) mma16816(d[nt], a0, a1, a2, a3, pf[mt][nt][0], pf[mt][nt][1]);
              }
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float& acc = o[h][2 * c + half][nt][e];
                  if (takes(nt, e & 1)) acc = fmaf(acc, alpha[nt][e & 1], d[nt][e] * v_scale);
                }
            }
          }
        }
      };
      bool strange = false;
      if (partial && cur.min_end < cur.max_end) {
        // Tokens of this chunk that some columns see and others do not: their p is zero there, but zero times NaN is
        // NaN.  Look whether such a token has a NaN (or its page a scale that is not finite).
        bool bad = !(fabsf(v_scale) <= 3.402823466e38f);
#pragma unroll
        for (int i = 0; i < S::kVVecs; ++i) {
          const uint32_t a = base + v_off + i * 32 * S::kVBytes;
          const uint2 v = lds8(a);
          bad |= has_nan_code(v.x) || has_nan_code(v.y);
          if constexpr (S::kVBytes == 16) {
            const uint2 u = lds8(a + 8);
            bad |= has_nan_code(u.x) || has_nan_code(u.y);
          }
        }
        strange = __any_sync(0xffffffffu, bad);
      }
      if (!strange) {
        product(std::false_type{}, 0, [](int, int) { return true; });
      } else {
        // once for every place where a column's context can end in this chunk, with V cut there
        const int lo = max(cur.min_end - token0, 0), hi = min(cur.max_end - token0, kChunk);
        for (int end = lo; end <= hi; ++end) {
          product(std::true_type{}, end, [&](int nt, int c) {
            return end > 0 && min(max(col_end[nt][c] - token0, 0), kChunk) == end;
          });
        }
        // columns that see nothing of the chunk keep their sums: alpha is one there, unless they have seen nothing yet
      }
    }

    // ---- join the warps
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
        const int r = 8 * nt + 2 * t + c;
        float* row = merge + (warp * S::kRows + r) * S::kPitch;
#pragma unroll
        for (int h = 0; h < S::kVH; ++h) {
          constexpr int kPer = S::kVBytes;  // elements of the head dimension that a lane has in a row
          float* d = row + 128 * h + kPer * g;
#pragma unroll
          for (int i = 0; i < kOT; i += 2) {
            *reinterpret_cast<float4*>(d + 2 * i) =
                make_float4(o[h][i][nt][c], o[h][i][nt][2 + c], o[h][i + 1][nt][c], o[h][i + 1][nt][2 + c]);
          }
        }
        if (g == 0) {
          merge_ml[(warp * S::kRows + r) * 2] = m[nt][c];
          merge_ml[(warp * S::kRows + r) * 2 + 1] = l[nt][c];
        }
      }
    __syncthreads();
    const bool begins = unit0 == 0, ends = unit_end == cur.s.units;
    float* part = parts + (2ll * cta + (begins ? 1 : 0)) * part_floats<S::kRows, kD>();
    for (int i = threadIdx.x; i < rows * (kD / 4); i += kThreads) {
      const int r = i / (kD / 4), d = (i - r * (kD / 4)) * 4;
      float top = merge_ml[r * 2];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, merge_ml[(w * S::kRows + r) * 2]);
      const float ref = top == __int_as_float(0xff800000) ? 0.0f : top;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_approx(merge_ml[(w * S::kRows + r) * 2] - ref);
        const float4 v = *reinterpret_cast<const float4*>(merge + (w * S::kRows + r) * S::kPitch + d);
        sum = fmaf(merge_ml[(w * S::kRows + r) * 2 + 1], f, sum);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
      }
      if (begins && ends) {
        store_row(p, cur.s, cur.kv_head, cur.row0 + r, d, acc, top, sum);
      } else {
        *reinterpret_cast<float4*>(part + r * kD + d) = acc;
        if (d == 0) {
          part[S::kRows * kD + 2 * r] = top;
          part[S::kRows * kD + 2 * r + 1] = sum;
        }
      }
    }
    if (begins && !ends && threadIdx.x == 0) {
      const long long tile_end = at + (cur.s.units - unit0);  // unit0 is 0: one past the tile's last unit
      splits[cta].last_cta = static_cast<int>((tile_end * ctas - 1) / total);
      splits[cta].b = cur.b;
      splits[cta].tile = cur.tile;
    }
    __syncthreads();  // the warps' sums have been read
    at += unit_end - unit0;
    cur.unit = unit_end - 1;
    cur.advance(p, run_end - at);
  }
  copy_wait<0>();
}

// Joins the parts of the tile that CTA blockIdx.x of the first kernel began and others finished.
template <int kD, int kNT, int kChunk>
__global__ void __launch_bounds__(kJoinThreads) kv_attention_join_kernel(const KvAttentionParams p) {
  constexpr int kRows = 8 * kNT, kUnit = kWarps * kChunk;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Split* splits = static_cast<const Split*>(p.workspace);
  const float* parts = reinterpret_cast<const float*>(static_cast<const char*>(p.workspace) + p.parts_offset);
  const int cta = static_cast<int>(blockIdx.x);
  if (p.cu_seqlens != nullptr && (p.fill_rest || p.lse != nullptr)) {  // rows behind the last sequence
    const int used = min(max(p.cu_seqlens[p.batch], 0), p.tokens);
    const long long n = static_cast<long long>(p.tokens - used) * p.heads;
    for (long long r = cta; r < n; r += gridDim.x) {
      const long long token = used + r / p.heads;
      const int head = static_cast<int>(r % p.heads);
      uint16_t* o = static_cast<uint16_t*>(p.out) + token * p.o_token + head * p.o_head;
      if (p.fill_rest) {
        for (int d = threadIdx.x; d < kD; d += kJoinThreads) o[d] = 0;
      }
      if (p.lse != nullptr && threadIdx.x == 0) p.lse[token * p.heads + head] = __int_as_float(0xff800000);
    }
  }
  const Split sp = splits[cta];
  if (sp.last_cta < 0) return;
  Cursor<kRows, kUnit> cur;
  cur.b = sp.b;
  cur.tile = sp.tile;
  cur.enter_sequence(p);
  cur.enter_tile(p);
  const int rows = min(kRows, cur.s.n * p.group - cur.row0);
  const int count = sp.last_cta - cta + 1;
  // the beginning of the tile is part 1 of this CTA, what follows is part 0 of the next ones
  const auto part = [&](int i) { return parts + (2ll * (cta + i) + (i == 0 ? 1 : 0)) * part_floats<kRows, kD>(); };
  for (int i = threadIdx.x; i < rows * (kD / 4); i += kJoinThreads) {
    const int r = i / (kD / 4), d = (i - r * (kD / 4)) * 4;
    float top = __int_as_float(0xff800000);
    for (int c = 0; c < count; ++c) top = fmaxf(top, part(c)[kRows * kD + 2 * r]);
    const float ref = top == __int_as_float(0xff800000) ? 0.0f : top;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
#pragma unroll 4
    for (int c = 0; c < count; ++c) {
      const float* x = part(c);
      const float f = exp2_approx(x[kRows * kD + 2 * r] - ref);
      const float4 v = *reinterpret_cast<const float4*>(x + r * kD + d);
      sum = fmaf(x[kRows * kD + 2 * r + 1], f, sum);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z);
      acc.w = fmaf(v.w, f, acc.w);
    }
    store_row(p, cur.s, cur.kv_head, cur.row0 + r, d, acc, top, sum);
  }
}

struct Plan {
  int ctas;
  size_t parts_offset, bytes;
};

// CTAs of a grid that fills the current device once, per device (the same whoever asks first)
template <int kD, int kNT, int kChunk, int kStages>
cudaError_t make_plan(Plan* plan) {
  using S = Shape<kD, kNT, kChunk, kStages>;
  static std::atomic<int> ctas_per_device[64] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  int ctas = ctas_per_device[dev].load();
  if (ctas == 0) {
    const auto kernel = kv_attention_kernel<kD, kNT, kChunk, kStages>;
    int sms = 0, per_sm = 0;
    err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (err != cudaSuccess) return err;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmemBytes);
    if (err != cudaSuccess) return err;
    err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, S::kSmemBytes);
    if (err != cudaSuccess) return err;
    if (per_sm < 1) return cudaErrorInvalidConfiguration;
    ctas = sms * per_sm;
    ctas_per_device[dev] = ctas;
  }
  plan->ctas = ctas;
  plan->parts_offset = (static_cast<size_t>(ctas) * sizeof(Split) + 255) / 256 * 256;
  plan->bytes = plan->parts_offset + 2 * static_cast<size_t>(ctas) * part_floats<S::kRows, kD>() * sizeof(float);
  return cudaSuccess;
}

template <int kD, int kNT, int kChunk, int kStages>
cudaError_t run_t(const KvAttentionParams& params, size_t* bytes, cudaStream_t stream) {
  using S = Shape<kD, kNT, kChunk, kStages>;
  Plan plan;
  cudaError_t err = make_plan<kD, kNT, kChunk, kStages>(&plan);
  if (err != cudaSuccess) return err;
  if (bytes != nullptr) {  // only asked for the size
    *bytes = plan.bytes;
    return cudaSuccess;
  }
  if (params.workspace_bytes < plan.bytes) return cudaErrorMemoryAllocation;
  KvAttentionParams p = params;
  p.parts_offset = plan.parts_offset;
  kv_attention_kernel<kD, kNT, kChunk, kStages><<<plan.ctas, kThreads, S::kSmemBytes, stream>>>(p);
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
  return cudaLaunchKernelEx(&cfg, kv_attention_join_kernel<kD, kNT, kChunk>, p);
}

template <int kD>
cudaError_t run_d(const KvAttentionParams& p, size_t* bytes, cudaStream_t stream) {
  // query rows that share a kv head, in an average sequence
  const long long rows = p.cu_seqlens == nullptr ? p.group : (static_cast<long long>(p.tokens) * p.group + p.batch - 1) / max(p.batch, 1);
  const bool wide = rows > 8;
  if (p.page_size >= 32) {
    return wide ? run_t<kD, 2, 32, 2>(p, bytes, stream) : run_t<kD, 1, 32, 2>(p, bytes, stream);
  }
  return wide ? run_t<kD, 2, 16, 3>(p, bytes, stream) : run_t<kD, 1, 16, 3>(p, bytes, stream);
}

}  // namespace

cudaError_t launch_kv_attention(const KvAttentionParams& p, size_t* bytes, cudaStream_t stream) {
  if (p.dim == 64) return run_d<64>(p, bytes, stream);
  if (p.dim == 128) return run_d<128>(p, bytes, stream);
  return run_d<256>(p, bytes, stream);
}

}  // namespace b200fp8
