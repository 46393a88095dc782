// Rotary positions of x [tokens, heads, dim] (any token and head pitch, dim contiguous), out of place or in place, and
// the transposed rotation, which is the gradient with regard to x (sin -> -sin).
//
// Bound by HBM: x in, y out, one table row per token.  A thread owns one slot (two 16-byte vectors, see rotary.cuh) of
// kHeads neighbouring heads of a token: it reads all of them before it writes any - so in place needs nothing more -
// with 2 * kHeads loads in flight that do not wait for the position and the table row, and takes its cosines and sines
// into registers once for all its heads (once per head they are twice the bytes of x, out of L1, and cost 15 %).
#include <type_traits>

#include "kernels.h"
#include "rotary.cuh"

namespace b200fp8 {
namespace {

constexpr int kThreads = 256;
constexpr long long kManyThreads = 148ll * 2048;  // one wave of one slot a thread

// kN: pairs of a slot (16 bytes of T each; 1: any alignment and any even rot).  Slots [0, rot / 2 / kN) of a head are
// rotated, the ones behind them copy 2 * kN elements each of [rot, dim).
template <typename T, int kN, bool kInterleaved, int kHeads>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  using V = typename std::conditional<kN == 1, T, uint4>::type;
  const int half = p.rot / 2;
  const int turning = half / kN;
  const int slots = turning + (p.copy_rest ? (p.dim - p.rot + 2 * kN - 1) / (2 * kN) : 0);
  const unsigned per_token = static_cast<unsigned>((p.heads + kHeads - 1) / kHeads) * static_cast<unsigned>(slots);
  const unsigned long long item = static_cast<unsigned long long>(blockIdx.x) * kThreads + threadIdx.x;
  const unsigned long long items = static_cast<unsigned long long>(p.tokens) * per_token;
  if (item >= items) return;
  long long token;
  unsigned in_token;
  if (items <= 0xffffffffull) {  // 32-bit division is several times cheaper
    const unsigned t = static_cast<unsigned>(item) / per_token;
    token = t;
    in_token = static_cast<unsigned>(item) - t * per_token;
  } else {
    token = static_cast<long long>(item / per_token);
    in_token = static_cast<unsigned>(item - static_cast<unsigned long long>(token) * per_token);
  }
  const unsigned group = in_token / static_cast<unsigned>(slots);
  const int slot = static_cast<int>(in_token - group * static_cast<unsigned>(slots));
  const int head0 = static_cast<int>(group) * kHeads;
  const bool turns = slot < turning;
  int at_a, at_b;
  if (turns) {
    at_a = kInterleaved ? 2 * slot * kN : slot * kN;
    at_b = kInterleaved ? at_a + kN : at_a + half;
  } else {
    at_a = p.rot + (slot - turning) * 2 * kN;
    at_b = at_a + kN;
  }
  const bool has_b = at_b < p.dim;
  const T* x = static_cast<const T*>(p.x) + token * p.x_token + head0 * p.x_head;
  V ra[kHeads], rb[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (head0 + h < p.heads) {
      ra[h] = *reinterpret_cast<const V*>(x + h * p.x_head + at_a);
      if (has_b) rb[h] = *reinterpret_cast<const V*>(x + h * p.x_head + at_b);
    }
  }
  T* y = static_cast<T*>(p.y) + token * p.y_token + head0 * p.y_head;
  if (!turns) {
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (head0 + h < p.heads) {
        *reinterpret_cast<V*>(y + h * p.y_head + at_a) = ra[h];
        if (has_b) *reinterpret_cast<V*>(y + h * p.y_head + at_b) = rb[h];
      }
    }
    return;
  }
  float c[kN], s[kN];
  const long long pos = p.positions_64 ? static_cast<const long long*>(p.positions)[token]
                                       : static_cast<const int*>(p.positions)[token];
  if (pos >= 0 && pos < p.max_pos) {
    const float* row = p.table + pos * p.rot + slot * kN;
    load_table<kN>(row, c);
    load_table<kN>(row + half, s);
  } else {  // a position the table does not have must not pass for a rotation
#pragma unroll
    for (int i = 0; i < kN; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
  }
  if (p.transpose) {
#pragma unroll
    for (int i = 0; i < kN; ++i) s[i] = -s[i];
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (head0 + h < p.heads) {
      float a[kN], b[kN];
      if constexpr (kN == 1) {
        a[0] = to_f32<T>(ra[h]);
        b[0] = to_f32<T>(rb[h]);
      } else {
        unpack16<T>(ra[h], a);
        unpack16<T>(rb[h], b);
      }
      rotate_slot<kN, kInterleaved>(a, b, c, s);
      if constexpr (kN == 1) {
        y[h * p.y_head + at_a] = from_f32<T>(a[0]);
        y[h * p.y_head + at_b] = from_f32<T>(b[0]);
      } else {
        *reinterpret_cast<uint4*>(y + h * p.y_head + at_a) = pack16<T>(a);
        *reinterpret_cast<uint4*>(y + h * p.y_head + at_b) = pack16<T>(b);
      }
    }
  }
}

template <typename T, int kN, int kHeads>
cudaError_t launch_t(const RotaryParams& p, cudaStream_t stream) {
  const unsigned long long slots = p.rot / 2 / kN + (p.copy_rest ? (p.dim - p.rot + 2 * kN - 1) / (2 * kN) : 0);
  const unsigned long long items = static_cast<unsigned long long>(p.tokens) * ((p.heads + kHeads - 1) / kHeads) * slots;
  const unsigned long long blocks = (items + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  if (p.interleaved) {
    rotary_kernel<T, kN, true, kHeads><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
  } else {
    rotary_kernel<T, kN, false, kHeads><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_any(const RotaryParams& p, cudaStream_t stream) {
  constexpr int kN = 16 / sizeof(T);
  const bool vector = p.vector_ok && (p.rot / 2) % kN == 0 && p.dim % kN == 0;
  if (!vector) return launch_t<T, 1, 1>(p, stream);
  // Few tokens: more threads rather than more loads a thread.  Device us with four heads a thread / one, 40 heads of 128:
  // 64 tokens 2.7 / 2.1, 256 2.7 / 2.6, 512 3.5 / 3.6, 2048 6.6 / 8.1, 8192 30.2 / 32.7.
  const long long threads = static_cast<long long>(p.tokens) * p.heads * (p.dim / (2 * kN));
  if (threads >= kManyThreads) return launch_t<T, kN, 4>(p, stream);
  return launch_t<T, kN, 1>(p, stream);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, cudaStream_t stream) {
  if (p.dtype == kQuantBf16) return launch_any<__nv_bfloat16>(p, stream);
  if (p.dtype == kQuantFp16) return launch_any<__half>(p, stream);
  return launch_any<float>(p, stream);
}

}  // namespace b200fp8
