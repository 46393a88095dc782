// Rotary positions of x [tokens, heads, dim] (any token and head pitch, dim contiguous), out of place or in place, and
// the transposed rotation, which is the gradient with regard to x (sin -> -sin).
//
// Bound by HBM: x in, y out, one table row per token.  One thread owns one slot of one head (two 16-byte vectors of
// x, see rotary.cuh), reads both before it writes either - so in place needs nothing more - and ends.  The two loads
// of a thread do not wait for the position and the table row (they are issued first), and 40 to 64 KB of x per SM are
// on their way at full occupancy, which covers HBM latency without a loop or a ring.  The table row of a token is
// read once per head from L1: twice the bytes of x, but L1 has ten times the bandwidth that HBM leaves an SM.
#include "kernels.h"
#include "rotary.cuh"

namespace b200fp8 {
namespace {

constexpr int kThreads = 256;

// kN: pairs of a slot (16 bytes of T each; 1: any alignment and any even rot).  Slots [0, rot / 2 / kN) of a head are
// rotated, the ones behind them copy kN elements each of [rot, dim).
template <typename T, int kN, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  const int half = p.rot / 2;
  const int turning = half / kN;
  const int slots = turning + (p.copy_rest ? (p.dim - p.rot) / kN : 0);
  const unsigned per_token = static_cast<unsigned>(p.heads) * static_cast<unsigned>(slots);
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
  const unsigned head = in_token / static_cast<unsigned>(slots);
  const int slot = static_cast<int>(in_token - head * static_cast<unsigned>(slots));
  const T* x = static_cast<const T*>(p.x) + token * p.x_token + static_cast<long long>(head) * p.x_head;
  T* y = static_cast<T*>(p.y) + token * p.y_token + static_cast<long long>(head) * p.y_head;
  if (slot >= turning) {  // beyond the rotated part
    const int at = p.rot + (slot - turning) * kN;
    if constexpr (kN == 1) {
      y[at] = x[at];
    } else {
      *reinterpret_cast<uint4*>(y + at) = *reinterpret_cast<const uint4*>(x + at);
    }
    return;
  }
  const int at_a = kInterleaved ? 2 * slot * kN : slot * kN;
  const int at_b = kInterleaved ? at_a + kN : at_a + half;
  float a[kN], b[kN], c[kN], s[kN];
  if constexpr (kN == 1) {
    a[0] = to_f32<T>(x[at_a]);
    b[0] = to_f32<T>(x[at_b]);
  } else {
    const uint4 ra = *reinterpret_cast<const uint4*>(x + at_a);
    const uint4 rb = *reinterpret_cast<const uint4*>(x + at_b);
    unpack16<T>(ra, a);
    unpack16<T>(rb, b);
  }
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
  rotate_slot<kN, kInterleaved>(a, b, c, s);
  if constexpr (kN == 1) {
    y[at_a] = from_f32<T>(a[0]);
    y[at_b] = from_f32<T>(b[0]);
  } else {
    *reinterpret_cast<uint4*>(y + at_a) = pack16<T>(a);
    *reinterpret_cast<uint4*>(y + at_b) = pack16<T>(b);
  }
}

template <typename T, int kN>
cudaError_t launch_t(const RotaryParams& p, cudaStream_t stream) {
  const unsigned long long slots = p.rot / 2 / kN + (p.copy_rest ? (p.dim - p.rot) / kN : 0);
  const unsigned long long items = static_cast<unsigned long long>(p.tokens) * p.heads * slots;
  if (items == 0) return cudaSuccess;
  const unsigned long long blocks = (items + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  if (p.interleaved) {
    rotary_kernel<T, kN, true><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
  } else {
    rotary_kernel<T, kN, false><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_any(const RotaryParams& p, cudaStream_t stream) {
  constexpr int kN = 16 / sizeof(T);
  const bool vector = p.vector_ok && (p.rot / 2) % kN == 0 && p.dim % kN == 0;
  return vector ? launch_t<T, kN>(p, stream) : launch_t<T, 1>(p, stream);
}

}  // namespace

cudaError_t launch_rotary(const RotaryParams& p, cudaStream_t stream) {
  if (p.dtype == kQuantBf16) return launch_any<__nv_bfloat16>(p, stream);
  if (p.dtype == kQuantFp16) return launch_any<__half>(p, stream);
  return launch_any<float>(p, stream);
}

}  // namespace b200fp8
