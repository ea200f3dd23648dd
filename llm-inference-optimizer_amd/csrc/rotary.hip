// Rotary positions of a [batch, tokens, heads, head_dim] tensor (rotary.h has
// the formula and how angles are computed).
//
// Bound by HBM: every element is read and written once.  A wave takes a token
// (with many tokens) or some heads of one (with few), computes the token's
// angles once, and gives each head's row to D / 8 lanes (16-bit; D / 4 in 32
// bits) of one packet, whose angles stay in registers over the heads.  In the
// half layout a lane also loads the packet that rotates into its own: the row
// is in the L1 by then, so HBM sees it once.  The first heads' packets are
// loaded before the angles are computed, which take about as long as the loads.
//
// Measured: 16384 tokens of 28 heads of 128 (bf16, 235 MB read and written)
// 36.0 us, 6.5 TB/s, the rate of a plain copy of that size, and 8192 in fp32 36.8;
// 100 of the 128 rotated, halves of no whole packets whose partners are loaded one
// by one, 59.6 us.  4 tokens of 12 heads 2.5 us, a launch and two dependent round
// trips to memory.
#include "rotary.h"

namespace mi355 {
namespace {

struct Args {
  const void* x;
  void* y;
  RotaryArgs rot;
  int64_t sb, st, sh;  // strides of x in elements
  int rows, tokens, heads, d, lanes, heads_per_wave;
};

constexpr int kAhead = 2;  // heads of a lane in flight
constexpr int kWaves = 4;  // of a workgroup, each for itself

template <typename T, int MODE> __global__ __launch_bounds__(64 * kWaves) void rotary_rows(Args a) {
  constexpr int W = pack_width<T>::value;
  typedef typename T::bits bits;
  __shared__ float angles[kWaves][2 * kMaxPairs];
  const int index = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(wave);
  if (token >= a.rows) return;
  float* cs = angles[wave];
  const int b = token / a.tokens, t = token - b * a.tokens;
  const int64_t position = MODE == ROTARY_NONE ? 0 : a.rot.positions[b * a.rot.pos_stride_b + t * a.rot.pos_stride_t];
  RotaryLane<T, MODE> lane(a.rot, (index % a.lanes) * W);
  const int step = 64 / a.lanes;
  const int last = lane.d0 < a.d ? min(a.heads, (static_cast<int>(blockIdx.y) + 1) * a.heads_per_wave) : 0;
  int h = blockIdx.y * a.heads_per_wave + index / a.lanes;
  const bits* x = static_cast<const bits*>(a.x) + b * a.sb + t * a.st + h * a.sh;
  bits* y = static_cast<bits*>(a.y) + (static_cast<int64_t>(token) * a.heads + h) * a.d + lane.d0;
  RotaryPacket<T, MODE> p[kAhead];
  const auto load = [&](int u) {
    if (h + u * step < last) p[u].load(x + u * step * a.sh, lane, a.rot);
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(u);  // on their way while the angles are computed
  if constexpr (MODE != ROTARY_NONE) {
    rotary_angles(cs, a.rot, position, index, 64);
    wave_sync();
    lane.angles(a.rot, cs);
  }
  while (h < last) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (h >= last) break;
      float v[W];
      p[u].turn(v, lane);
      Packet<T> o;
      o.pack(v);
      if (h + kAhead * step < last) p[u].load(x + kAhead * step * a.sh, lane, a.rot);
      *reinterpret_cast<u32x4*>(y) = o.raw;
      h += step;
      x += step * a.sh;
      y += step * a.d;
    }
  }
}

// Any head width and alignment: a lane per element.
template <typename T> __global__ __launch_bounds__(256) void rotary_generic(Args a) {
  __shared__ float cs[2 * kMaxPairs];
  const float* sn = cs + kMaxPairs;
  const int b = blockIdx.x / a.tokens, t = blockIdx.x - b * a.tokens;
  if (a.rot.rotary > 0)  // else there may be no positions
    rotary_angles(cs, a.rot, a.rot.positions[b * a.rot.pos_stride_b + t * a.rot.pos_stride_t], threadIdx.x, 256);
  __syncthreads();
  const int half = a.rot.rotary / 2;
  for (int h = blockIdx.y * a.heads_per_wave; h < min(a.heads, (static_cast<int>(blockIdx.y) + 1) * a.heads_per_wave); ++h) {
    const int64_t row = b * a.sb + t * a.st + h * a.sh;
    const int64_t out = (static_cast<int64_t>(blockIdx.x) * a.heads + h) * a.d;
    for (int d = threadIdx.x; d < a.d; d += 256) {
      float y = load_elem<T>(a.x, row + d);
      if (d < a.rot.rotary) {
        const bool lo = a.rot.interleaved ? (d & 1) == 0 : d < half;
        const int other = a.rot.interleaved ? d ^ 1 : lo ? d + half : d - half;
        const int j = a.rot.interleaved ? d >> 1 : lo ? d : d - half;
        const float o = load_elem<T>(a.x, row + other);
        y = y * cs[j] + (lo ? -(o * sn[j]) : o * sn[j]);
      }
      store_elem<T>(a.y, out + d, y);
    }
  }
}

template <typename T> int rotary_typed(Args a, hipStream_t s) {
  constexpr int W = pack_width<T>::value;
  const int64_t es = sizeof(typename T::bits), rows = a.rows;
  // whole packets, and a wave's lanes for a row at most
  const bool vec = a.d % W == 0 && a.d / W <= 64 && aligned16(a.x) && aligned16(a.y) &&
                   (a.sb * es | a.st * es | a.sh * es) % 16 == 0;
  a.lanes = vec ? row_lanes(a.d / W) : 64;
  // one pass over heads per wave until the tokens alone fill the chip (28 heads
  // of 128, a pass against a token per wave: 4.31 / 4.64 us for 512 tokens, 5.88
  // / 5.21 us for 1024)
  a.heads_per_wave = rows < 1024 ? 64 / a.lanes : a.heads;
  const dim3 grid(static_cast<unsigned>(vec ? (rows + kWaves - 1) / kWaves : rows),
                  static_cast<unsigned>((a.heads + a.heads_per_wave - 1) / a.heads_per_wave));
  static const char* what = "rotary launch";
  if (vec) {
    switch (rotary_mode(a.rot, W)) {
      case ROTARY_NONE: return launch(rotary_rows<T, ROTARY_NONE>, grid, 256, 0, a, s, what);
      case ROTARY_HALF: return launch(rotary_rows<T, ROTARY_HALF>, grid, 256, 0, a, s, what);
      case ROTARY_PAIRS: return launch(rotary_rows<T, ROTARY_PAIRS>, grid, 256, 0, a, s, what);
      default: return launch(rotary_rows<T, ROTARY_ODD>, grid, 256, 0, a, s, what);
    }
  }
  return launch(rotary_generic<T>, grid, 256, 0, a, s, what);
}

}  // namespace

int rotary_launch(const void* x, void* y, const RotaryArgs& rot, int64_t batch, int64_t tokens, int heads, int d,
                  int64_t sb, int64_t st, int64_t sh, int dtype, hipStream_t stream) {
  const Args a{x, y, rot, sb, st, sh, static_cast<int>(batch * tokens), static_cast<int>(tokens), heads, d, 0, 0};
  if (dtype == MI355_F32) return rotary_typed<F32>(a, stream);
  if (dtype == MI355_F16) return rotary_typed<F16>(a, stream);
  return rotary_typed<BF16>(a, stream);
}

}  // namespace mi355
