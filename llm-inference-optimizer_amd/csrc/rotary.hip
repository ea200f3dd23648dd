// Rotary positions of a [batch, tokens, heads, head_dim] tensor (rotary.h has
// the formula and how angles are computed).
//
// Bound by HBM: every element is read and written once.  A workgroup takes a
// token (with many tokens) or some heads of one (with few), computes the
// token's angles once, and gives each head's row to D / 8 lanes (16-bit; D / 4
// in 32 bits) of one packet.  In the half layout a lane also loads the packet
// that rotates into its own: the row is in the L1 by then, so HBM sees it once.
#include "rotary.h"

namespace mi355 {
namespace {

struct Args {
  const void* x;
  void* y;
  RotaryArgs rot;
  int64_t tokens, sb, st, sh;  // tokens per batch row; strides of x in elements
  int heads, d, lanes, heads_per_wg;
};

template <typename T> __global__ __launch_bounds__(256) void rotary_rows(Args a) {
  constexpr int W = pack_width<T>::value;
  __shared__ float cs[2 * kMaxPairs];
  const int64_t b = blockIdx.x / a.tokens, t = blockIdx.x % a.tokens;
  rotary_angles(cs, a.rot, a.rot.positions[b * a.rot.pos_stride_b + t * a.rot.pos_stride_t]);
  __syncthreads();
  const int d0 = (threadIdx.x % a.lanes) * W;
  const int first = blockIdx.y * a.heads_per_wg;
  const int last = min(a.heads, first + a.heads_per_wg);
  if (d0 >= a.d) return;
  for (int h = first + threadIdx.x / a.lanes; h < last; h += 256 / a.lanes) {
    const typename T::bits* row = static_cast<const typename T::bits*>(a.x) + b * a.sb + t * a.st + h * a.sh;
    RotaryPacket<T> p;
    p.load(row, d0, a.rot);
    float y[W];
    p.rotate(y, row, d0, a.rot, cs);
    Packet<T> o;
    o.pack(y);
    typename T::bits* out = static_cast<typename T::bits*>(a.y) + (static_cast<int64_t>(blockIdx.x) * a.heads + h) * a.d;
    *reinterpret_cast<u32x4*>(out + d0) = o.raw;
  }
}

// Any head width and alignment: a lane per element.
template <typename T> __global__ __launch_bounds__(256) void rotary_generic(Args a) {
  __shared__ float cs[2 * kMaxPairs];
  const float* sn = cs + kMaxPairs;
  const int64_t b = blockIdx.x / a.tokens, t = blockIdx.x % a.tokens;
  rotary_angles(cs, a.rot, a.rot.positions[b * a.rot.pos_stride_b + t * a.rot.pos_stride_t]);
  __syncthreads();
  const int half = a.rot.rotary / 2;
  for (int h = blockIdx.y * a.heads_per_wg; h < min(a.heads, (static_cast<int>(blockIdx.y) + 1) * a.heads_per_wg); ++h) {
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

template <typename T> int rotary_typed(Args a, int64_t batch, hipStream_t s) {
  constexpr int W = pack_width<T>::value;
  const int64_t es = sizeof(typename T::bits), rows = batch * a.tokens;
  const bool vec = a.d % W == 0 && aligned16(a.x) && aligned16(a.y) && (a.sb * es | a.st * es | a.sh * es) % 16 == 0;
  a.lanes = vec ? row_lanes(a.d / W) : 256;
  // one pass over heads per workgroup until the tokens alone fill the chip
  const int pass = 256 / a.lanes;
  a.heads_per_wg = rows < 1024 ? pass : a.heads;
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>((a.heads + a.heads_per_wg - 1) / a.heads_per_wg));
  return launch(vec ? rotary_rows<T> : rotary_generic<T>, grid, 256, 0, a, s, "rotary launch");
}

}  // namespace

int rotary_launch(const void* x, void* y, const RotaryArgs& rot, int64_t batch, int64_t tokens, int heads, int d,
                  int64_t sb, int64_t st, int64_t sh, int dtype, hipStream_t stream) {
  const Args a{x, y, rot, tokens, sb, st, sh, heads, d, 0, 0};
  if (dtype == MI355_F32) return rotary_typed<F32>(a, batch, stream);
  if (dtype == MI355_F16) return rotary_typed<F16>(a, batch, stream);
  return rotary_typed<BF16>(a, batch, stream);
}

}  // namespace mi355
