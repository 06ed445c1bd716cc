// Dropout whose mask is drawn from a counter for every value and never stored.
//
//   out[r, c] = keep(r, c) ? x[r, c] * factor : 0   (+ residual[r, c])
//
// keep(r, c): 16 bits of Philox4x32 at counter (c / 8, r, offset) reach the threshold.  The mask is
// a function of the value's row and column alone, so the backward pass draws the same one from the
// same seed and offset, whatever the strides; the gradient of x is this kernel on the output's gradient.
//
// Bound by memory: every value is read once and written once.  A thread takes one piece of eight columns, or
// two that lie a block apart where 16-bit rows are streamed, with all its loads in flight before the first is used.
#include "rowvec.h"

namespace hades {
namespace {

constexpr int kThreads = 256;
// pieces of a thread
template <typename T, bool kOnce>
constexpr int drop_pieces() { return kOnce && sizeof(T) == 2 ? 2 : 1; }

template <typename T>
struct DropoutArgs {
  const T* x;
  const T* residual;   // may be null
  T* out;
  int64_t x_stride, res_stride, pieces;   // pieces = rows * pieces of a row
  int64_t cols;
  FastDiv per_row;
  DropArgs drop;
};

template <typename T, bool kOnce>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs<T> a) {
  constexpr int kPieces = drop_pieces<T, kOnce>();
  const DropKeys keys(a.drop);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads * kPieces);
  const int64_t row0 = a.pieces < (int64_t(1) << 31) ? int64_t(a.per_row.div(uint32_t(first))) : first / a.per_row.d;
  const uint32_t rest = static_cast<uint32_t>(first - row0 * a.per_row.d);
  int64_t row[kPieces];
  uint32_t piece[kPieces];
  int valid[kPieces];
  typename Vec8<T>::V v[kPieces], res[kPieces];   // as they lie in memory: nothing waits before all are under way
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const uint32_t at = rest + threadIdx.x + k * kThreads;
    const uint32_t down = a.per_row.div(at);
    row[k] = row0 + down;
    piece[k] = at - down * a.per_row.d;
    const bool in = first + threadIdx.x + k * kThreads < a.pieces;
    const int64_t left = a.cols - static_cast<int64_t>(piece[k]) * kPiece;
    valid[k] = in ? (left < kPiece ? static_cast<int>(left) : kPiece) : 0;
    const int64_t col = static_cast<int64_t>(piece[k]) * kPiece;
    v[k] = load8_raw<T, kOnce>(a.x + row[k] * a.x_stride + col, valid[k]);
  }
  if (a.residual != nullptr) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k)
      res[k] = load8_raw<T, kOnce>(a.residual + row[k] * a.res_stride + static_cast<int64_t>(piece[k]) * kPiece,
                                   valid[k]);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    f32x8 y = __builtin_convertvector(v[k], f32x8);
    if (keys.on()) y = keys.apply(y, static_cast<uint32_t>(row[k]), piece[k]);
    if (a.residual != nullptr) y += __builtin_convertvector(res[k], f32x8);
    store8(a.out + row[k] * a.cols + static_cast<int64_t>(piece[k]) * kPiece, y, valid[k]);
  }
}

template <typename T>
int launch(const void* x, int64_t x_stride, const void* residual, int64_t res_stride, void* out,
           int64_t rows, int64_t cols, const DropArgs& drop, hipStream_t st) {
  DropoutArgs<T> a;
  a.x = static_cast<const T*>(x);
  a.residual = static_cast<const T*>(residual);
  a.out = static_cast<T*>(out);
  a.x_stride = x_stride;
  a.res_stride = res_stride;
  a.cols = cols;
  const int64_t per_row = ceil_div(cols, kPiece);
  a.pieces = rows * per_row;
  a.per_row = FastDiv(static_cast<uint32_t>(per_row));
  a.drop = drop;
  // 2^27 bfloat16 values streamed 87 us, 119 with residual, else 103 and 137; 2^25 values streamed 24 and 35 us, else
  // 21 and 30 (their inputs were in the last-level cache)
  const bool once = streamed(rows * cols * static_cast<int64_t>(sizeof(T)) * (residual ? 2 : 1));
  const int64_t blocks = ceil_div(a.pieces, int64_t(kThreads) * (once ? drop_pieces<T, true>() : drop_pieces<T, false>()));
  HADES_REQUIRE(blocks < (int64_t(1) << 24), "dropout: too many values for one call");
  const dim3 grid(static_cast<unsigned>(blocks)), block(kThreads);
  if (once) HADES_LAUNCH((dropout_kernel<T, true>), grid, block, 0, st, a);
  else HADES_LAUNCH((dropout_kernel<T, false>), grid, block, 0, st, a);
  return HADES_OK;
}

}  // namespace
}  // namespace hades

using namespace hades;

extern "C" int hades_dropout(const void* x, int64_t x_stride, const void* residual, int64_t res_stride,
                             void* out, int64_t rows, int64_t cols, int dtype, double p, uint64_t seed,
                             int64_t offset, const int64_t* offset_ptr, void* stream) {
  HADES_REQUIRE(rows >= 0 && cols >= 0, "rows and cols must be >= 0");
  HADES_REQUIRE(rows < (int64_t(1) << 32) && cols < (int64_t(1) << 31),
                "dropout: at most 2^32 - 1 rows of 2^31 - 1 columns");
  HADES_REQUIRE(dtype == HADES_F32 || dtype == HADES_F16 || dtype == HADES_BF16,
                "Type can only be float, half or bfloat16");
  DropArgs drop;
  HADES_REQUIRE(make_drop(p, seed, offset, offset_ptr, 1.0, &drop), "p must lie in [0, 1]");
  if (rows == 0 || cols == 0) return HADES_OK;
  HADES_REQUIRE(x && out, "null pointer argument");
  HADES_REQUIRE(x_stride >= cols || rows == 1, "row stride below cols");
  HADES_REQUIRE(!residual || res_stride >= cols || rows == 1, "row stride below cols");
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == HADES_F32) return launch<float>(x, x_stride, residual, res_stride, out, rows, cols, drop, st);
  if (dtype == HADES_F16) return launch<f16>(x, x_stride, residual, res_stride, out, rows, cols, drop, st);
  return launch<bf16>(x, x_stride, residual, res_stride, out, rows, cols, drop, st);
}
