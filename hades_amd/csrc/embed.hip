// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i, :]  = f(i, :) * weight[ids[i], :]                     (hades_embed)
//   grad[v, :] = sum over i with ids[i] = v of f(i, :) * g[i, :]  (hades_embed_grad)
//
// f = scale, or with dropout keep(i, c) * scale / (1 - p) (rowvec.h).  An id outside [0, num_rows) is
// padding: a row of zeros, no gradient.
//
// Lookup: bound by memory (n rows read, n rows written).  The batch is one flat list of pieces of
// eight columns; a thread takes four that lie a block apart, so four row loads are in flight once
// their ids are there, and one token of a wide row still spreads over the block.
//
// Gradient: every row of the dense gradient is written once, n rows of g are read once; sums are
// held in float32 and their order is fixed by (n, dim) and the sorted tokens, so results are the same
// from run to run.  Three parts:
//   tokens  positions in token order (stable) and row_start[v] = first of token v
//   sum     chunks of kShort or kLong sorted positions, whatever the tokens' frequencies: one lane
//           group walks a chunk's rows for its columns and writes every token that lies inside the
//           chunk; what crosses a border goes to a partial row.  Further blocks of the same launch
//           write the zeros of the tokens that do not occur.
//   join    adds the partial rows of the tokens that cross chunk borders, in chunk order.
#include "internal.h"
#include "rowvec.h"

namespace hades {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 4;    // pieces per thread of the flat kernels
constexpr uint32_t kNoToken = 0xffffffffu;

// ---- lookup -------------------------------------------------------------------------------------
template <typename T, typename I>
struct EmbedArgs {
  const T* weight;
  const I* ids;
  T* out;
  int64_t stride, num_rows, dim, pieces;
  FastDiv per_row;
  DropArgs drop;
};

template <typename T, typename I>
__global__ __launch_bounds__(kThreads) void embed_kernel(EmbedArgs<T, I> a) {
  const DropKeys keys(a.drop);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads * kPieces);
  const int64_t row0 = a.pieces < (int64_t(1) << 31) ? int64_t(a.per_row.div(uint32_t(first))) : first / a.per_row.d;
  const uint32_t rest = static_cast<uint32_t>(first - row0 * a.per_row.d);
  int64_t row[kPieces], id[kPieces];
  uint32_t piece[kPieces];
  int valid[kPieces];
  f32x8 v[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const uint32_t at = rest + threadIdx.x + k * kThreads;
    const uint32_t down = a.per_row.div(at);
    row[k] = row0 + down;
    piece[k] = at - down * a.per_row.d;
    const bool in = first + threadIdx.x + k * kThreads < a.pieces;
    const int64_t left = a.dim - static_cast<int64_t>(piece[k]) * kPiece;
    valid[k] = in ? (left < kPiece ? static_cast<int>(left) : kPiece) : 0;
    id[k] = in ? static_cast<int64_t>(a.ids[row[k]]) : int64_t(-1);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const bool live = static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(a.num_rows);
    v[k] = load8(a.weight + (live ? id[k] : 0) * a.stride + static_cast<int64_t>(piece[k]) * kPiece,
                 live ? valid[k] : 0);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const f32x8 y = keys.on() ? keys.apply(v[k], static_cast<uint32_t>(row[k]), piece[k]) : v[k] * keys.factor;
    store8(a.out + row[k] * a.dim + static_cast<int64_t>(piece[k]) * kPiece, y, valid[k]);
  }
}

template <typename T, typename I>
int launch_embed(const void* weight, int64_t stride, int64_t num_rows, const void* ids, int64_t n, void* out,
                 int64_t dim, const DropArgs& drop, hipStream_t st) {
  EmbedArgs<T, I> a;
  a.weight = static_cast<const T*>(weight);
  a.ids = static_cast<const I*>(ids);
  a.out = static_cast<T*>(out);
  a.stride = stride;
  a.num_rows = num_rows;
  a.dim = dim;
  const int64_t per_row = ceil_div(dim, kPiece);
  a.pieces = n * per_row;
  a.per_row = FastDiv(static_cast<uint32_t>(per_row));
  a.drop = drop;
  const int64_t blocks = ceil_div(a.pieces, int64_t(kThreads) * kPieces);
  HADES_REQUIRE(blocks < (int64_t(1) << 24), "embed: too many values for one call");
  HADES_LAUNCH((embed_kernel<T, I>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
  return HADES_OK;
}

// ---- gradient: tokens ---------------------------------------------------------------------------
template <typename I>
__global__ __launch_bounds__(kThreads) void token_key_kernel(const I* __restrict__ ids, int64_t n, int64_t rows,
                                                             int64_t num_rows, int64_t padding,
                                                             int64_t* __restrict__ keys) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= rows) return;
  const int64_t id = i < n ? static_cast<int64_t>(ids[i]) : int64_t(-1);
  const bool live = static_cast<uint64_t>(id) < static_cast<uint64_t>(num_rows) && id != padding;
  keys[i] = live ? id : num_rows;   // padding sorts behind every token
}

// row_start[v] = number of sorted tokens below v, for v in [0, num_rows]
__global__ __launch_bounds__(kThreads) void row_start_kernel(const uint32_t* __restrict__ token, int64_t n,
                                                             int64_t num_rows, uint32_t* __restrict__ row_start) {
  const int64_t v = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (v > num_rows) return;
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (token[mid] < static_cast<uint32_t>(v)) lo = mid + 1; else hi = mid;
  }
  row_start[v] = static_cast<uint32_t>(lo);
}

// ---- gradient: sums -----------------------------------------------------------------------------
constexpr int kLong = 32;    // sorted positions of a chunk
constexpr int kShort = 8;    // ... where chunks of kLong would leave the chip short of waves
constexpr int64_t kLongFrom = 2048;   // waves

struct GradPlan {
  int group;        // lanes that walk a chunk's rows together: 8, 16, 32 or 64
  int slices;       // groups side by side along a row
  int chunk;
  int64_t chunks;
  int64_t pieces;   // of a row
};

GradPlan plan_grad(int64_t n, int64_t dim) {
  GradPlan p;
  p.pieces = ceil_div(dim, kPiece);
  p.group = 8;
  while (p.group < kWave && p.group < p.pieces) p.group *= 2;
  p.slices = static_cast<int>(ceil_div(p.pieces, p.group));
  const int64_t waves = ceil_div(ceil_div(n, kLong) * p.slices * p.group, kWave);
  p.chunk = waves >= kLongFrom ? kLong : kShort;
  p.chunks = ceil_div(n, p.chunk);
  return p;
}

template <typename T, typename O>
struct GradArgs {
  const T* grad;
  const uint32_t* perm;        // batch position of every sorted position
  const uint32_t* token;       // its token
  const uint32_t* row_start;   // [num_rows + 1]
  O* out;
  float* partial;              // [2 * chunks][dim]: of every chunk the token it begins inside, the one it ends inside
  int64_t grad_stride, out_stride, num_rows, dim, chunks;
  int slices, accumulate;
  unsigned sum_blocks;
  FastDiv per_row, per_chunk;
  int64_t zero_pieces;
  DropArgs drop;
};

template <typename T, typename O>
__device__ __forceinline__ void put_row(const GradArgs<T, O>& a, uint32_t token, int64_t col, f32x8 v, int valid) {
  O* p = a.out + static_cast<int64_t>(token) * a.out_stride + col;
  if (a.accumulate) v += load8(p, valid);
  store8(p, v, valid);
}

__device__ __forceinline__ void put_partial(float* __restrict__ p, f32x8 v, int valid) { store8(p, v, valid); }

template <typename T, typename O, int G, int CH>
__global__ __launch_bounds__(kThreads) void embed_grad_sum_kernel(GradArgs<T, O> a) {
  if (blockIdx.x >= a.sum_blocks) {
    // the rows of tokens that do not occur
    const int64_t first = static_cast<int64_t>(blockIdx.x - a.sum_blocks) * (kThreads * kPieces);
    const int64_t row0 = a.zero_pieces < (int64_t(1) << 31) ? int64_t(a.per_row.div(uint32_t(first)))
                                                            : first / a.per_row.d;
    const uint32_t rest = static_cast<uint32_t>(first - row0 * a.per_row.d);
    const f32x8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      if (first + threadIdx.x + k * kThreads >= a.zero_pieces) break;
      const uint32_t at = rest + threadIdx.x + k * kThreads;
      const uint32_t down = a.per_row.div(at);
      const int64_t v = row0 + down;
      if (a.row_start[v] != a.row_start[v + 1]) continue;
      const int64_t col = static_cast<int64_t>(at - down * a.per_row.d) * kPiece;
      store8(a.out + v * a.out_stride + col, zero, a.dim - col < kPiece ? int(a.dim - col) : kPiece);
    }
    return;
  }
  constexpr int kGroups = kThreads / G;
  constexpr int U = 8;   // rows in flight
  const DropKeys keys(a.drop);
  const int lane = threadIdx.x & (G - 1);
  const uint32_t item = blockIdx.x * kGroups + threadIdx.x / G;
  const uint32_t chunk = a.per_chunk.div(item);
  const uint32_t piece = (item - chunk * a.slices) * G + lane;
  const int64_t col = static_cast<int64_t>(piece) * kPiece;
  const int64_t left = a.dim - col;
  const int valid = left < 0 ? 0 : (left < kPiece ? static_cast<int>(left) : kPiece);
  const int64_t live = a.row_start[a.num_rows];
  const int64_t p0 = static_cast<int64_t>(chunk) * CH;
  if (p0 >= live || valid == 0) return;
  const int len = live - p0 < CH ? static_cast<int>(live - p0) : CH;
  const uint32_t before = p0 > 0 ? a.token[p0 - 1] : kNoToken;
  const uint32_t after = p0 + len < live ? a.token[p0 + len] : kNoToken;
  uint32_t cur = a.token[p0];
  bool head = before == cur;   // the token summed now began in an earlier chunk
  const f32x8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  f32x8 acc = zero;
  float* const slot = a.partial + 2 * static_cast<int64_t>(chunk) * a.dim + col;
  for (int t = 0; t < len; t += U) {
    f32x8 row[U];
    uint32_t tok[U], pos[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t j = p0 + (t + k < len ? t + k : len - 1);   // the last row again behind the end: not added
      pos[k] = a.perm[j];
      tok[k] = a.token[j];
    }
#pragma unroll
    for (int k = 0; k < U; ++k)
      row[k] = load8<T, true>(a.grad + static_cast<int64_t>(pos[k]) * a.grad_stride + col, valid);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (t + k >= len) break;
      if (tok[k] != cur) {
        if (head) put_partial(slot, acc, valid);
        else put_row(a, cur, col, acc, valid);
        acc = zero;
        cur = tok[k];
        head = false;
      }
      acc += keys.on() ? keys.apply(row[k], pos[k], piece) : row[k] * keys.factor;
    }
  }
  if (head) put_partial(slot, acc, valid);
  else if (after == cur) put_partial(slot + a.dim, acc, valid);
  else put_row(a, cur, col, acc, valid);
}

// Block (chunk c, slice): the token that begins in chunk c and goes on behind it, if there is one.
// Its lane groups take the partial rows in turn; the groups' sums are added in order.
template <typename T, typename O, int G, int CH>
__global__ __launch_bounds__(kThreads) void embed_grad_join_kernel(GradArgs<T, O> a) {
  constexpr int kGroups = kThreads / G;
  constexpr int U = 8;
  __shared__ f32x8 part[kThreads];
  const int64_t live = a.row_start[a.num_rows];
  const int64_t c = a.per_chunk.div(blockIdx.x);
  const int64_t border = (c + 1) * CH;
  if (border >= live) return;
  const uint32_t token = a.token[border - 1];
  if (a.token[border] != token || static_cast<int64_t>(a.row_start[token]) < c * CH) return;
  const int64_t parts = (static_cast<int64_t>(a.row_start[token + 1]) - 1) / CH - c + 1;
  const int group = threadIdx.x / G, lane = threadIdx.x & (G - 1);
  const int64_t col = (static_cast<int64_t>(blockIdx.x - static_cast<uint32_t>(c) * a.slices) * G + lane) * kPiece;
  const int64_t left = a.dim - col;
  const int valid = left < 0 ? 0 : (left < kPiece ? static_cast<int>(left) : kPiece);
  f32x8 acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t t = group; t < parts; t += kGroups * U) {
    f32x8 row[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t i = t + k * kGroups;
      const int64_t slot = i == 0 ? 2 * c + 1 : 2 * (c + i);
      row[k] = load8(a.partial + (i < parts ? slot * a.dim + col : 0), i < parts ? valid : 0);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) acc += row[k];
  }
  part[threadIdx.x] = acc;
  __syncthreads();
  if (group != 0 || valid == 0) return;
  for (int g = 1; g < kGroups; ++g) acc += part[g * G + lane];
  put_row(a, token, col, acc, valid);
}

inline size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

struct GradWs {
  void* sort;
  size_t sort_bytes;
  int64_t* keys;
  uint32_t* row_start;
  float* partial;
  size_t bytes;
};

GradWs carve_grad(void* base, int64_t n, int64_t dim, int64_t num_rows) {
  const GradPlan p = plan_grad(n, dim);
  GradWs w;
  Carver c(base);
  w.sort_bytes = round256(sort_ids_workspace_bytes(n));
  w.sort = c.take<char>(w.sort_bytes);
  w.keys = c.take<int64_t>(n);
  w.row_start = c.take<uint32_t>(num_rows + 1);
  w.partial = c.take<float>(2 * p.chunks * dim);
  w.bytes = c.total();
  return w;
}

template <typename T, typename O, int G, int CH>
int launch_sums(GradArgs<T, O>& a, const GradPlan& p, hipStream_t st) {
  const int64_t sum_blocks = ceil_div(p.chunks * p.slices * G, kThreads);
  const int64_t zero_blocks = a.accumulate ? 0 : ceil_div(a.zero_pieces, int64_t(kThreads) * kPieces);
  HADES_REQUIRE(p.chunks * p.slices < (int64_t(1) << 31) && sum_blocks + zero_blocks < (int64_t(1) << 24) &&
                    p.chunks * p.slices < (int64_t(1) << 24),
                "embed_grad: too many values for one call");
  a.sum_blocks = static_cast<unsigned>(sum_blocks);
  if (sum_blocks + zero_blocks > 0)
    HADES_LAUNCH((embed_grad_sum_kernel<T, O, G, CH>), dim3(static_cast<unsigned>(sum_blocks + zero_blocks)),
                 dim3(kThreads), 0, st, a);
  if (p.chunks > 1)
    HADES_LAUNCH((embed_grad_join_kernel<T, O, G, CH>), dim3(static_cast<unsigned>(p.chunks * p.slices)),
                 dim3(kThreads), 0, st, a);
  return HADES_OK;
}

template <typename T, typename O>
int launch_grad(const void* grad, int64_t grad_stride, const uint32_t* perm, const uint32_t* token, void* out,
                int64_t out_stride, int64_t num_rows, int64_t dim, const GradPlan& p, const GradWs& w,
                int accumulate, const DropArgs& drop, hipStream_t st) {
  GradArgs<T, O> a;
  a.grad = static_cast<const T*>(grad);
  a.perm = perm;
  a.token = token;
  a.row_start = w.row_start;
  a.out = static_cast<O*>(out);
  a.partial = w.partial;
  a.grad_stride = grad_stride;
  a.out_stride = out_stride;
  a.num_rows = num_rows;
  a.dim = dim;
  a.chunks = p.chunks;
  a.slices = p.slices;
  a.accumulate = accumulate;
  a.per_row = FastDiv(static_cast<uint32_t>(p.pieces));
  a.per_chunk = FastDiv(static_cast<uint32_t>(p.slices));
  a.zero_pieces = num_rows * p.pieces;
  a.drop = drop;
#define HADES_SUMS(G_)                                                             \
  return p.chunk == kLong ? launch_sums<T, O, G_, kLong>(a, p, st) : launch_sums<T, O, G_, kShort>(a, p, st)
  switch (p.group) {
    case 8: HADES_SUMS(8);
    case 16: HADES_SUMS(16);
    case 32: HADES_SUMS(32);
    default: HADES_SUMS(64);
  }
#undef HADES_SUMS
}

}  // namespace
}  // namespace hades

using namespace hades;

extern "C" {

int hades_embed(const void* weight, int64_t weight_stride, int64_t num_rows, const void* ids, int64_t n,
                void* out, int64_t dim, int dtype, int itype, float scale, double p, uint64_t seed,
                int64_t offset, const int64_t* offset_ptr, void* stream) {
  HADES_REQUIRE(n >= 0 && num_rows >= 0 && dim >= 1, "n and num_rows must be >= 0 and dim >= 1");
  HADES_REQUIRE(n < (int64_t(1) << 32) && dim < (int64_t(1) << 31), "embed: n or dim too large");
  HADES_REQUIRE(dtype == HADES_F32 || dtype == HADES_F16 || dtype == HADES_BF16,
                "Type can only be float, half or bfloat16");
  HADES_REQUIRE(itype == HADES_I32 || itype == HADES_I64, "ID can only be int32 or int64");
  HADES_REQUIRE(weight_stride >= dim || num_rows <= 1, "row stride below dim");
  DropArgs drop;
  HADES_REQUIRE(make_drop(p, seed, offset, offset_ptr, scale, &drop), "p must lie in [0, 1]");
  if (n == 0) return HADES_OK;
  HADES_REQUIRE((weight || num_rows == 0) && ids && out, "null pointer argument");
  hipStream_t st = static_cast<hipStream_t>(stream);
#define HADES_EMBED(T_)                                                                               \
  return itype == HADES_I64                                                                           \
             ? launch_embed<T_, int64_t>(weight, weight_stride, num_rows, ids, n, out, dim, drop, st) \
             : launch_embed<T_, int32_t>(weight, weight_stride, num_rows, ids, n, out, dim, drop, st)
  if (dtype == HADES_F32) HADES_EMBED(float);
  if (dtype == HADES_F16) HADES_EMBED(f16);
  HADES_EMBED(bf16);
#undef HADES_EMBED
}

size_t hades_embed_grad_workspace_bytes(int64_t n, int64_t dim, int64_t num_rows) {
  if (n < 0 || dim < 1 || num_rows < 0) return 0;
  return carve_grad(nullptr, n > 0 ? n : 1, dim, num_rows).bytes;
}

int hades_embed_grad(const void* grad, int64_t grad_stride, const void* ids, int64_t n, void* out,
                     int64_t out_stride, int64_t num_rows, int64_t dim, int dtype, int out_dtype, int itype,
                     int64_t padding_idx, int accumulate, float scale, double p, uint64_t seed, int64_t offset,
                     const int64_t* offset_ptr, void* workspace, size_t workspace_bytes, void* stream) {
  HADES_REQUIRE(n >= 0 && num_rows >= 0 && dim >= 1, "n and num_rows must be >= 0 and dim >= 1");
  HADES_REQUIRE(n < (int64_t(1) << 30) && num_rows < (int64_t(1) << 31) && dim < (int64_t(1) << 31),
                "embed_grad: n must be below 2^30, num_rows and dim below 2^31");
  HADES_REQUIRE(dtype == HADES_F32 || dtype == HADES_F16 || dtype == HADES_BF16,
                "Type can only be float, half or bfloat16");
  HADES_REQUIRE(out_dtype == dtype || out_dtype == HADES_F32, "the gradient's type is the rows' or float");
  HADES_REQUIRE(itype == HADES_I32 || itype == HADES_I64, "ID can only be int32 or int64");
  HADES_REQUIRE(grad_stride >= dim || n <= 1, "row stride below dim");
  HADES_REQUIRE(out_stride >= dim || num_rows <= 1, "row stride below dim");
  DropArgs drop;
  HADES_REQUIRE(make_drop(p, seed, offset, offset_ptr, scale, &drop), "p must lie in [0, 1]");
  if (num_rows == 0 || (n == 0 && accumulate)) return HADES_OK;
  HADES_REQUIRE(out && (n == 0 || (grad && ids)), "null pointer argument");
  const int64_t rows = n > 0 ? n : 1;   // a batch of no tokens: one padding position
  const GradWs w = carve_grad(workspace, rows, dim, num_rows);
  if (workspace == nullptr || workspace_bytes < w.bytes)
    return set_error(HADES_ERR_WORKSPACE, "embed_grad workspace too small: need %zu bytes, got %zu", w.bytes,
                     workspace_bytes);
  HADES_REQUIRE((align_of_ptr(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const GradPlan plan = plan_grad(rows, dim);
  const dim3 block(kThreads), kgrid(static_cast<unsigned>(ceil_div(rows, kThreads)));
  if (itype == HADES_I64)
    HADES_LAUNCH((token_key_kernel<int64_t>), kgrid, block, 0, st, static_cast<const int64_t*>(ids), n, rows,
                 num_rows, padding_idx, w.keys);
  else
    HADES_LAUNCH((token_key_kernel<int32_t>), kgrid, block, 0, st, static_cast<const int32_t*>(ids), n, rows,
                 num_rows, padding_idx, w.keys);
  SortResult sr;
  const int rc = sort_ids(w.keys, rows, num_rows + 1, w.sort, w.sort_bytes, st, &sr);
  if (rc != HADES_OK) return rc;
  HADES_REQUIRE(!sr.key64, "internal: token keys must be 32-bit");
  const uint32_t* token = static_cast<const uint32_t*>(sr.sorted_keys);
  HADES_LAUNCH(row_start_kernel, dim3(static_cast<unsigned>(ceil_div(num_rows + 1, kThreads))), block, 0, st, token,
               rows, num_rows, w.row_start);
#define HADES_GRAD(T_, O_)                                                                               \
  return launch_grad<T_, O_>(grad, grad_stride, sr.perm, token, out, out_stride, num_rows, dim, plan, w, \
                             accumulate != 0, drop, st)
  if (dtype == HADES_F32) HADES_GRAD(float, float);
  if (dtype == HADES_F16) {
    if (out_dtype == HADES_F16) HADES_GRAD(f16, f16);
    HADES_GRAD(f16, float);
  }
  if (out_dtype == HADES_BF16) HADES_GRAD(bf16, bf16);
  HADES_GRAD(bf16, float);
#undef HADES_GRAD
}

}  // extern "C"
