// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   out[i, :]  = f(i, :) * weight[ids[i], :]                     (hades_embed)
//   grad[v, :] = sum over i with ids[i] = v of f(i, :) * g[i, :]  (hades_embed_grad)
//
// f = scale, or with dropout keep(i, c) * scale / (1 - p) (rowvec.h).  An id outside [0, num_rows) is
// padding: a row of zeros, no gradient.
//
// Lookup: bound by memory (n rows read, n rows written past the cache).  Wide 16-bit rows get a block each;
// else the batch is one flat list of pieces of eight columns, two 16-byte loads a thread.  32 768 rows of
// 4 096 bfloat16 with dropout: 67 us, 268 MB written and 97 MB of distinct rows read.
//
// Gradient: every row of the dense gradient is written once (those that the sort's launches zero ahead are written
// again where their token occurs), n rows of g are read once; sums are held in float32 and their order is fixed by
// (n, dim) and the sorted tokens, so results are the same from run to run.  Three parts:
//   tokens  positions in token order (stable) and row_start[v] = first of token v: one kernel for up to
//           4 096 ids, two for up to 131 072, beyond that and for tables of more than 2^20 rows the
//           library's radix sort.  Blocks of the same launches write zeros meanwhile.
//   sum     chunks of 8, 16 or 32 sorted positions, whatever the tokens' frequencies: one lane
//           group walks the rows of a chunk for its columns and writes every token that begins in the
//           chunk and ends there or in the next one, whose first rows it then takes too.  A longer
//           token leaves a partial row in every chunk that it touches.  Further blocks of the same
//           launch write the zeros of the tokens that do not occur.
//   join    adds the partial rows of the long tokens, in chunk order.
// 32 768 x 4 096 bfloat16 into 131 072 rows: 235 us for 1.34 GB (5.7 TB/s), of it tokens 6 + 14 (with 80 MiB of the
// zeros), sum 203, join 9; 2 048 x 1 024 float32 into 32 000 rows: 31 us for 139 MB, of it tokens 8, sum 19, join 4.
#include "internal.h"
#include "rowvec.h"

namespace hades {
namespace {

constexpr int kThreads = 256;
constexpr int kZeroUnits = 2;   // 16-byte units a thread zeroes (1.07 GB: 164 us; 1 or 4 units 203)

// ---- lookup -------------------------------------------------------------------------------------
// pieces of a thread: two 16-byte loads, whatever the type
template <typename T>
constexpr int embed_pieces() { return sizeof(T) == 2 ? 2 : 1; }

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
  constexpr int kPieces = embed_pieces<T>();
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
    store8<T, true>(a.out + row[k] * a.dim + static_cast<int64_t>(piece[k]) * kPiece, y, valid[k]);
  }
}

// A block a row, for wide 16-bit rows: row and id are the same for all lanes, so what depends on them is scalar
// work.  With dropout the flat list's 129 vector instructions a piece take as long as memory does.
template <typename T, typename I>
__global__ __launch_bounds__(1024) void embed_row_kernel(EmbedArgs<T, I> a) {
  constexpr int kPieces = embed_pieces<T>();
  const DropKeys keys(a.drop);
  const int64_t row = blockIdx.x;
  const int64_t id = static_cast<int64_t>(a.ids[row]);
  const bool live = static_cast<uint64_t>(id) < static_cast<uint64_t>(a.num_rows);
  const T* const from = a.weight + (live ? id : 0) * a.stride;
  T* const to = a.out + row * a.dim;
  const int dim = static_cast<int>(a.dim);
  const int pieces = static_cast<int>(a.per_row.d), step = blockDim.x;
  for (int first = threadIdx.x; first < pieces; first += step * kPieces) {
    typename Vec8<T>::V v[kPieces];
    int valid[kPieces];
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int piece = first + k * step;
      valid[k] = piece < pieces ? (dim - piece * kPiece < kPiece ? dim - piece * kPiece : kPiece) : 0;
      v[k] = load8_raw(from + piece * kPiece, live ? valid[k] : 0);
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int piece = first + k * step;
      f32x8 y = __builtin_convertvector(v[k], f32x8);
      y = keys.on() ? keys.apply(y, static_cast<uint32_t>(row), static_cast<uint32_t>(piece)) : y * keys.factor;
      store8<T, true>(to + piece * kPiece, y, valid[k]);
    }
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
  // us without / with dropout, flat list against a block a row: 32 768 rows of 4 096 bfloat16 72 / 84 against 63 / 69,
  // 65 536 rows of 1 024 31 / 32 either way, of 640 20 / 21 against 21 / 26; 16 384 rows of 2 048 float32 41 against 44
  if constexpr (sizeof(T) == 2) {
    if (per_row >= 2 * kWave && n < (int64_t(1) << 22) && dim < (int64_t(1) << 27)) {
      const int64_t block = ceil_div(ceil_div(per_row, embed_pieces<T>()), kWave) * kWave;
      HADES_LAUNCH((embed_row_kernel<T, I>), dim3(static_cast<unsigned>(n)),
                   dim3(static_cast<unsigned>(block < 1024 ? block : 1024)), 0, st, a);
      return HADES_OK;
    }
  }
  const int64_t blocks = ceil_div(a.pieces, int64_t(kThreads) * embed_pieces<T>());
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

// Two kernels sort a batch of up to kTiles tiles: the first groups every tile's positions by bucket (a range
// of 2^shift tokens), the second gives every bucket a block that fetches its pieces of all tiles and puts them
// in token order.  Neither needs another block's result of the same launch, so the sort is two short launches
// where the radix sort makes six to nine that wait for one another.
constexpr int kTileIds = 1024;      // ids of a tile, a thread each
constexpr int kTileWaves = kTileIds / kWave;
constexpr int kTiles = 128;
constexpr int kMinBucketBits = 8;   // a block for every compute unit
constexpr int kMaxBucketBits = 10;
constexpr int kMaxShift = 10;

// The sort's launches leave most of the chip's memory bandwidth idle: blocks from `from` on write zeros over the
// first rows of a dense gradient meanwhile, whether their tokens occur or not (the sums come later).
struct ZeroJob {
  char* p;         // 16-byte aligned
  int64_t bytes;   // a multiple of 16
  unsigned from;
};
constexpr int kZeroJobUnits = 2;   // 16-byte units a thread
constexpr int64_t kZeroJobBlock = int64_t(kTileIds) * kZeroJobUnits * 16;

// true: the block belonged to the job
__device__ __forceinline__ bool zero_job(const ZeroJob& z) {
  if (blockIdx.x < z.from) return false;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 zero = {0, 0, 0, 0};
  const int64_t first = static_cast<int64_t>(blockIdx.x - z.from) * kZeroJobBlock + threadIdx.x * 16;
#pragma unroll
  for (int k = 0; k < kZeroJobUnits; ++k) {
    const int64_t at = first + k * (kTileIds * 16);
    if (at < z.bytes) __builtin_nontemporal_store(zero, reinterpret_cast<u32x4*>(z.p + at));
  }
  return true;
}

// lanes of the wave whose value agrees with the lane's in the low `bits` bits, among `of`
__device__ __forceinline__ uint64_t peers_of(uint32_t v, int bits, uint64_t of) {
  for (int b = 0; b < bits; ++b) {
    const bool one = (v >> b) & 1u;
    const uint64_t ones = __ballot(one);
    of &= one ? ones : ~ones;
  }
  return of;
}

// tok / pos [tile][kTileIds]: the tile's tokens and their positions, grouped by bucket in order of position;
// offsets[bucket][tile]: where a bucket begins in its tile, [buckets][tile]: the tile's number of tokens
template <typename I>
__global__ __launch_bounds__(kTileIds) void token_tile_kernel(const I* __restrict__ ids, int64_t n, int64_t num_rows,
                                                              int64_t padding, int shift, int bits, int tiles,
                                                              uint32_t* __restrict__ tok, uint32_t* __restrict__ pos,
                                                              uint32_t* __restrict__ offsets, ZeroJob zero) {
  if (zero_job(zero)) return;
  extern __shared__ uint32_t counts[];   // [kTileWaves][2^bits]
  __shared__ uint32_t scan[kTileWaves + 1];
  const int buckets = 1 << bits;
  const int wave = threadIdx.x / kWave;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kTileIds + threadIdx.x;
  const int64_t id = i < n ? static_cast<int64_t>(ids[i]) : int64_t(-1);
  const bool real = static_cast<uint64_t>(id) < static_cast<uint64_t>(num_rows) && id != padding;
  const uint32_t bucket = real ? static_cast<uint32_t>(id) >> shift : 0u;
  for (int k = threadIdx.x; k < kTileWaves * buckets; k += kTileIds) counts[k] = 0;
  __syncthreads();
  const uint64_t peers = peers_of(bucket, bits, __ballot(real));
  const uint32_t rank = ballot_rank(peers);
  if (real && rank == 0) counts[wave * buckets + bucket] = static_cast<uint32_t>(__popcll(peers));
  __syncthreads();
  uint32_t total = 0;
  if (threadIdx.x < static_cast<uint32_t>(buckets)) {
    for (int w = 0; w < kTileWaves; ++w) {
      const uint32_t c = counts[w * buckets + threadIdx.x];
      counts[w * buckets + threadIdx.x] = total;
      total += c;
    }
  }
  uint32_t all;
  const uint32_t start = block_exclusive_sum<uint32_t, kTileIds>(total, scan, &all);
  if (threadIdx.x < static_cast<uint32_t>(buckets)) {
    offsets[static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x] = start;
    for (int w = 0; w < kTileWaves; ++w) counts[w * buckets + threadIdx.x] += start;
  }
  if (threadIdx.x == 0) offsets[static_cast<int64_t>(buckets) * tiles + blockIdx.x] = all;
  __syncthreads();
  if (real) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kTileIds + counts[wave * buckets + bucket] + rank;
    tok[at] = static_cast<uint32_t>(id);
    pos[at] = static_cast<uint32_t>(i);
  }
}

__global__ __launch_bounds__(kTileIds) void token_bucket_kernel(const uint32_t* __restrict__ tok,
                                                                const uint32_t* __restrict__ pos,
                                                                const uint32_t* __restrict__ offsets, int tiles,
                                                                int64_t num_rows, int shift,
                                                                uint32_t* __restrict__ perm,
                                                                uint32_t* __restrict__ token,
                                                                uint32_t* __restrict__ row_start, ZeroJob zero) {
  if (zero_job(zero)) return;
  extern __shared__ uint32_t counts[];   // [kTileWaves][2^shift]
  __shared__ uint32_t scan[kTileWaves + 1];
  __shared__ uint32_t first[kTiles];     // of the bucket's list, in order of position: a tile's first entry
  __shared__ uint32_t place[kTiles];     // entry e of tile t is tok[place[t] + e]
  const int range = 1 << shift;
  const uint32_t v0 = blockIdx.x << shift;
  const uint32_t rows = static_cast<uint32_t>(num_rows);
  const uint32_t mine = rows - v0 < static_cast<uint32_t>(range) ? rows - v0 : static_cast<uint32_t>(range);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  uint32_t begin = 0, size = 0;
  if (static_cast<int>(threadIdx.x) < tiles) {
    begin = offsets[static_cast<int64_t>(blockIdx.x) * tiles + threadIdx.x];
    size = offsets[static_cast<int64_t>(blockIdx.x + 1) * tiles + threadIdx.x] - begin;
  }
  for (int k = threadIdx.x; k < kTileWaves * range; k += kTileIds) counts[k] = 0;
  uint32_t list, base;   // length of the bucket's list, and tokens of the buckets below
  const uint32_t entry = block_exclusive_sum<uint32_t, kTileIds>(size, scan, &list);
  block_exclusive_sum<uint32_t, kTileIds>(begin, scan, &base);
  if (static_cast<int>(threadIdx.x) < tiles) {
    first[threadIdx.x] = entry;
    place[threadIdx.x] = threadIdx.x * kTileIds + begin - entry;
  }
  __syncthreads();
  // a wave takes a stretch of the list, so that places by wave, step and lane keep the order of positions
  volatile uint32_t* const own = counts + wave * range;   // lanes read what other lanes of the wave wrote
  const uint32_t part = (list + kTileIds - 1) / kTileIds * kWave;
  const uint32_t lo = wave * part, hi = lo + part < list ? lo + part : list;
  const auto where = [&](uint32_t e) {   // in tok and pos: the last tile whose first entry is not above e
    int a = 0, b = tiles;
    while (b - a > 1) {
      const int mid = (a + b) >> 1;
      if (first[mid] <= e) a = mid; else b = mid;
    }
    return place[a] + e;
  };
  for (uint32_t e = lo + lane; e - lane < hi; e += kWave) {
    const bool in = e < hi;
    const uint32_t at = in ? tok[where(e)] - v0 : 0u;
    const uint64_t peers = peers_of(at, shift, __ballot(in));
    if (in && ballot_rank(peers) == 0) own[at] = own[at] + static_cast<uint32_t>(__popcll(peers));
  }
  __syncthreads();
  // a thread a token: the waves' counts become their first places
  uint32_t total = 0;
  if (threadIdx.x < mine) {
    for (int w = 0; w < kTileWaves; ++w) {
      const uint32_t c = counts[w * range + threadIdx.x];
      counts[w * range + threadIdx.x] = total;
      total += c;
    }
  }
  const uint32_t start = base + block_exclusive_sum<uint32_t, kTileIds>(total, scan, &total);
  if (threadIdx.x < mine) {
    row_start[v0 + threadIdx.x] = start;
    for (int w = 0; w < kTileWaves; ++w) counts[w * range + threadIdx.x] += start;
  }
  if (v0 + mine == rows && threadIdx.x == 0) row_start[rows] = base + list;
  __syncthreads();
  for (uint32_t e = lo + lane; e - lane < hi; e += kWave) {
    const bool in = e < hi;
    const uint32_t from = in ? where(e) : 0u;
    const uint32_t at = in ? tok[from] - v0 : 0u;
    const uint64_t peers = peers_of(at, shift, __ballot(in));
    const uint32_t rank = ballot_rank(peers);
    if (in) {
      const uint32_t to = own[at];
      perm[to + rank] = pos[from];
      token[to + rank] = v0 + at;
      if (rank == 0) own[at] = to + static_cast<uint32_t>(__popcll(peers));
    }
  }
}

// A batch of a few ids a thread without the first kernel: the block of a bucket looks at all ids itself, a wave at
// 64 * kSmallSteps of them one after another.  us of the whole gradient with this kernel / with two, bfloat16:
// 1 500 x 128 into 32 000 rows 17.3 / 22.3, 3 000 x 512 into 32 000 19.7 / 24.4, 4 096 x 1 024 into 32 000
// 22.7 / 27.6; with eight steps a wave 8 192 x 128 into 32 000 takes 24.8 / 25.4, 6 000 x 512 float32 into
// 50 257 34.8 / 30.7.
constexpr int kSmallSteps = 4;
constexpr int64_t kSmallIds = int64_t(kTileIds) * kSmallSteps;

template <typename I>
__global__ __launch_bounds__(kTileIds) void token_small_kernel(const I* __restrict__ ids, int64_t n, int64_t num_rows,
                                                               int64_t padding, int shift, uint32_t* __restrict__ perm,
                                                               uint32_t* __restrict__ token,
                                                               uint32_t* __restrict__ row_start, ZeroJob zero) {
  if (zero_job(zero)) return;
  extern __shared__ uint32_t counts[];   // [kTileWaves][2^shift]
  __shared__ uint32_t scan[kTileWaves + 1];
  const int range = 1 << shift;
  const uint32_t v0 = blockIdx.x << shift;
  const uint32_t rows = static_cast<uint32_t>(num_rows);
  const uint32_t mine = rows - v0 < static_cast<uint32_t>(range) ? rows - v0 : static_cast<uint32_t>(range);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  // every wave takes as many steps, so that places by wave, step and lane keep the order of positions
  const int steps = static_cast<int>((n + kTileIds - 1) / kTileIds);
  const uint32_t from = wave * steps * kWave + lane;
  int64_t id[kSmallSteps];
#pragma unroll
  for (int k = 0; k < kSmallSteps; ++k)
    id[k] = k < steps && from + k * kWave < n ? static_cast<int64_t>(ids[from + k * kWave]) : int64_t(-1);
  for (int k = threadIdx.x; k < kTileWaves * range; k += kTileIds) counts[k] = 0;
  uint32_t below = 0;
  uint32_t at[kSmallSteps];
  bool in[kSmallSteps];
#pragma unroll
  for (int k = 0; k < kSmallSteps; ++k) {
    const bool real = static_cast<uint64_t>(id[k]) < static_cast<uint64_t>(num_rows) && id[k] != padding;
    at[k] = static_cast<uint32_t>(id[k]) - v0;
    in[k] = real && at[k] < mine;
    if (!in[k]) at[k] = 0;
    below += real && static_cast<uint32_t>(id[k]) < v0;
  }
  uint32_t base;   // tokens below the range
  block_exclusive_sum<uint32_t, kTileIds>(below, scan, &base);
  volatile uint32_t* const own = counts + wave * range;   // lanes read what other lanes of the wave wrote
  uint64_t peers[kSmallSteps];
#pragma unroll
  for (int k = 0; k < kSmallSteps; ++k) {
    peers[k] = __ballot(in[k]);
    if (peers[k] == 0) continue;   // (the same for the whole wave)
    peers[k] = peers_of(at[k], shift, peers[k]);
    if (in[k] && ballot_rank(peers[k]) == 0) own[at[k]] = own[at[k]] + static_cast<uint32_t>(__popcll(peers[k]));
  }
  __syncthreads();
  uint32_t total = 0;
  if (threadIdx.x < mine) {
    for (int w = 0; w < kTileWaves; ++w) {
      const uint32_t c = counts[w * range + threadIdx.x];
      counts[w * range + threadIdx.x] = total;
      total += c;
    }
  }
  uint32_t all;
  const uint32_t start = base + block_exclusive_sum<uint32_t, kTileIds>(total, scan, &all);
  if (threadIdx.x < mine) {
    row_start[v0 + threadIdx.x] = start;
    for (int w = 0; w < kTileWaves; ++w) counts[w * range + threadIdx.x] += start;
  }
  if (v0 + mine == rows && threadIdx.x == 0) row_start[rows] = base + all;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSmallSteps; ++k) {
    if (!in[k]) continue;
    const uint32_t rank = ballot_rank(peers[k]);
    const uint32_t to = own[at[k]];
    perm[to + rank] = from + k * kWave;
    token[to + rank] = v0 + at[k];
    if (rank == 0) own[at[k]] = to + static_cast<uint32_t>(__popcll(peers[k]));
  }
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
// Sorted positions of a chunk: the fewer, the more waves and the more partial rows.  us of the whole
// gradient with chunks of 8 / 16 / 32: 16 384 rows of 1 024 bfloat16 into 32 000: 44 / 39 / -, 65 536 rows of 999
// float32: 150 / 135 / 144, 32 768 rows of 4 096 bfloat16 into 131 072: - / 244 / 237.
constexpr int kChunkShort = 8;
constexpr int kChunk = 16;
constexpr int kChunkLong = 32;
constexpr int64_t kChunkWaves = 2048;       // waves that chunks of kChunk have to give
constexpr int64_t kChunkLongWaves = 8192;   // ... and of kChunkLong

struct GradPlan {
  int group;        // lanes that walk a chunk's rows together: 8, 16, 32 or 64
  int slices;       // groups side by side along a row
  int chunk;
  int reach;        // chunks that a token may touch before it is a long one
  int64_t chunks;
  int64_t pieces;   // of a row
};

GradPlan plan_grad(int64_t n, int64_t dim) {
  GradPlan p;
  p.pieces = ceil_div(dim, kPiece);
  p.group = 8;
  while (p.group < kWave && p.group < p.pieces) p.group *= 2;
  p.slices = static_cast<int>(ceil_div(p.pieces, p.group));
  const auto waves = [&](int chunk) { return ceil_div(ceil_div(n, chunk) * p.slices * p.group, kWave); };
  p.chunk = waves(kChunkLong) >= kChunkLongWaves ? kChunkLong : (waves(kChunk) >= kChunkWaves ? kChunk : kChunkShort);
  p.chunks = ceil_div(n, p.chunk);
  // a batch of up to 64 positions has no long tokens and needs no join
  p.reach = p.chunks <= 8 && p.chunk == kChunkShort ? 8 : 2;
  return p;
}

template <typename T, typename O>
struct GradArgs {
  const T* grad;
  const uint32_t* perm;        // batch position of every sorted position
  const uint32_t* token;       // its token
  const uint32_t* row_start;   // [num_rows + 1]
  O* out;
  float* partial;              // [2 * chunks][partial_stride], see is_long
  int64_t grad_stride, out_stride, partial_stride, num_rows, dim, chunks;
  int slices, accumulate, reach;
  int once;                    // rows of grad: see streamed
  unsigned sum_blocks;
  FastDiv per_row, per_chunk;
  int64_t zero_units, zero_from;   // rows from zero_from on
  DropArgs drop;
};

template <typename T, typename O>
__device__ __forceinline__ void put_row(const GradArgs<T, O>& a, uint32_t token, int64_t col, f32x8 v, int valid) {
  O* p = a.out + static_cast<int64_t>(token) * a.out_stride + col;
  if (a.accumulate) v += load8(p, valid);
  store8(p, v, valid);
}

// a token whose rows reach beyond `reach` chunks, the one that it begins in among them
template <int CH>
__device__ __forceinline__ bool is_long(int64_t begin, int64_t end, int reach) { return end > (begin / CH + reach) * CH; }

template <typename T, typename O, int G, int CH>
__global__ __launch_bounds__(kThreads) void embed_grad_sum_kernel(GradArgs<T, O> a) {
  if (blockIdx.x >= a.sum_blocks) {
    // the rows of tokens that do not occur, in units of 16 bytes that are aligned whatever the rows are: the
    // first and the last unit of a row may be part of one
    constexpr int kUnit = 16 / sizeof(O);
    typedef O UnitV __attribute__((ext_vector_type(kUnit)));
    const int64_t first = static_cast<int64_t>(blockIdx.x - a.sum_blocks) * (kThreads * kZeroUnits);
    const int64_t row0 = a.zero_units < (int64_t(1) << 31) ? int64_t(a.per_row.div(uint32_t(first)))
                                                           : first / a.per_row.d;
    const uint32_t rest = static_cast<uint32_t>(first - row0 * a.per_row.d);
#pragma unroll
    for (int k = 0; k < kZeroUnits; ++k) {
      if (first + threadIdx.x + k * kThreads >= a.zero_units) break;
      const uint32_t at = rest + threadIdx.x + k * kThreads;
      const uint32_t down = a.per_row.div(at);
      const int64_t v = a.zero_from + row0 + down;
      if (a.row_start[v] != a.row_start[v + 1]) continue;
      O* const row = a.out + v * a.out_stride;
      const int64_t skew = static_cast<int64_t>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(O));
      const int64_t col = static_cast<int64_t>(at - down * a.per_row.d) * kUnit - skew;
      if (col >= 0 && a.dim - col >= kUnit) {
        UnitV zero;
#pragma unroll
        for (int j = 0; j < kUnit; ++j) zero[j] = static_cast<O>(0.0f);
        __builtin_nontemporal_store(zero, reinterpret_cast<UnitV*>(row + col));
      } else {
        for (int j = 0; j < kUnit; ++j)
          if (col + j >= 0 && col + j < a.dim) row[col + j] = static_cast<O>(0.0f);
      }
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
  int64_t p0 = static_cast<int64_t>(chunk) * CH;
  if (p0 >= live || valid == 0) return;
  int64_t p1 = p0 + CH < live ? p0 + CH : live;
  // the chunk's first token began before it: the chunk before takes all of it, or it is a long one
  uint32_t cur = a.token[p0];
  bool part = false;   // the token summed now is a long one: its row is partial
  {
    const int64_t begin = a.row_start[cur], end = a.row_start[cur + 1];
    if (is_long<CH>(begin, end, a.reach)) part = true;
    else if (begin < p0) p0 = end;
  }
  // ... and the last one goes on behind it: taken to its end, unless it is long
  const uint32_t last = a.token[p1 - 1];
  const int64_t last_begin = a.row_start[last], last_end = a.row_start[last + 1];
  if (last_begin >= static_cast<int64_t>(chunk) * CH && !is_long<CH>(last_begin, last_end, a.reach)) p1 = last_end;
  if (p0 >= p1) return;
  cur = a.token[p0];
  const f32x8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  f32x8 acc = zero;
  // slot 0: a long token that began earlier; slot 1: one that begins here
  float* const slot = a.partial + 2 * static_cast<int64_t>(chunk) * a.partial_stride + col;
  const int len = static_cast<int>(p1 - p0);
  for (int t = 0; t < len; t += U) {
    typename Vec8<T>::V row[U];
    uint32_t tok[U], pos[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t j = p0 + (t + k < len ? t + k : len - 1);   // the last row again behind the end: not added
      pos[k] = a.perm[j];
      tok[k] = a.token[j];
    }
    if (a.once) {
#pragma unroll
      for (int k = 0; k < U; ++k)
        row[k] = load8_raw<T, true>(a.grad + static_cast<int64_t>(pos[k]) * a.grad_stride + col, valid);
    } else {
#pragma unroll
      for (int k = 0; k < U; ++k)
        row[k] = load8_raw<T>(a.grad + static_cast<int64_t>(pos[k]) * a.grad_stride + col, valid);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (t + k >= len) break;
      if (tok[k] != cur) {
        if (part) store8(slot, acc, kPiece);   // (only the chunk's first token can end here as a long one)
        else put_row(a, cur, col, acc, valid);
        acc = zero;
        cur = tok[k];
        part = false;
      }
      const f32x8 v = __builtin_convertvector(row[k], f32x8);
      acc += keys.on() ? keys.apply(v, pos[k], piece) : v * keys.factor;
    }
  }
  if (part || (cur == last && is_long<CH>(last_begin, last_end, a.reach))) {
    const bool begins = static_cast<int64_t>(a.row_start[cur]) >= static_cast<int64_t>(chunk) * CH;
    store8(slot + (begins ? a.partial_stride : 0), acc, kPiece);
  } else {
    put_row(a, cur, col, acc, valid);
  }
}

// A block looks at kJoinChunks chunks for long tokens that begin in them, one a lane group at a time, and
// adds their partial rows for one slice of columns.  A token of more than kJoinAlone parts is left to the
// whole block: its groups take the parts in turn, and their sums are added in order.
constexpr int kJoinThreads = 512;
constexpr int kJoinChunks = 8;    // at most kJoinThreads / 64
constexpr int kJoinAlone = 32;

template <typename T, typename O, int G, int CH>
__global__ __launch_bounds__(kJoinThreads) void embed_grad_join_kernel(GradArgs<T, O> a) {
  constexpr int kGroups = kJoinThreads / G;
  constexpr int U = 8;
  __shared__ f32x8 sums[kJoinThreads];
  __shared__ uint32_t token_of[kJoinChunks];
  __shared__ int parts_of[kJoinChunks];   // 0: no long token begins in the chunk
  const int64_t live = a.row_start[a.num_rows];
  const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kJoinChunks;
  if (threadIdx.x < kJoinChunks) {
    const int64_t c = c0 + threadIdx.x, border = (c + 1) * CH;
    int parts = 0;
    if (border < live) {
      const uint32_t token = a.token[border - 1];
      const int64_t begin = a.row_start[token], end = a.row_start[token + 1];
      if (begin >= c * CH && is_long<CH>(begin, end, a.reach)) parts = static_cast<int>((end - 1) / CH - c + 1);
      token_of[threadIdx.x] = token;
    }
    parts_of[threadIdx.x] = parts;
  }
  __syncthreads();
  const int group = threadIdx.x / G, lane = threadIdx.x & (G - 1);
  const int64_t col = (static_cast<int64_t>(blockIdx.y) * G + lane) * kPiece;
  const int64_t left = a.dim - col;
  const int valid = left < 0 ? 0 : (left < kPiece ? static_cast<int>(left) : kPiece);
  // parts at, at + step, ... of the token that begins in chunk c
  const auto sum = [&](int64_t c, int parts, int at, int step) {
    f32x8 acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int t = at; t < parts; t += step * U) {
      f32x8 row[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int s = t + k * step;
        const int64_t slot = s == 0 ? 2 * c + 1 : 2 * (c + s);
        row[k] = load8(a.partial + (s < parts ? slot * a.partial_stride + col : 0), s < parts && valid > 0 ? kPiece : 0);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) acc += row[k];
    }
    return acc;
  };
  if (group < kJoinChunks) {
    const int parts = parts_of[group];
    if (parts > 0 && parts <= kJoinAlone) put_row(a, token_of[group], col, sum(c0 + group, parts, 0, 1), valid);
  }
  for (int i = 0; i < kJoinChunks; ++i) {
    const int parts = parts_of[i];
    if (parts <= kJoinAlone) continue;   // (the same for all threads of the block)
    f32x8 acc = sum(c0 + i, parts, group, kGroups);
    sums[threadIdx.x] = acc;
    __syncthreads();
    if (group == 0 && valid > 0) {
      for (int g = 1; g < kGroups; ++g) acc += sums[g * G + lane];
      put_row(a, token_of[i], col, acc, valid);
    }
    __syncthreads();
  }
}

inline size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

// Whether the two bucket kernels sort the batch, and with which buckets.  Kernel times in us against the radix
// sort's (keys, passes, row_start), ids of a power law out of 50 000: 8 192 ids 12 / 25, 32 768 17 / 28, 131 072
// 35 / 37, 524 288 122 / 52 (the block of the most frequent token's bucket takes the longest: a power law puts
// a tenth of the ids into it); out of 262 144: 15 / 34, 16 / 40, 36 / 51, 115 / 70.
struct BucketPlan {
  bool use, small;   // small: one kernel
  int bits, shift;   // 2^bits buckets of 2^shift tokens
  int64_t tiles, buckets;
};

BucketPlan plan_buckets(int64_t n, int64_t num_rows) {
  BucketPlan b;
  const int bits = ilog2_ceil(static_cast<uint64_t>(num_rows));
  b.bits = bits - kMaxShift < kMinBucketBits ? kMinBucketBits : bits - kMaxShift;
  b.shift = bits - b.bits < 0 ? 0 : bits - b.bits;
  b.tiles = ceil_div(n, kTileIds);
  b.buckets = ceil_div(num_rows, int64_t(1) << b.shift);
  b.use = b.bits <= kMaxBucketBits && b.tiles <= kTiles;
  b.small = n <= kSmallIds;
  return b;
}

struct GradWs {
  void* sort;         // radix sort
  size_t sort_bytes;
  int64_t* keys;
  uint32_t* tile_tok; // bucket kernels
  uint32_t* tile_pos;
  uint32_t* offsets;
  uint32_t* perm;
  uint32_t* token;
  uint32_t* row_start;
  float* partial;
  size_t bytes;
};

GradWs carve_grad(void* base, int64_t n, int64_t dim, int64_t num_rows) {
  const GradPlan p = plan_grad(n, dim);
  const BucketPlan b = plan_buckets(n, num_rows);
  GradWs w = {};
  Carver c(base);
  if (b.use) {
    w.tile_tok = c.take<uint32_t>(b.tiles * kTileIds);
    w.tile_pos = c.take<uint32_t>(b.tiles * kTileIds);
    w.offsets = c.take<uint32_t>(((int64_t(1) << b.bits) + 1) * b.tiles);
    w.perm = c.take<uint32_t>(n);
    w.token = c.take<uint32_t>(n);
  } else {
    w.sort_bytes = round256(sort_ids_workspace_bytes(n));
    w.sort = c.take<char>(w.sort_bytes);
    w.keys = c.take<int64_t>(n);
  }
  w.row_start = c.take<uint32_t>(num_rows + 1);
  w.partial = c.take<float>(2 * p.chunks * p.pieces * kPiece);
  w.bytes = c.total();
  return w;
}

// What the sort's launches zero of a dense gradient: as much as memory takes beside them, of a gradient that
// has at least a row for each position of the batch.  us of the whole gradient with 0 / 20 + 36 / 30 + 50 / 60 +
// 100 MiB: 12 289 x 1 001 float16 into 50 257
// 47.5 / 40.9 / 38.5 / 43.2, 512 x 1 024 bfloat16 into 32 000 21.0 / 18.7 / 17.8 / 21.7.
struct EarlyZeros {
  int64_t rows;           // the first rows of the gradient
  ZeroJob first, second;
};
constexpr int64_t kZeroFirst = int64_t(30) << 20, kZeroSecond = int64_t(50) << 20;   // bytes
// beside the one kernel of a small batch with more than one step a wave, which takes longer; with 30 / 40 / 50 MiB:
// 2 048 x 1 024 float32 into 32 000 rows 32.4 / 31.0 / 31.7, 4 096 x 1 024 bfloat16 23.2 / 22.7 / 23.1; with one
// step, 1 000 x 1 024 bfloat16, 18.6 / 19.1 / 20.9
constexpr int64_t kZeroSmall = int64_t(40) << 20;

EarlyZeros plan_zeros(void* out, int64_t out_stride, int64_t n, int64_t num_rows, int64_t dim, int64_t value_bytes,
                      int accumulate, const BucketPlan& b) {
  EarlyZeros z = {};
  z.first.from = z.second.from = ~0u;
  if (!b.use || accumulate || out_stride != dim || (align_of_ptr(out) & 15) != 0 || n > num_rows) return z;
  const int64_t row = dim * value_bytes;
  const int64_t alone = b.small && b.tiles > 1 ? kZeroSmall : kZeroFirst;   // of the first launch
  const int64_t most = b.small ? alone : kZeroFirst + kZeroSecond;
  z.rows = (most / row < num_rows ? most / row : num_rows) & ~int64_t(7);   // eight rows are a multiple of 16 bytes
  const int64_t bytes = z.rows * row;
  z.first.p = static_cast<char*>(out);
  z.first.bytes = bytes < alone ? bytes : alone;
  z.second.p = z.first.p + z.first.bytes;
  z.second.bytes = bytes - z.first.bytes;
  return z;
}

// the job behind the `blocks` blocks of a launch; returns the launch's blocks
unsigned with_zeros(ZeroJob* z, int64_t blocks) {
  z->from = static_cast<unsigned>(blocks);
  return static_cast<unsigned>(blocks + ceil_div(z->bytes, kZeroJobBlock));
}

// positions in token order, their tokens, and row_start
template <typename I>
int sort_tokens(const I* ids, int64_t n, int64_t rows, int64_t num_rows, int64_t padding, const GradWs& w,
                EarlyZeros& z, const uint32_t** perm, const uint32_t** token, hipStream_t st) {
  const BucketPlan b = plan_buckets(rows, num_rows);
  if (b.use && b.small) {
    const dim3 grid(with_zeros(&z.first, b.buckets));
    HADES_LAUNCH((token_small_kernel<I>), grid, dim3(kTileIds), (kTileWaves << b.shift) * sizeof(uint32_t), st, ids, n,
                 num_rows, padding, b.shift, w.perm, w.token, w.row_start, z.first);
    *perm = w.perm;
    *token = w.token;
    return HADES_OK;
  }
  if (b.use) {
    const dim3 grid(with_zeros(&z.first, b.tiles)), bgrid(with_zeros(&z.second, b.buckets));
    HADES_LAUNCH((token_tile_kernel<I>), grid, dim3(kTileIds), (kTileWaves << b.bits) * sizeof(uint32_t), st, ids, n,
                 num_rows, padding, b.shift, b.bits, static_cast<int>(b.tiles), w.tile_tok, w.tile_pos, w.offsets,
                 z.first);
    HADES_LAUNCH(token_bucket_kernel, bgrid, dim3(kTileIds), (kTileWaves << b.shift) * sizeof(uint32_t), st, w.tile_tok,
                 w.tile_pos, w.offsets, static_cast<int>(b.tiles), num_rows, b.shift, w.perm, w.token, w.row_start,
                 z.second);
    *perm = w.perm;
    *token = w.token;
    return HADES_OK;
  }
  const dim3 block(kThreads);
  HADES_LAUNCH((token_key_kernel<I>), dim3(static_cast<unsigned>(ceil_div(rows, kThreads))), block, 0, st, ids, n, rows,
               num_rows, padding, w.keys);
  SortResult sr;
  const int rc = sort_ids(w.keys, rows, num_rows + 1, w.sort, w.sort_bytes, st, &sr);
  if (rc != HADES_OK) return rc;
  HADES_REQUIRE(!sr.key64, "internal: token keys must be 32-bit");
  *perm = sr.perm;
  *token = static_cast<const uint32_t*>(sr.sorted_keys);
  HADES_LAUNCH(row_start_kernel, dim3(static_cast<unsigned>(ceil_div(num_rows + 1, kThreads))), block, 0, st, *token,
               rows, num_rows, w.row_start);
  return HADES_OK;
}

// Blocks of the sums and of the zeros behind them, and whether their launch and the join's fit HIP's limits: fewer
// than 2^32 threads along a dimension, at most 65 535 blocks along y.  (The join's x has 64 threads a chunk: below
// 2^31, as a batch of 2^28 positions or more has chunks of 32.)
struct SumGrid {
  int64_t sum_blocks, zero_blocks;
  bool fits;
};

SumGrid plan_sum_grid(const GradPlan& p, int64_t zero_units) {
  SumGrid g;
  g.sum_blocks = ceil_div(p.chunks * p.slices * p.group, kThreads);
  g.zero_blocks = ceil_div(zero_units, int64_t(kThreads) * kZeroUnits);
  g.fits = g.sum_blocks + g.zero_blocks < (int64_t(1) << 24) && (p.chunks <= p.reach || p.slices <= 65535);
  return g;
}

// 16-byte units of the rows that the sums' launch zeroes (where their tokens do not occur); one more unit a row
// where a row may begin inside one
int64_t zero_units_of_row(const void* out, int64_t out_stride, int64_t dim, int64_t value_bytes) {
  const int64_t unit = 16 / value_bytes;
  const bool aligned = (align_of_ptr(out) & 15) == 0 && out_stride % unit == 0;
  return ceil_div(dim, unit) + (aligned ? 0 : 1);
}

template <typename T, typename O, int G, int CH>
int launch_sums(GradArgs<T, O>& a, const GradPlan& p, const SumGrid& g, hipStream_t st) {
  a.sum_blocks = static_cast<unsigned>(g.sum_blocks);
  if (g.sum_blocks + g.zero_blocks > 0)
    HADES_LAUNCH((embed_grad_sum_kernel<T, O, G, CH>), dim3(static_cast<unsigned>(g.sum_blocks + g.zero_blocks)),
                 dim3(kThreads), 0, st, a);
  if (p.chunks > p.reach)   // (there are no long tokens otherwise)
    HADES_LAUNCH((embed_grad_join_kernel<T, O, G, CH>),
                 dim3(static_cast<unsigned>(ceil_div(p.chunks, kJoinChunks)), static_cast<unsigned>(p.slices)),
                 dim3(kJoinThreads), 0, st, a);
  return HADES_OK;
}

template <typename T, typename O>
int launch_grad(const void* grad, int64_t grad_stride, const uint32_t* perm, const uint32_t* token, void* out,
                int64_t out_stride, int64_t n, int64_t num_rows, int64_t dim, const GradPlan& p, const GradWs& w,
                int accumulate, int64_t zero_from, int64_t zero_row, int64_t zero_units, const SumGrid& grid,
                const DropArgs& drop, hipStream_t st) {
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
  a.partial_stride = p.pieces * kPiece;   // whole pieces: aligned whatever dim is
  a.slices = p.slices;
  a.reach = p.reach;
  a.accumulate = accumulate;
  a.once = streamed(n * dim * static_cast<int64_t>(sizeof(T)));
  a.per_row = FastDiv(static_cast<uint32_t>(zero_row));
  a.per_chunk = FastDiv(static_cast<uint32_t>(p.slices));
  a.zero_units = zero_units;
  a.zero_from = zero_from;
  a.drop = drop;
#define HADES_SUMS(G_)                                                                   \
  do {                                                                                   \
    if (p.chunk == kChunkLong) return launch_sums<T, O, G_, kChunkLong>(a, p, grid, st); \
    if (p.chunk == kChunk) return launch_sums<T, O, G_, kChunk>(a, p, grid, st);         \
    return launch_sums<T, O, G_, kChunkShort>(a, p, grid, st);                           \
  } while (0)
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
  const uint32_t *perm = nullptr, *token = nullptr;
  const int64_t value_bytes = out_dtype == HADES_F32 ? 4 : 2;
  EarlyZeros zeros = plan_zeros(out, out_stride, rows, num_rows, dim, value_bytes, accumulate,
                                plan_buckets(rows, num_rows));
  const int64_t zero_row = zero_units_of_row(out, out_stride, dim, value_bytes);
  const int64_t zero_units = accumulate ? 0 : (num_rows - zeros.rows) * zero_row;
  const SumGrid grid = plan_sum_grid(plan, zero_units);
  HADES_REQUIRE(grid.fits, "embed_grad: too many values for one call");   // (before the first launch)
  const int rc = itype == HADES_I64
                     ? sort_tokens(static_cast<const int64_t*>(ids), n, rows, num_rows, padding_idx, w, zeros, &perm,
                                   &token, st)
                     : sort_tokens(static_cast<const int32_t*>(ids), n, rows, num_rows, padding_idx, w, zeros, &perm,
                                   &token, st);
  if (rc != HADES_OK) return rc;
#define HADES_GRAD(T_, O_)                                                                               \
  return launch_grad<T_, O_>(grad, grad_stride, perm, token, out, out_stride, n, num_rows, dim, plan, w, \
                             accumulate != 0, zeros.rows, zero_row, zero_units, grid, drop, st)
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
