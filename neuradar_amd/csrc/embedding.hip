// Rows of an embedding table, and the table's gradient.
//
//   rows      out[i, :] = round(scale * table[idx[i], :])                                     (nr_embedding_fwd)
//   gradient  g_table[v, :] (+)= round(scale * sum over i with idx[i] = v of g[i, :])         (nr_embedding_bwd)
//
// The gradient is a sum over equal indices.  Adding rows to the table as they come needs float atomics, whose order -- and with
// it the result -- changes from run to run, and a row that many tokens share becomes one queue at the memory side.  Here equal
// indices are brought together first, their positions in ascending order; then every sum is formed in registers in one fixed
// order and each touched row is written once.  Sums are held in 64 bits inside a block and in fp32 in the workspace; their order
// follows from the sizes, the types and the indices alone: two calls give the same bits.  Three ways, by sizes (make_own_plan,
// make_plan):
//   * up to 16 384 indices, one launch: a block owns a range of rows, picks its tokens out of all indices and orders them in LDS
//     (own_kernel);
//   * more indices and a table whose copies are small: the same on chunks of the indices, and a launch that adds the chunks' tables;
//   * else: (index, position) pairs are sorted, least significant digit first, digits of up to 11 bits (one pass for 2 047 rows,
//     two for 4 M), a count, a scan and a scatter per pass.  A block sums a fixed stretch of SORTED positions, whatever the
//     indices are -- a row that owns half of the batch is spread over as many blocks as its tokens need.  Groups of lanes walk
//     shorter stretches, 8 rows of g in flight each; a sum whose neighbours lie in other stretches goes through LDS to its first
//     group, one that leaves the block is left in the workspace and added up in block order by a last launch.
// Bound by memory where rows are long (read g once, write the table once), by the chain of launches and of dependent steps inside
// a block where they are few.  Measured, kernels alone: rows 262 144 x 1 024 bf16 114 us (0.69 GB of traffic: 6.0 TB/s; 153 us on
// a cold table); gradient 16 384 x 16 on 60 rows 11 us, 113 840 x 32 on 1 999 rows 19 + 4, 8 192 x 8 on 2^22 rows 26 (134 MB of
// zeros alone: 18), 100 003 x 257 on 7 rows 33 + 4 (103 MB: 20), 131 072 x 512 bf16 on 131 072 rows 109 (sort 45, which also
// writes the zeros; sums 54 at 3.2 TB/s; join 9).
#include <type_traits>

#include "rows_dev.h"

namespace {

constexpr int kMaxDim = 65536;
constexpr int kThreads = 256;
constexpr int kRounds = 4;                            // rounds of 64 tokens that a wave ranks in one tile of the sort
constexpr int kTile = kThreads * kRounds;             // tokens per block of the sort
constexpr int kMaxDigitBits = 11;
constexpr int64_t kZeroBlocks = 2048;                 // blocks of a launch that write zeros

// ---------------------------------------------------------------------------------------------------------------- rows
constexpr int kRowUnroll = 4;

// Flat over the 16-byte vectors of the output, four per thread: every lane has work whatever the width is.  Where dim is not a
// multiple of the vector a row's last one starts earlier and lies over the one before (both write the same values there), so that
// every access is a whole vector; only rows shorter than a vector are taken in pieces.  (200 000 rows of 13 fp16 values: 6.0 -> 4.6 us,
// 50 021 rows of 33 4.3 -> 3.7, against a last vector in pieces.)
template <typename T, typename I, bool STREAM>
__global__ void __launch_bounds__(kThreads)
rows_kernel(const T* __restrict__ table, int64_t rows, int dim, int64_t row_stride, const I* __restrict__ idx, int64_t n, float scale,
            T* __restrict__ out, int64_t out_stride, uint32_t nv, uint32_t magic) {
  constexpr int N = 16 / (int)sizeof(T);
  const int64_t base = (int64_t)blockIdx.x * (kThreads * kRowUnroll);
  const int64_t row0 = base / nv;
  const uint32_t rem0 = (uint32_t)(base - row0 * nv);
  int64_t r[kRowUnroll], v[kRowUnroll];
  int col[kRowUnroll];
#pragma unroll
  for (int u = 0; u < kRowUnroll; ++u) {
    const uint32_t l = rem0 + (uint32_t)(u * kThreads) + threadIdx.x;
    const uint32_t q = magic == 0u ? l : __umulhi(l, magic);
    r[u] = row0 + q;
    col[u] = max(min((int)(l - q * nv) * N, dim - N), 0);
    v[u] = r[u] < n ? (int64_t)idx[r[u]] : -1;
  }
  float x[kRowUnroll][N];
#pragma unroll
  for (int u = 0; u < kRowUnroll; ++u) {
    if (v[u] >= 0 && v[u] < rows) {
      const T* t = table + v[u] * row_stride + col[u];
      if (dim >= N) nr_load_pack<T, N>(t, x[u]);
      else nr_load_some<T, N>(t, dim, x[u]);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[u][k] = __builtin_nanf("");
    }
  }
#pragma unroll
  for (int u = 0; u < kRowUnroll; ++u) {
    if (r[u] >= n) continue;
#pragma unroll
    for (int k = 0; k < N; ++k) x[u][k] *= scale;
    T* o = out + r[u] * out_stride + col[u];
    if (dim < N) nr_store_some<T, N>(o, dim, x[u]);
    else if (STREAM) nr_store_pack_stream<T, N>(o, x[u]);
    else nr_store_pack<T, N>(o, x[u]);
  }
}

// thread t of `threads`: its share of `halves` 16-bit zeros at p
__device__ __forceinline__ void clear_halves(uint16_t* __restrict__ p, int64_t halves, int64_t t, int64_t threads) {
  typedef NrPack<uint16_t, 8> Pack;
  Pack* q = reinterpret_cast<Pack*>(p);
  const int64_t packs = halves / 8;
  int64_t i = t;
  for (; i + 3 * threads < packs; i += 4 * threads)
#pragma unroll
    for (int u = 0; u < 4; ++u) q[i + u * threads].v = (Pack::vec)(uint16_t)0;
  for (; i < packs; i += threads) q[i].v = (Pack::vec)(uint16_t)0;
  for (int64_t rest = packs * 8 + t; rest < halves; rest += threads) p[rest] = 0;
}

// ---------------------------------------------------------------------------------------------------------------- sort
struct SortPass {
  const uint32_t* keys;   // NULL: this pass reads the indices themselves
  const uint32_t* pos;
  uint32_t* keys_out;
  uint32_t* pos_out;
  uint32_t* counts;       // [blocks][digits]
  uint32_t* totals;       // [digits]
  int64_t n, rows, padding;
  int shift, bits;
  uint32_t blocks;
  // the result's zeros: a share of them with each launch of the sort, in blocks behind its own -- the sort waits for memory more
  // than it uses it (131 072 x 512 bf16: 21 us as a launch of its own)
  uint16_t* zeros;
  int64_t halves;
  uint32_t zero_blocks;
};

// Whether this block is one of those behind `blocks`, and its work is done.
__device__ __forceinline__ bool clears(const SortPass& s, uint32_t blocks) {
  if (blockIdx.x < blocks) return false;
  clear_halves(s.zeros, s.halves, (int64_t)(blockIdx.x - blocks) * kThreads + threadIdx.x, (int64_t)s.zero_blocks * kThreads);
  return true;
}

template <typename I>
__device__ __forceinline__ uint32_t key_of(const SortPass& s, const I* __restrict__ idx, int64_t i) {
  if (s.keys != nullptr) return s.keys[i];
  const int64_t v = (int64_t)idx[i];
  return (v >= 0 && v < s.rows && v != s.padding) ? (uint32_t)v : (uint32_t)s.rows;
}

template <typename I>
__global__ void __launch_bounds__(kThreads)
sort_count_kernel(SortPass s, const I* __restrict__ idx) {
  __shared__ uint32_t cnt[1 << kMaxDigitBits];
  if (clears(s, s.blocks)) return;
  const int digits = 1 << s.bits;
  const int64_t base = (int64_t)blockIdx.x * kTile;
  uint32_t key[kRounds];
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    const int64_t i = base + u * kThreads + threadIdx.x;
    key[u] = i < s.n ? key_of(s, idx, i) : 0u;
  }
  for (int d = threadIdx.x; d < digits; d += kThreads) cnt[d] = 0u;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kRounds; ++u)
    if (base + u * kThreads + threadIdx.x < s.n) atomicAdd(&cnt[(key[u] >> s.shift) & (uint32_t)(digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kThreads) s.counts[(int64_t)blockIdx.x * digits + d] = cnt[d];
}

// counts[b][d] -> tokens of digit d in blocks before b; totals[d].  A block takes 16 digits; 16 threads, one per digit, walk a
// sixteenth of the sort's blocks (neighbouring threads read neighbouring digits), the parts are then shifted by what lies before them.
constexpr int kScanDigits = 16;
__global__ void __launch_bounds__(kThreads)
sort_scan_kernel(SortPass s) {
  constexpr int kParts = kThreads / kScanDigits;  // parts of the blocks
  __shared__ uint32_t part[kParts][kScanDigits];
  const int digits = 1 << s.bits;
  if (clears(s, (uint32_t)(digits + kScanDigits - 1) / kScanDigits)) return;
  const int d = blockIdx.x * kScanDigits + threadIdx.x % kScanDigits, q = threadIdx.x / kScanDigits;
  const uint32_t per = (s.blocks + kParts - 1) / kParts, b0 = q * per, b1 = b0 + per < s.blocks ? b0 + per : s.blocks;
  uint32_t sum = 0u;
  if (d < digits)
    for (uint32_t b = b0; b < b1; b += 4) {
      uint32_t c[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) c[u] = b + u < b1 ? s.counts[(int64_t)(b + u) * digits + d] : 0u;
#pragma unroll
      for (int u = 0; u < 4; ++u) sum += c[u];
    }
  part[q][threadIdx.x % kScanDigits] = sum;
  __syncthreads();
  uint32_t before = 0u, total = 0u;
#pragma unroll
  for (int k = 0; k < kParts; ++k) {
    const uint32_t c = part[k][threadIdx.x % kScanDigits];
    before += k < q ? c : 0u;
    total += c;
  }
  if (d >= digits) return;
  for (uint32_t b = b0; b < b1; b += 4) {
    uint32_t c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) c[u] = b + u < b1 ? s.counts[(int64_t)(b + u) * digits + d] : 0u;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (b + u < b1) s.counts[(int64_t)(b + u) * digits + d] = before;
      before += c[u];
    }
  }
  if (q == 0) s.totals[d] = total;
}

// A wave ranks 64 tokens at a time: lanes of equal digit find each other by one ballot per bit, the lowest of them advances the
// wave's counter by their number.  Waves own consecutive quarters of the tile, so the order of equal digits is kept.
template <typename I>
__global__ void __launch_bounds__(kThreads)
sort_scatter_kernel(SortPass s, const I* __restrict__ idx) {
  constexpr int kWaves = kThreads / NR_WAVE, kPer = (1 << kMaxDigitBits) / kThreads;  // digits per thread at most
  __shared__ uint32_t cnt[kWaves][1 << kMaxDigitBits];
  __shared__ uint32_t s_wave[kWaves];
  if (clears(s, s.blocks)) return;
  const int digits = 1 << s.bits, lane = nr_lane(), wave = threadIdx.x / NR_WAVE;
  const int64_t base = (int64_t)blockIdx.x * kTile + (int64_t)wave * (NR_WAVE * kRounds);
  uint32_t key[kRounds], pos[kRounds], rank[kRounds], total[kPer], before[kPer];
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    const int64_t i = base + u * NR_WAVE + lane;
    const bool in = i < s.n;
    key[u] = in ? key_of(s, idx, i) : 0u;
    pos[u] = in ? (s.pos != nullptr ? s.pos[i] : (uint32_t)i) : 0u;
  }
  // (thread t: digits t * per ... + per of the tables of counts)
  const int per = digits > kThreads ? digits / kThreads : 1;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int d = threadIdx.x * per + k;
    const bool in = k < per && d < digits;
    total[k] = in ? s.totals[d] : 0u;
    before[k] = in ? s.counts[(int64_t)blockIdx.x * digits + d] : 0u;
  }
  for (int d = lane; d < digits; d += NR_WAVE) cnt[wave][d] = 0u;  // (a wave counts in its own row only: no barrier)
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    const bool in = base + u * NR_WAVE + lane < s.n;
    const uint32_t d = (key[u] >> s.shift) & (uint32_t)(digits - 1);
    uint64_t peers = __ballot(in);
    for (int b = 0; b < s.bits; ++b) {
      const uint64_t ones = __ballot((d >> b) & 1u);
      peers &= ((d >> b) & 1u) ? ones : ~ones;
    }
    const int leader = in ? __ffsll((unsigned long long)peers) - 1 : lane;
    uint32_t old = 0u;
    if (in && lane == leader) old = atomicAdd(&cnt[wave][d], (uint32_t)__popcll(peers));
    old = __shfl(old, leader, NR_WAVE);
    rank[u] = old + (uint32_t)__popcll(peers & ((1ull << lane) - 1ull));
  }
  // first place of each digit: exclusive prefix of the totals over the threads, then over a thread's own digits
  uint32_t sum = 0u;
#pragma unroll
  for (int k = 0; k < kPer; ++k) sum += total[k];
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < NR_WAVE; o <<= 1) {
    const uint32_t t = __shfl_up(incl, o, NR_WAVE);
    if (lane >= o) incl += t;
  }
  if (lane == NR_WAVE - 1) s_wave[wave] = incl;
  __syncthreads();
  uint32_t first = incl - sum;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) first += w < wave ? s_wave[w] : 0u;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int d = threadIdx.x * per + k;
    if (k < per && d < digits) {
      uint32_t at = first + before[k];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t own = cnt[w][d];
        cnt[w][d] = at;
        at += own;
      }
    }
    first += total[k];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kRounds; ++u) {
    if (base + u * NR_WAVE + lane >= s.n) continue;
    const uint32_t to = cnt[wave][(key[u] >> s.shift) & (uint32_t)(digits - 1)] + rank[u];
    s.keys_out[to] = key[u];
    s.pos_out[to] = pos[u];
  }
}

// ----------------------------------------------------------------------------------------------------------------- sum
struct SumArgs {
  const uint32_t* keys;  // sorted
  const uint32_t* pos;
  int64_t n, rows;
  int dim;
  int64_t grad_stride;
  float scale;
  void* out;
  int out_dtype, accumulate;
  float* head;      // [blocks][dim]: the part of a sum that started in an earlier block
  float* tail;      // [blocks][dim]: the part of a sum that goes on in the next one
  uint32_t* flags;  // [blocks]: kHead | kSpan | kTail
  int group, groups, per_group;  // lanes per row, rows at a time, sorted positions per group
};
constexpr uint32_t kHead = 1u, kSpan = 2u, kTail = 4u;

// A sum is held in 64 bits while it is in registers, and between the groups of a block where 4 columns make a vector (fp32 rows).  14 000
// addends a row: off by 3.5e-8 of the largest (the result's own rounding alone: 2.5e-8), 1.4e-7 with all of it in fp32, which takes 1.1 us
// less of the kernel's 33 (113 840 tokens on 1 999 rows: 2.8e-8 and 8.7e-8, 1.2 of 19).  It is rounded to fp32 where it goes to the
// workspace, and between the groups where 8 columns make a vector, whose 64 bits would not fit beside a full list of tokens (16-bit
// rows; 2^-24 of a sum of 16-bit values).
template <int N>
using Part = std::conditional_t<N == 4, double, float>;

template <int N>
__device__ __forceinline__ void part_get(const Part<N>* p, double (&x)[N]) {
  typedef Part<N> vec __attribute__((ext_vector_type(16 / sizeof(Part<N>))));
  constexpr int M = 16 / (int)sizeof(Part<N>);
#pragma unroll
  for (int q = 0; q < N / M; ++q) {
    const vec v = reinterpret_cast<const vec*>(p)[q];
#pragma unroll
    for (int k = 0; k < M; ++k) x[q * M + k] = (double)v[k];
  }
}
template <int N>
__device__ __forceinline__ void part_put(Part<N>* p, const double (&x)[N]) {
  typedef Part<N> vec __attribute__((ext_vector_type(16 / sizeof(Part<N>))));
  constexpr int M = 16 / (int)sizeof(Part<N>);
#pragma unroll
  for (int q = 0; q < N / M; ++q) {
    vec v;
#pragma unroll
    for (int k = 0; k < M; ++k) v[k] = (Part<N>)x[q * M + k];
    reinterpret_cast<vec*>(p)[q] = v;
  }
}

// The first `m` columns of a sum to the workspace.
template <int N>
__device__ __forceinline__ void leave(float* p, int m, const double (&x)[N]) {
  float y[N];
#pragma unroll
  for (int k = 0; k < N; ++k) y[k] = (float)x[k];
  nr_store_some<float, N>(p, m, y);
}

// o (+)= y, the first `m` columns
template <int N, typename O>
__device__ __forceinline__ void write_as(O* o, int m, bool accumulate, float (&y)[N]) {
  if (accumulate) {
    float was[N];
    nr_load_some<O, N>(o, m, was);
#pragma unroll
    for (int k = 0; k < N; ++k) y[k] += was[k];
  }
  nr_store_some<O, N>(o, m, y);
}
template <int N>
__device__ __forceinline__ void write_row(const SumArgs& a, uint32_t row, int col, const double (&x)[N]) {
  const int64_t at = (int64_t)row * a.dim + col;
  const int m = a.dim - col;
  float y[N];
#pragma unroll
  for (int k = 0; k < N; ++k) y[k] = (float)(x[k] * (double)a.scale);
  if (a.out_dtype == NR_DTYPE_F32) write_as<N, float>(static_cast<float*>(a.out) + at, m, a.accumulate != 0, y);
  else if (a.out_dtype == NR_DTYPE_BF16) write_as<N, __bf16>(static_cast<__bf16*>(a.out) + at, m, a.accumulate != 0, y);
  else write_as<N, _Float16>(static_cast<_Float16*>(a.out) + at, m, a.accumulate != 0, y);
}

constexpr int kMaxStretch = 4096;  // sorted positions of one block (32 KB of LDS)
constexpr int kFlight = 8;         // rows of g requested before the first of them is added

// One group's stretch [q0, q1) of sorted tokens, on its columns: sums that start and end inside are written; a first sum that
// started before the stretch is left in `head`, a last one that goes on behind it in `tail`.  key_at(q): the key of token q, also
// of the one before the stretch and the one behind it; pos_at(q): its row of g.  Returns kHead | kSpan | kTail.  (Keys and
// positions of a batch are read before anything is written: the compiler cannot know that a result is not one of them.)  A
// row's last vector is read whole too, from as many columns earlier as it lacks, and its sum is moved into place at its end
// (131 072 x 513 bf16: 141 -> 119 us against pieces, whose branches keep the rows of a flight from being requested together).
template <typename T, int N, typename Key, typename Pos>
__device__ __forceinline__ uint32_t walk_stretch(const SumArgs& a, const T* __restrict__ grad, int q0, int q1, int col, uint32_t row0, Key key_at,
                                                 Pos pos_at, Part<N>* head, Part<N>* tail) {
  uint32_t flag = 0u;
  const int back = a.dim >= N ? max(col + N - a.dim, 0) : 0;
  const T* from = grad + (col - back);
  double acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.0;
  uint32_t key[kFlight + 1];
  key[kFlight] = key_at(q0);
  bool open_here = key_at(q0 - 1) != key[kFlight];
  for (int q = q0; q < q1; q += kFlight) {
    float x[kFlight][N];
    uint32_t pos[kFlight];
    key[0] = key[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const bool in = q + u < q1;
      pos[u] = in ? pos_at(q + u) : 0u;
      key[u + 1] = in ? key_at(q + u + 1) : 0u;
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (q + u >= q1) continue;
      const T* row = from + (int64_t)pos[u] * a.grad_stride;
      if (a.dim >= N) nr_load_pack<T, N>(row, x[u]);
      else nr_load_some<T, N>(row, a.dim, x[u]);
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (q + u >= q1) break;
      const bool goes_on = key[u] == key[u + 1];
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += (double)x[u][k];
      if (goes_on && q + u + 1 < q1) continue;
#pragma unroll
      for (int step = 1; step < N; step *= 2) {
        if ((back & step) == 0) continue;
#pragma unroll
        for (int k = 0; k + step < N; ++k) acc[k] = acc[k + step];
      }
      Part<N>* part = nullptr;
      if (!open_here) {
        part = head;
        flag |= goes_on ? kHead | kSpan : kHead;
      } else if (goes_on) {
        part = tail;
        flag |= kTail;
      }
      if (part != nullptr) {
        part_put<N>(part, acc);
      } else {
        write_row<N>(a, row0 + key[u], col, acc);
      }
      open_here = true;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.0;
    }
  }
  return flag;
}

// Which groups hand a sum on whole, one bit each (call with all threads, between barriers of the caller's).
__device__ __forceinline__ void mark_spans(const unsigned char* flags, int groups, uint64_t* span) {
  const int g = threadIdx.x;
  const uint64_t bits = __ballot(g < groups && (flags[g < groups ? g : 0] & kSpan) != 0u);
  if (nr_lane() == 0) span[g / NR_WAVE] = bits;
}

// The first group from g on that does not hand its sum on (groups: there is none).
__device__ __forceinline__ int first_stop(const uint64_t* span, int g, int groups) {
  for (int w = g / NR_WAVE; w * NR_WAVE < groups; ++w) {
    const uint64_t stops = ~span[w] & (w == g / NR_WAVE ? ~0ull << (g % NR_WAVE) : ~0ull);
    if (stops != 0ull) {
      const int at = w * NR_WAVE + __ffsll((unsigned long long)stops) - 1;
      return at < groups ? at : groups;
    }
  }
  return groups;
}

// Head r <- head r + r + 1 + ... up to the first that does not hand its sum on: by doubling, every group at once, so that a row
// whose tokens fill the block costs log2(groups) steps and not `groups` of them (256 groups of one lane: 54 -> 25 us).  All
// threads call it, behind a barrier; `used`: groups with tokens; `head`: this thread's columns of group 0.  A group's own sum stays
// in registers and its columns move as 16-byte vectors (3 822 tokens on one row of 8 fp16 values: 11.6 us of the kernel -> 3.9).
template <int N>
__device__ __forceinline__ void chain_heads(const uint64_t* span, int r, bool work, int groups, int used, Part<N>* head, int step) {
  uint64_t any = 0ull;
  for (int w = 0; w * NR_WAVE < groups; ++w) any |= span[w];
  if (any == 0ull) return;
  const int run = work ? first_stop(span, r, groups) - r : 0;  // groups from r on that hand on
  Part<N>* at = head + r * step;
  double own[N] = {}, x[N];
  if (run > 0) part_get<N>(at, own);
  for (int d = 1; d < used; d *= 2) {
    const bool add = run >= d && r + d < groups;
    if (add) part_get<N>(at + d * step, x);
    __syncthreads();
    if (add) {
#pragma unroll
      for (int k = 0; k < N; ++k) own[k] += x[k];
      part_put<N>(at, own);
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
sum_kernel(SumArgs a, const T* __restrict__ grad) {
  constexpr int N = 16 / (int)sizeof(T);
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  const int per_block = a.groups * a.per_group, step = a.group * N;
  Part<N>* s_head = reinterpret_cast<Part<N>*>(lds);  // [groups][group * N]
  Part<N>* s_tail = s_head + a.groups * step;
  uint32_t* s_key = reinterpret_cast<uint32_t*>(s_tail + a.groups * step);  // [per_block + 2]: the keys before, in and behind the stretch
  uint32_t* s_pos = s_key + per_block + 2;          // [per_block]
  unsigned char* s_flag = reinterpret_cast<unsigned char*>(s_pos + per_block);  // [groups]
  unsigned char* s_left = s_flag + a.groups;        // [groups]: what a group leaves for the blocks around this one
  __shared__ int s_valid;
  __shared__ uint64_t s_span[kThreads / NR_WAVE];
  const int64_t p0 = (int64_t)blockIdx.x * per_block;
  constexpr uint32_t kNone = 0xFFFFFFFFu;
  const uint32_t ignored = (uint32_t)a.rows;
  if (threadIdx.x == 0) s_valid = 0;
  __syncthreads();
  int valid = 0;
  for (int i = threadIdx.x; i < per_block + 2; i += kThreads) {
    const int64_t p = p0 + i - 1;
    const uint32_t key = (p >= 0 && p < a.n) ? a.keys[p] : kNone;
    s_key[i] = key;
    if (i >= 1 && i <= per_block) {
      s_pos[i - 1] = p < a.n ? a.pos[p] : 0u;
      if (key < ignored) valid = i;
    }
  }
  if (valid > 0) atomicMax(&s_valid, valid);  // (keys ascend: what gets no gradient is behind everything else)
  __syncthreads();
  const int count = s_valid;
  const int r = threadIdx.x / a.group, lane = threadIdx.x - r * a.group;
  const int col = (blockIdx.y * a.group + lane) * N;
  const bool work = r < a.groups && col < a.dim;
  Part<N>* head = s_head + r * step + lane * N;
  Part<N>* tail = s_tail + r * step + lane * N;
  if (work) {
    const int q0 = r * a.per_group, q1 = q0 + a.per_group < count ? q0 + a.per_group : count;
    uint32_t flag = 0u;
    if (q0 < q1)
      flag = walk_stretch<T, N>(a, grad, q0, q1, col, 0u, [&](int q) { return s_key[q + 1]; }, [&](int q) { return s_pos[q]; }, head, tail);
    if (lane == 0) s_flag[r] = (unsigned char)flag;
  }
  __syncthreads();
  mark_spans(s_flag, a.groups, s_span);
  __syncthreads();
  chain_heads<N>(s_span, r, work, a.groups, (count + a.per_group - 1) / a.per_group, s_head + lane * N, step);
  // sums that cross stretches: their first group adds the parts behind it.  Group 0 also takes a sum that came in from the
  // block before.
  if (work) {
    const uint32_t own = s_flag[r];
    double acc[N];
    uint32_t flag = 0u;
    const int64_t slot = (int64_t)blockIdx.x * a.dim + col;
    if (r == 0 && (own & kHead)) {
      part_get<N>(head, acc);
      flag |= first_stop(s_span, 0, a.groups) < a.groups ? kHead : kHead | kSpan;
      leave<N>(a.head + slot, a.dim - col, acc);
    }
    if (own & kTail) {
      const bool more = r + 1 < a.groups;
      double next[N] = {};
      part_get<N>(tail, acc);
      if (more) part_get<N>(head + step, next);
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += next[k];
      if (more && first_stop(s_span, r + 1, a.groups) < a.groups) {
        write_row<N>(a, s_key[(r + 1) * a.per_group], col, acc);
      } else {
        leave<N>(a.tail + slot, a.dim - col, acc);
        flag |= kTail;
      }
    }
    if (blockIdx.y == 0 && lane == 0) s_left[r] = (unsigned char)flag;
  }
  __syncthreads();
  if (blockIdx.y == 0 && threadIdx.x == 0) {
    uint32_t flag = 0u;
    for (int j = 0; j < a.groups; ++j) flag |= s_left[j];
    a.flags[blockIdx.x] = flag;
  }
}

// ------------------------------------------------------------------------------------------- few indices, or a small table
// No sort of the whole.  A block OWNS a range of rows (and of columns): it reads the indices, keeps those of its range in
// ascending position (one ballot per 64), orders that short list by row, and sums it as above; the rows of its range that
// nothing looks up it clears itself.  The indices are read by every block (128 KB from L2 at 16 384 of 8 bytes), and its list has
// to fit into LDS, which limits the method to kOwnMax of them: one launch, no workspace.  More indices are taken in chunks, each
// into a table of its own, in fp32; a second launch adds those in order -- where they are small (kOwnTables): two launches
// instead of five or eight.
// A list is as long as the range's share of the tokens: 64 on average, all of them at worst, and then a block per column range
// does a chunk's work.  So columns are split down to 64 bytes, and the chunks down to 2 048, where there are fewer rows than
// blocks to fill the chip with.
constexpr int kOwnThreads = 1024;
constexpr int kOwnRounds = 16;
constexpr int kOwnMax = kOwnThreads * kOwnRounds;  // 14 bits of position, 18 of row in a list entry
constexpr int kOwnPosBits = 14;
constexpr int kOwnRangeMax = 1 << (32 - kOwnPosBits - 1);
constexpr int kOwnBlocks = 256;
constexpr int kOwnChunkMin = 2048;
constexpr int kOwnLanes = 32;    // half a kilobyte of a row per block at most (a kilobyte: 40 % slower where one row has a fifth of
                                 // the tokens, 64 bytes: 30 % slower where all have the same share; 4 096 rows of 1 024 in bf16)
constexpr int64_t kOwnLateBytes = 65536;  // of zeros per block, from which on half of them wait for the sums' loads (3 us of stores)
constexpr int kOwnSplit = 65536; // bytes of gradient that a block sums at most, on average, before a chunk is cut
constexpr int64_t kOwnTables = (int64_t)64 << 20;  // bytes of the chunks' tables.  26 MB: 27 us against 41 sorted (40 000 tokens
                                                   // on 30 000 rows of 64 in fp32), 78 MB: 57 against 75, 156 MB: 78 against 76; in
                                                   // bf16 the sort's own traffic is half of that, 128 MB: 58 against 44
constexpr int kCountSort = 256;  // lists up to this length: every entry counts the smaller ones
constexpr int kOwnDigitBits = 9;  // (32 KB of counters)
constexpr int kOwnPartBytes = 2 * kOwnThreads * 32;  // a lane's columns in two sums: 4 in 64 bits or 8 in 32
static_assert(sizeof(Part<4>) * 4 == 32 && sizeof(Part<8>) * 8 == 32, "a lane's part of a sum");

struct OwnArgs {
  SumArgs sum;
  int64_t padding;
  int range, key_bits;  // rows per block; bits of a row inside its range
  int named_words;      // (range + 31) / 32 where a range takes long to clear, else 0
  int chunk, rounds;    // tokens per blockIdx.z, a multiple of 64; rounds of kOwnThreads that they take
};

// Zeros in rows first, first + groups, ... below `end` of the range, in this thread's columns; without those marked in `named`.
template <int N>
__device__ __forceinline__ void clear_rows(const SumArgs& a, const uint32_t* named, int first, int end, int64_t row0, int col) {
  const float zero[N] = {};
#pragma unroll 4
  for (int q = first; q < end; q += a.groups) {
    if (named != nullptr && ((named[q / 32] >> (q % 32)) & 1u)) continue;
    const int64_t at = (row0 + q) * a.dim + col;
    if (a.out_dtype == NR_DTYPE_F32) nr_store_some<float, N>(static_cast<float*>(a.out) + at, a.dim - col, zero);
    else nr_store_some<__bf16, N>(static_cast<__bf16*>(a.out) + at, a.dim - col, zero);  // (zero is zero in both 16-bit types)
  }
}

template <typename T, typename I>
__global__ void __launch_bounds__(kOwnThreads)
own_kernel(OwnArgs o, const T* __restrict__ grad, const I* __restrict__ idx) {
  constexpr int N = 16 / (int)sizeof(T), kWaves = kOwnThreads / NR_WAVE;
  SumArgs a = o.sum;
  const int64_t base = (int64_t)blockIdx.z * o.chunk;
  const int n = a.n - base < o.chunk ? (int)(a.n - base) : o.chunk;
  grad += base * a.grad_stride;
  idx += base;
  if (gridDim.z > 1) a.out = static_cast<float*>(a.out) + (int64_t)blockIdx.z * a.rows * a.dim;  // (partial tables, in fp32)
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  const int step = a.group * N, lane = nr_lane(), wave = threadIdx.x / NR_WAVE;
  Part<N>* s_head = reinterpret_cast<Part<N>*>(lds);         // [groups][group * N]
  Part<N>* s_tail = s_head + a.groups * step;
  uint32_t* s_digit = lds;                                   // [waves][512]: before the sums
  uint32_t* s_list = lds + kOwnPartBytes / 4;                // [chunk]
  uint32_t* s_named = s_list + o.chunk;                      // [named_words]: rows that have tokens, where they are cleared late
  unsigned char* s_flag = reinterpret_cast<unsigned char*>(s_named + o.named_words);  // [groups]
  __shared__ uint32_t s_count[kWaves];
  __shared__ uint64_t s_span[kWaves];
  const int64_t row0 = (int64_t)blockIdx.x * o.range;
  const int range = row0 + o.range < a.rows ? o.range : (int)(a.rows - row0);
  const int r = threadIdx.x / a.group, glane = threadIdx.x - r * a.group;
  const int col = (blockIdx.y * a.group + glane) * N;
  const bool work = r < a.groups && col < a.dim;

  uint32_t item[kOwnRounds];
  constexpr uint32_t kNone = 0xFFFFFFFFu;
  const uint32_t padding = o.padding >= row0 && o.padding < row0 + range ? (uint32_t)(o.padding - row0) : kNone;
  const int first = wave * (NR_WAVE * o.rounds) + lane;
  I raw[kOwnRounds];  // (all loads before the first test: past the end the last index again)
#pragma unroll
  for (int u = 0; u < kOwnRounds; ++u)
    if (u < o.rounds) raw[u] = idx[first + u * NR_WAVE < n ? first + u * NR_WAVE : n - 1];
#pragma unroll
  for (int u = 0; u < kOwnRounds; ++u) {
    item[u] = kNone;
    const int i = first + u * NR_WAVE;
    if (u < o.rounds) {
      const uint64_t d = (uint64_t)(int64_t)raw[u] - (uint64_t)row0;  // (below the range: far above it; the lowest index of all, too)
      if (i < n && d < (uint64_t)range && (uint32_t)d != padding) item[u] = ((uint32_t)d << kOwnPosBits) | (uint32_t)i;
    }
  }
  // Zeros: the rows of the range, or of its first half, are all cleared here, beside the loads of the indices (those that are
  // looked up are written again, behind the barriers below).  Where a range is large, the other half is cleared beside the loads
  // of the sums, without the rows that have tokens: neither of the two latencies is left without stores (8 192 tokens on 2^22 rows of 8: 31 -> 27 us).
  const int early = o.named_words > 0 ? range / 2 : range;
  if (!a.accumulate) {
    if (gridDim.y == 1) {
      const int words = a.out_dtype == NR_DTYPE_F32 ? 2 : 1;
      clear_halves(static_cast<uint16_t*>(a.out) + row0 * a.dim * words, (int64_t)early * a.dim * words, threadIdx.x, kOwnThreads);
    } else if (work) {
      clear_rows<N>(a, nullptr, r, early, row0, col);
    }
    for (int w = threadIdx.x; w < o.named_words; w += kOwnThreads) s_named[w] = 0u;
  }
  uint32_t mine = 0u;
#pragma unroll
  for (int u = 0; u < kOwnRounds; ++u) mine += (uint32_t)__popcll(__ballot(item[u] != kNone));
  if (lane == 0) s_count[wave] = mine;
  __syncthreads();
  uint32_t at = 0u, total = 0u;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    at += w < wave ? s_count[w] : 0u;
    total += s_count[w];
  }
  const int m = (int)total;
  if (m == 0 && (a.accumulate || o.named_words == 0)) return;
#pragma unroll
  for (int u = 0; u < kOwnRounds; ++u) {
    if (u >= o.rounds) break;
    const uint64_t hit = __ballot(item[u] != kNone);
    if (hit == 0ull) continue;
    if (item[u] != kNone) s_list[at + (uint32_t)__popcll(hit & ((1ull << lane) - 1ull))] = item[u];
    at += (uint32_t)__popcll(hit);
  }
  __syncthreads();
  if (range > 1 && m <= kCountSort) {
    // the entries are all different and ordered like (row, position): an entry's place is the number of smaller ones
    uint32_t own = 0u;
    int place = 0;
    if ((int)threadIdx.x < m) {
      own = s_list[threadIdx.x];
      for (int j = 0; j < m; ++j) place += s_list[j] < own ? 1 : 0;
    }
    __syncthreads();
    if ((int)threadIdx.x < m) s_list[place] = own;
    __syncthreads();
  } else if (range > 1) {
    // by 9 bits of the row at a time, as in sort_scatter_kernel: the list through registers and back
    const int rounds = (m + kOwnThreads - 1) / kOwnThreads;
    for (int shift = 0; shift < o.key_bits; shift += kOwnDigitBits) {
      constexpr int kDigits = 1 << kOwnDigitBits;
      for (int d = threadIdx.x; d < kWaves * kDigits; d += kOwnThreads) s_digit[d] = 0u;
      uint32_t rank[kOwnRounds];
#pragma unroll
      for (int u = 0; u < kOwnRounds; ++u) {
        const int i = wave * (NR_WAVE * rounds) + u * NR_WAVE + lane;
        item[u] = u < rounds && i < m ? s_list[i] : kNone;
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kOwnRounds; ++u) {
        const bool in = item[u] != kNone;
        const uint32_t d = (item[u] >> (kOwnPosBits + shift)) & (kDigits - 1);
        uint64_t peers = __ballot(in);
        rank[u] = 0u;
        if (peers == 0ull) continue;
#pragma unroll
        for (int b = 0; b < kOwnDigitBits; ++b) {
          const uint64_t ones = __ballot((d >> b) & 1u);
          peers &= ((d >> b) & 1u) ? ones : ~ones;
        }
        const int leader = in ? __ffsll((unsigned long long)peers) - 1 : lane;
        uint32_t old = 0u;
        if (in && lane == leader) old = atomicAdd(&s_digit[wave * kDigits + d], (uint32_t)__popcll(peers));
        old = __shfl(old, leader, NR_WAVE);
        rank[u] = old + (uint32_t)__popcll(peers & ((1ull << lane) - 1ull));
      }
      __syncthreads();
      // exclusive prefix over (digit, wave): a thread per digit adds its waves, the first wave scans the sums
      __shared__ uint32_t s_first[kDigits];
      if (threadIdx.x < kDigits) {
        uint32_t sum = 0u;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const uint32_t c = s_digit[w * kDigits + threadIdx.x];
          s_digit[w * kDigits + threadIdx.x] = sum;
          sum += c;
        }
        s_first[threadIdx.x] = sum;
      }
      __syncthreads();
      if (wave == 0) {
        constexpr int kPer = kDigits / NR_WAVE;
        uint32_t c[kPer], sum = 0u;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          c[k] = s_first[lane * kPer + k];
          sum += c[k];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int d = 1; d < NR_WAVE; d <<= 1) {
          const uint32_t t = __shfl_up(incl, d, NR_WAVE);
          if (lane >= d) incl += t;
        }
        uint32_t run = incl - sum;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          s_first[lane * kPer + k] = run;
          run += c[k];
        }
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kOwnRounds; ++u) {
        if (item[u] == kNone) continue;
        const uint32_t d = (item[u] >> (kOwnPosBits + shift)) & (kDigits - 1);
        s_list[s_first[d] + s_digit[wave * kDigits + d] + rank[u]] = item[u];
      }
      __syncthreads();
    }
  }
  if (!a.accumulate && o.named_words > 0) {
    for (int q = threadIdx.x; q < m; q += kOwnThreads) {  // (one token of each row)
      const uint32_t key = s_list[q] >> kOwnPosBits;
      if (q == 0 || s_list[q - 1] >> kOwnPosBits != key) atomicOr(&s_named[key / 32], 1u << (key % 32));
    }
    __syncthreads();
  }
  // the sums: the groups share the list evenly, a batch of loads at least
  const int share = (m + a.groups - 1) / a.groups, per = share > kFlight ? share : kFlight;
  auto key_at = [&](int q) { return q >= 0 && q < m ? s_list[q] >> kOwnPosBits : kNone; };
  Part<N>* head = s_head + r * step + glane * N;
  Part<N>* tail = s_tail + r * step + glane * N;
  const int q0 = r * per, q1 = q0 + per < m ? q0 + per : m;
  if (work) {
    uint32_t flag = 0u;
    if (q0 < q1)
      flag = walk_stretch<T, N>(a, grad, q0, q1, col, (uint32_t)row0, key_at,
                                [&](int q) { return s_list[q] & ((1u << kOwnPosBits) - 1u); }, head, tail);
    if (glane == 0) s_flag[r] = (unsigned char)flag;
    if (!a.accumulate && o.named_words > 0) clear_rows<N>(a, s_named, early + r, range, row0, col);
  }
  __syncthreads();
  mark_spans(s_flag, a.groups, s_span);
  __syncthreads();
  chain_heads<N>(s_span, r, work, a.groups, (m + per - 1) / per, s_head + glane * N, step);
  if (work && (s_flag[r] & kTail)) {  // (the last token's sum ends with the list: a group follows)
    double acc[N], next[N];
    part_get<N>(tail, acc);
    part_get<N>(head + step, next);
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] += next[k];
    write_row<N>(a, (uint32_t)row0 + key_at(q1 - 1), col, acc);
  }
}

// out (+)= round(scale * (tables[0] + tables[1] + ...)), 4 elements per thread
template <typename O>
__global__ void __launch_bounds__(kThreads)
merge_kernel(const float* __restrict__ tables, int chunks, int64_t elements, float scale, int accumulate, O* __restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4;
  if (i >= elements) return;
  const int m = elements - i < 4 ? (int)(elements - i) : 4;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  for (int c = 0; c < chunks; c += kFlight) {
    float x[kFlight][4];
#pragma unroll
    for (int u = 0; u < kFlight; ++u)
      if (c + u < chunks) nr_load_some<float, 4>(tables + (c + u) * elements + i, m, x[u]);
#pragma unroll
    for (int u = 0; u < kFlight; ++u)
      if (c + u < chunks)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] += (double)x[u][k];
  }
  float y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] = (float)(acc[k] * (double)scale);
  write_as<4, O>(out + i, m, accumulate != 0, y);
}

// A sum that starts in block b and leaves it: tail[b] + head[b + 1] + ... + the head that ends it.  A row that thousands of
// tokens share crosses hundreds of blocks: groups of threads add consecutive shares of them, then the shares are added in order.
constexpr int kJoinThreads = 512;
constexpr int kJoinGroups = 64;
__global__ void __launch_bounds__(kJoinThreads)
join_kernel(SumArgs a, uint32_t blocks) {
  const uint32_t b = blockIdx.x;
  const uint32_t near = b + 1 + threadIdx.x < blocks ? a.flags[b + 1 + threadIdx.x] : kSpan;
  const int64_t per_block = (int64_t)a.groups * a.per_group;
  const uint32_t key = a.keys[(b + 1) * per_block < a.n ? (b + 1) * per_block - 1 : a.n - 1];
  if ((a.flags[b] & kTail) == 0u) return;
  __shared__ uint32_t s_end;
  __shared__ double s_part[kJoinThreads * 4];
  if (threadIdx.x == 0) s_end = blocks;
  __syncthreads();
  for (uint32_t j0 = b + 1; j0 < blocks; j0 += kJoinThreads) {  // the first block from b + 1 on that ends the sum
    const uint32_t j = j0 + threadIdx.x;
    if (j < blocks && ((j0 == b + 1 ? near : a.flags[j]) & kSpan) == 0u) atomicMin(&s_end, j);
    __syncthreads();
    const uint32_t end = s_end;
    __syncthreads();
    if (end < blocks) break;
  }
  const int heads = (int)((s_end < blocks ? s_end : blocks - 1) - b);  // blocks b + 1 .. s_end (every sum ends: the last token's with it)
  const int nv = (a.dim + 3) / 4, lanes = nv < kJoinThreads ? nv : kJoinThreads;
  int groups = kJoinThreads / lanes < kJoinGroups ? kJoinThreads / lanes : kJoinGroups;
  if (groups > (heads + kFlight - 1) / kFlight) groups = (heads + kFlight - 1) / kFlight;
  const int per = (heads + groups - 1) / groups;
  const int r = threadIdx.x / lanes, lane = threadIdx.x - r * lanes;
  for (int col0 = 0; col0 < a.dim; col0 += lanes * 4) {
    const int col = col0 + lane * 4;
    const bool work = r < groups && col < a.dim;
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    if (work) {
      if (r == 0) {
        float tail[4];
        nr_load_some<float, 4>(a.tail + (int64_t)b * a.dim + col, a.dim - col, tail);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = (double)tail[k];
      }
      const int h1 = (r + 1) * per < heads ? (r + 1) * per : heads;
      for (int h = r * per; h < h1; h += kFlight) {
        float x[kFlight][4];
#pragma unroll
        for (int u = 0; u < kFlight; ++u)
          if (h + u < h1) nr_load_some<float, 4>(a.head + (int64_t)(b + 1 + h + u) * a.dim + col, a.dim - col, x[u]);
#pragma unroll
        for (int u = 0; u < kFlight; ++u)
          if (h + u < h1)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] += (double)x[u][k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) s_part[(r * lanes + lane) * 4 + k] = acc[k];
    }
    __syncthreads();
    if (work && r == 0) {
      for (int g = 1; g < groups; ++g)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] += s_part[(g * lanes + lane) * 4 + k];
      write_row<4>(a, key, col, acc);
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads)
clear_kernel(uint16_t* __restrict__ p, int64_t halves) {
  clear_halves(p, halves, (int64_t)blockIdx.x * kThreads + threadIdx.x, (int64_t)gridDim.x * kThreads);
}

// ---------------------------------------------------------------------------------------------------------------- host
int dtype_size(int dtype) { return dtype == NR_DTYPE_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == NR_DTYPE_F32 || dtype == NR_DTYPE_BF16 || dtype == NR_DTYPE_F16; }
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

struct Plan {
  int bits, passes, digit_bits;
  uint32_t sort_blocks, sum_blocks;
  int group, groups, per_group, col_tiles;
  int64_t off_pairs, off_counts, off_totals, off_flags, off_parts, bytes;
};

// Everything that follows from the sizes and from the gradient's element size, which sets the columns of a lane: the digits of the
// sort, the stretches of the sum and the workspace.
Plan make_plan(int64_t rows, int dim, int64_t n, int elem_size) {
  Plan p = {};
  while ((rows >> p.bits) != 0) ++p.bits;  // keys 0 .. rows
  p.passes = (p.bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (p.bits + p.passes - 1) / p.passes;
  p.sort_blocks = (uint32_t)nr_cdiv(n, kTile);
  const int vec = 16 / elem_size, nv = (dim + vec - 1) / vec;
  p.col_tiles = (nv + kThreads - 1) / kThreads;
  p.group = (nv + p.col_tiles - 1) / p.col_tiles;
  p.groups = kThreads / p.group;
  p.per_group = 64;
  while (p.groups * p.per_group > kMaxStretch) p.per_group /= 2;
  // (three blocks to a CU: 100 000 x 512 bf16 61 us against 73 with four, 131 072 x 512 91 against 104 with two)
  while (p.per_group > kFlight && nr_cdiv(n, (int64_t)p.groups * p.per_group) * p.col_tiles < 3 * kOwnBlocks) p.per_group /= 2;
  p.sum_blocks = (uint32_t)nr_cdiv(n, (int64_t)p.groups * p.per_group);
  auto place = [&p](int64_t bytes) {
    const int64_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.off_pairs = place(4 * n * (int64_t)sizeof(uint32_t));
  p.off_counts = place(((int64_t)1 << p.digit_bits) * p.sort_blocks * (int64_t)sizeof(uint32_t));
  p.off_totals = place(((int64_t)1 << p.digit_bits) * (int64_t)sizeof(uint32_t));
  p.off_flags = place((int64_t)p.sum_blocks * (int64_t)sizeof(uint32_t));
  p.off_parts = place(2 * (int64_t)p.sum_blocks * dim * (int64_t)sizeof(float));
  return p;
}

// Owners: how many columns, rows and tokens a block takes.  chunks == 0: the tokens are sorted instead.
struct OwnPlan {
  int group, groups, col_tiles, range, ranges, key_bits, chunk, chunks;
};
OwnPlan make_own_plan(int64_t rows, int dim, int64_t n, int elem_size) {
  OwnPlan p = {};
  if (rows > (int64_t)kOwnRangeMax * kOwnBlocks) return p;  // (18 bits of a list entry for the row)
  const int vec = 16 / elem_size, nv = (dim + vec - 1) / vec;
  const int64_t least = nr_cdiv(n, kOwnMax), most = nr_cdiv(n, kOwnChunkMin);
  // at most kOwnBlocks blocks, one to a CU: more would wait for the first to end (113 840 tokens on 1 999 rows: 259 blocks 26 to 32 us,
  // 252 blocks 24 us)
  auto cut = [&](int64_t chunks, int lanes) {
    p.chunk = (int)(nr_cdiv(nr_cdiv(n, chunks), NR_WAVE) * NR_WAVE);
    p.chunks = (int)nr_cdiv(n, p.chunk);
    p.col_tiles = (nv + lanes - 1) / lanes;
    const int64_t want = kOwnBlocks / ((int64_t)p.col_tiles * p.chunks);
    int64_t range = nr_cdiv(rows, want > 0 ? want : 1);
    if (range > kOwnRangeMax) range = kOwnRangeMax;
    p.range = (int)range;
    p.ranges = (int)nr_cdiv(rows, range);
  };
  auto blocks = [&] { return (int64_t)p.ranges * p.col_tiles * p.chunks; };
  int lanes = nv < kOwnLanes ? nv : kOwnLanes;  // half a kilobyte of a row, then down to 64 bytes while there are CUs without a block
  if (least == 1) {
    while (lanes > 4 && rows * ((nv + lanes - 1) / lanes) < kOwnBlocks) lanes = (lanes + 1) / 2;
    cut(1, lanes);
    // (a second launch costs 3 us: only for blocks with much to read.  16 384 tokens on one row of 1 024: 56 -> 34 us)
    if (blocks() <= kOwnBlocks / 2 && nr_cdiv(n, p.ranges) * nr_cdiv(nv, p.col_tiles) * 16 > kOwnSplit) {
      const int64_t more = kOwnBlocks / blocks();
      cut(more < most ? more : most, lanes);
      if (p.chunks > 1 && (double)p.chunks * (double)rows * dim * sizeof(float) > (double)kOwnTables) cut(1, lanes);
    }
  } else {
    cut(least, lanes);
    const int64_t more = kOwnBlocks / ((int64_t)p.ranges * p.col_tiles);
    if (more > least) cut(more < most ? more : most, lanes);
    while (lanes > 4 && blocks() <= kOwnBlocks / 2) cut(p.chunks, lanes = (lanes + 1) / 2);
    if (p.chunks > 65535 || (double)p.chunks * (double)rows * dim * sizeof(float) > (double)kOwnTables) p.chunks = 0;
  }
  p.group = (nv + p.col_tiles - 1) / p.col_tiles;
  p.groups = kOwnThreads / p.group;
  while (((p.range - 1) >> p.key_bits) != 0) ++p.key_bits;
  return p;
}

bool sizes_ok(int64_t rows, int dim, int64_t n) {
  return rows >= 0 && rows <= 0x7FFFFFFE && dim >= 0 && dim <= kMaxDim && n >= 0 && n <= 0x7FFFFFFF;
}

template <typename T, typename I>
int launch_rows(const void* table, int64_t rows, int dim, int64_t row_stride, const void* idx, int64_t n, float scale, void* out,
                int64_t out_stride, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(T);
  const uint32_t nv = (uint32_t)((dim + N - 1) / N);
  // l / nv = umulhi(l, magic) while l * nv < 2^32: l < nv + 1 024, nv <= 16 384
  const uint32_t magic = nv == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + nv - 1) / nv);
  const bool past = n * dim * (int64_t)sizeof(T) > kStreamBytes;
  auto kernel = past ? rows_kernel<T, I, true> : rows_kernel<T, I, false>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)nr_cdiv(n * nv, kThreads * kRowUnroll)), dim3(kThreads), 0, stream, static_cast<const T*>(table),
                     rows, dim, row_stride, static_cast<const I*>(idx), n, scale, static_cast<T*>(out), out_stride, nv, magic);
  NR_LAUNCH_CHECK();
  return 0;
}

template <typename I>
int launch_sort(const Plan& p, SortPass s, const void* idx, uint32_t* const (&pairs)[4], hipStream_t stream) {
  // zeros in equal shares, of whole vectors
  uint16_t* zeros = s.zeros;
  const int64_t halves = zeros != nullptr ? s.halves : 0, share = nr_cdiv(nr_cdiv(halves, 3 * p.passes), 8) * 8;
  int64_t done = 0;
  auto launch = [&](auto kernel, uint32_t blocks, auto... args) {
    s.zeros = zeros + done;
    s.halves = halves - done < share ? halves - done : share;
    const int64_t want = nr_cdiv(s.halves, kThreads * 32);
    s.zero_blocks = (uint32_t)(want < kZeroBlocks ? want : kZeroBlocks);
    done += s.halves;
    hipLaunchKernelGGL(kernel, dim3(blocks + s.zero_blocks), dim3(kThreads), 0, stream, s, args...);
  };
  for (int pass = 0; pass < p.passes; ++pass) {
    s.shift = pass * p.digit_bits;
    s.bits = p.digit_bits;
    s.keys = pass == 0 ? nullptr : pairs[(pass - 1) % 2 * 2];
    s.pos = pass == 0 ? nullptr : pairs[(pass - 1) % 2 * 2 + 1];
    s.keys_out = pairs[pass % 2 * 2];
    s.pos_out = pairs[pass % 2 * 2 + 1];
    launch(sort_count_kernel<I>, p.sort_blocks, static_cast<const I*>(idx));
    launch(sort_scan_kernel, (uint32_t)nr_cdiv(1 << s.bits, kScanDigits));
    launch(sort_scatter_kernel<I>, p.sort_blocks, static_cast<const I*>(idx));
    NR_LAUNCH_CHECK();
  }
  return 0;
}

template <typename T>
int launch_sum(const Plan& p, const SumArgs& a, const void* grad, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(T);
  const int per_block = a.groups * a.per_group;
  const size_t lds = (size_t)(2 * per_block + 2) * 4 + (size_t)(2 * a.groups * a.group * N) * sizeof(Part<N>) + (size_t)(2 * a.groups);
  hipLaunchKernelGGL(sum_kernel<T>, dim3(p.sum_blocks, (uint32_t)p.col_tiles), dim3(kThreads), lds, stream, a, static_cast<const T*>(grad));
  NR_LAUNCH_CHECK();
  hipLaunchKernelGGL(join_kernel, dim3(p.sum_blocks), dim3(kJoinThreads), 0, stream, a, p.sum_blocks);
  NR_LAUNCH_CHECK();
  return 0;
}

constexpr size_t own_lds(int list_words, int named_words) { return kOwnPartBytes + (size_t)(list_words + named_words) * 4 + kOwnThreads; }

template <typename T, typename I>
int launch_own(const OwnPlan& p, const OwnArgs& o, const void* grad, const void* idx, hipStream_t stream) {
  hipLaunchKernelGGL((own_kernel<T, I>), dim3((uint32_t)p.ranges, (uint32_t)p.col_tiles, (uint32_t)p.chunks), dim3(kOwnThreads),
                     own_lds(o.chunk, o.named_words), stream, o, static_cast<const T*>(grad), static_cast<const I*>(idx));
  NR_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int init_own() {
  if (int rc = nr_raise_lds(own_kernel<T, int64_t>, own_lds(kOwnMax, kOwnRangeMax / 32))) return rc;
  return nr_raise_lds(own_kernel<T, int32_t>, own_lds(kOwnMax, kOwnRangeMax / 32));
}

template <typename O>
int launch_merge(const OwnPlan& p, const float* tables, int64_t elements, float scale, int accumulate, void* out, hipStream_t stream) {
  hipLaunchKernelGGL(merge_kernel<O>, dim3((uint32_t)nr_cdiv(elements, kThreads * 4)), dim3(kThreads), 0, stream, tables, p.chunks, elements,
                     scale, accumulate, static_cast<O*>(out));
  NR_LAUNCH_CHECK();
  return 0;
}

}  // namespace

int nr_init_embedding() {
  if (int rc = init_own<float>()) return rc;
  if (int rc = init_own<__bf16>()) return rc;
  return init_own<_Float16>();
}

extern "C" int nr_embedding_fwd(const void* table, int dtype, int64_t rows, int dim, int64_t row_stride, const void* idx, int idx_bytes,
                                int64_t n, float scale, void* out, int64_t out_stride, nr_stream_t stream) {
  if (!dtype_ok(dtype) || !sizes_ok(rows, dim, n) || (idx_bytes != 4 && idx_bytes != 8) || row_stride < 0 || out_stride < dim) return NR_EINVAL;
  if (n == 0 || dim == 0) return 0;
  if (idx == nullptr || out == nullptr || (table == nullptr && rows > 0)) return NR_EINVAL;
  if (!aligned(idx, idx_bytes) || !aligned(table, dtype_size(dtype)) || !aligned(out, dtype_size(dtype))) return NR_EINVAL;
  const int vec = 16 / dtype_size(dtype);
  if (nr_cdiv(n * ((dim + vec - 1) / vec), kThreads * kRowUnroll) > 0x7FFFFFFF) return NR_EINVAL;  // (blocks of one launch)
  const bool wide = idx_bytes == 8;
  auto launch = dtype == NR_DTYPE_F32    ? (wide ? launch_rows<float, int64_t> : launch_rows<float, int32_t>)
                : dtype == NR_DTYPE_BF16 ? (wide ? launch_rows<__bf16, int64_t> : launch_rows<__bf16, int32_t>)
                                         : (wide ? launch_rows<_Float16, int64_t> : launch_rows<_Float16, int32_t>);
  return launch(table, rows, dim, row_stride, idx, n, scale, out, out_stride, nr_s(stream));
}

extern "C" int64_t nr_embedding_bwd_workspace_bytes(int64_t rows, int dim, int64_t n, int grad_dtype) {
  if (!dtype_ok(grad_dtype) || !sizes_ok(rows, dim, n)) return NR_EINVAL;
  if (n == 0 || dim == 0 || rows == 0) return 0;
  const OwnPlan own = make_own_plan(rows, dim, n, dtype_size(grad_dtype));
  if (own.chunks == 1) return 0;
  if (own.chunks > 1) return own.chunks * rows * dim * (int64_t)sizeof(float);
  return make_plan(rows, dim, n, dtype_size(grad_dtype)).bytes;
}

extern "C" int nr_embedding_bwd(const void* grad, int grad_dtype, int64_t grad_stride, const void* idx, int idx_bytes, int64_t n, int64_t rows,
                                int dim, float scale, int64_t padding, void* grad_table, int table_dtype, int accumulate, void* workspace,
                                nr_stream_t stream) {
  if (!dtype_ok(grad_dtype) || !dtype_ok(table_dtype) || !sizes_ok(rows, dim, n) || (idx_bytes != 4 && idx_bytes != 8) || grad_stride < 0)
    return NR_EINVAL;
  if (rows == 0 || dim == 0) return 0;
  if (grad_table == nullptr || !aligned(grad_table, dtype_size(table_dtype))) return NR_EINVAL;
  if (n > 0 && (grad == nullptr || idx == nullptr || !aligned(grad, dtype_size(grad_dtype)) || !aligned(idx, idx_bytes))) return NR_EINVAL;
  hipStream_t st = nr_s(stream);
  SumArgs a = {};
  a.n = n;
  a.rows = rows;
  a.dim = dim;
  a.grad_stride = grad_stride;
  a.scale = scale;
  a.out = grad_table;
  a.out_dtype = table_dtype;
  a.accumulate = accumulate;
  const OwnPlan own = n > 0 ? make_own_plan(rows, dim, n, dtype_size(grad_dtype)) : OwnPlan{};
  if (n > 0 && own.chunks != 1 && (workspace == nullptr || !aligned(workspace, 256))) return NR_EINVAL;
  if (own.chunks > 0) {
    a.group = own.group;
    a.groups = own.groups;
    if (own.chunks > 1) {
      a.out = workspace;
      a.out_dtype = NR_DTYPE_F32;
      a.accumulate = 0;
      a.scale = 1.0f;
    }
    const int named = own.col_tiles == 1 && (int64_t)own.range * dim * (int64_t)sizeof(float) >= kOwnLateBytes ? (own.range + 31) / 32 : 0;
    const OwnArgs o = {a, padding, own.range, own.key_bits, named, own.chunk, (own.chunk + kOwnThreads - 1) / kOwnThreads};
    const bool wide = idx_bytes == 8;
    auto launch = grad_dtype == NR_DTYPE_F32    ? (wide ? launch_own<float, int64_t> : launch_own<float, int32_t>)
                  : grad_dtype == NR_DTYPE_BF16 ? (wide ? launch_own<__bf16, int64_t> : launch_own<__bf16, int32_t>)
                                                : (wide ? launch_own<_Float16, int64_t> : launch_own<_Float16, int32_t>);
    if (int rc = launch(own, o, grad, idx, st)) return rc;
    if (own.chunks == 1) return 0;
    auto merge = table_dtype == NR_DTYPE_F32 ? launch_merge<float> : table_dtype == NR_DTYPE_BF16 ? launch_merge<__bf16> : launch_merge<_Float16>;
    return merge(own, static_cast<const float*>(workspace), rows * dim, scale, accumulate, grad_table, st);
  }
  const int64_t halves = accumulate ? 0 : rows * dim * (dtype_size(table_dtype) / 2);  // zeros where nothing is looked up
  if (n == 0 && halves > 0) {
    const int64_t blocks = nr_cdiv(halves, kThreads * 32);
    hipLaunchKernelGGL(clear_kernel, dim3((uint32_t)(blocks < kZeroBlocks ? blocks : kZeroBlocks)), dim3(kThreads), 0, st,
                       static_cast<uint16_t*>(grad_table), halves);
    NR_LAUNCH_CHECK();
  }
  if (n == 0) return 0;
  const Plan p = make_plan(rows, dim, n, dtype_size(grad_dtype));
  char* ws = static_cast<char*>(workspace);
  uint32_t* pairs[4];
  for (int k = 0; k < 4; ++k) pairs[k] = reinterpret_cast<uint32_t*>(ws + p.off_pairs) + (int64_t)k * n;
  SortPass s = {};
  s.counts = reinterpret_cast<uint32_t*>(ws + p.off_counts);
  s.totals = reinterpret_cast<uint32_t*>(ws + p.off_totals);
  s.n = n;
  s.rows = rows;
  s.padding = padding;
  s.blocks = p.sort_blocks;
  s.zeros = static_cast<uint16_t*>(grad_table);
  s.halves = halves;
  if (int rc = idx_bytes == 8 ? launch_sort<int64_t>(p, s, idx, pairs, st) : launch_sort<int32_t>(p, s, idx, pairs, st)) return rc;
  a.keys = pairs[(p.passes - 1) % 2 * 2];
  a.pos = pairs[(p.passes - 1) % 2 * 2 + 1];
  a.flags = reinterpret_cast<uint32_t*>(ws + p.off_flags);
  a.head = reinterpret_cast<float*>(ws + p.off_parts);
  a.tail = a.head + (int64_t)p.sum_blocks * dim;
  a.group = p.group;
  a.groups = p.groups;
  a.per_group = p.per_group;
  if (grad_dtype == NR_DTYPE_F32) return launch_sum<float>(p, a, grad, st);
  if (grad_dtype == NR_DTYPE_BF16) return launch_sum<__bf16>(p, a, grad, st);
  return launch_sum<_Float16>(p, a, grad, st);
}
