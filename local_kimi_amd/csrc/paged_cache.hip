// The paged cache of full attention layers, for gfx950: norms and rotation of new
// queries and keys, their write to the pages, copies of pages.

#include <algorithm>
#include <cstdlib>

#include "lk_common.hpp"
#include "lk_paged.h"
#include "lk_pages.hpp"

namespace lk {
namespace {

// ---------------------------------------------------------------------------
// Head norms, rotation, append

constexpr int kHeadThreads = 256;
constexpr int kHeadMaxDim = 256;

struct HeadArgs {
  const void *q, *k, *v, *q_weight, *k_weight;
  const float* cos_sin;
  const void* positions;
  void *q_out, *k_out, *v_out;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int64_t k_page, k_page_row, k_page_head, v_page, v_page_row, v_page_head;
  PageTable table;
  Sequences sq;
  int64_t table_rows;
  int heads, kv_heads, d, d_v, rotary, offset;
  int slots;  // rows of a token: heads of q, k (and v)
  float eps;
  int interleaved, positions_64, weight_dtype;
};

// G neighbouring values as stored: 16 bytes, or 8 of the 16-bit types at G = 4.
template <int DT, int G>
struct Group {
  static constexpr int kWords = G * (DT == LK_DTYPE_F32 ? 4 : 2) / 4;
  uint32_t w[kWords];
};

template <int DT, int G>
__device__ inline void unpack(const Group<DT, G>& x, float (&f)[G]) {
#pragma unroll
  for (int i = 0; i < G; ++i) {
    if constexpr (DT == LK_DTYPE_F32) f[i] = __uint_as_float(x.w[i]);
    else f[i] = value_of<DT == LK_DTYPE_BF16>(i % 2 ? x.w[i / 2] >> 16 : x.w[i / 2] & 0xFFFFu);
  }
}

template <int DT, int G>
__device__ inline Group<DT, G> pack(const float (&f)[G]) {
  Group<DT, G> x;
#pragma unroll
  for (int i = 0; i < Group<DT, G>::kWords; ++i) {
    if constexpr (DT == LK_DTYPE_F32) x.w[i] = __float_as_uint(f[i]);
    else x.w[i] = pack2<DT == LK_DTYPE_BF16>(f[2 * i], f[2 * i + 1]);
  }
  return x;
}

// `at` counts values; groups start on their own size (strides and offsets are multiples of 8
// values, bases of 16 bytes).
template <int DT, int G>
__device__ inline Group<DT, G> load_group(const void* base, int64_t at) {
  constexpr int kWords = Group<DT, G>::kWords;
  Group<DT, G> x;
  const char* const p = static_cast<const char*>(base) + at * (DT == LK_DTYPE_F32 ? 4 : 2);
  if constexpr (kWords == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    x.w[0] = v.x, x.w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      x.w[i] = v.x, x.w[i + 1] = v.y, x.w[i + 2] = v.z, x.w[i + 3] = v.w;
    }
  }
  return x;
}

// STREAM: past the caches, for outputs that are larger than them.
template <int DT, int G, bool STREAM>
__device__ inline void store_group(void* base, int64_t at, const Group<DT, G>& x) {
  constexpr int kWords = Group<DT, G>::kWords, kStep = kWords == 2 ? 2 : 4;
  typedef uint32_t words_t __attribute__((ext_vector_type(kStep)));
  char* const p = static_cast<char*>(base) + at * (DT == LK_DTYPE_F32 ? 4 : 2);
#pragma unroll
  for (int i = 0; i < kWords; i += kStep) {
    words_t v;
#pragma unroll
    for (int k = 0; k < kStep; ++k) v[k] = x.w[i + k];
    words_t* const to = reinterpret_cast<words_t*>(p + 4 * i);
    if constexpr (STREAM) __builtin_nontemporal_store(v, to);
    else *to = v;
  }
}

template <int G>
__device__ inline void load_weights(const void* base, int at, int dtype, float (&f)[G]) {
  if (dtype == LK_DTYPE_F32) unpack<LK_DTYPE_F32, G>(load_group<LK_DTYPE_F32, G>(base, at), f);
  else if (dtype == LK_DTYPE_F16) unpack<LK_DTYPE_F16, G>(load_group<LK_DTYPE_F16, G>(base, at), f);
  else unpack<LK_DTYPE_BF16, G>(load_group<LK_DTYPE_BF16, G>(base, at), f);
}

template <int LPR>
__device__ inline float lanes_sum(float v) {
  v += dpp_f32<kQuadXor1>(v);
  v += dpp_f32<kQuadXor2>(v);
  if constexpr (LPR >= 8) v += dpp_f32<kRowHalfMirror>(v);
  if constexpr (LPR >= 16) v += dpp_f32<kRowMirror>(v);
  if constexpr (LPR >= 32) v += __shfl_xor(v, 16);
  return v;
}

// A row (a head of a token) is LPR lanes', a lane has two groups of G of its values: the
// partners of a rotation, so that nothing is exchanged but the sum of squares. A
// block takes 256 / LPR x R rows of the call's tokens x (heads of q, of k, of v), each LPR
// lanes R that follow one another, mostly of one token: its angles are read once.
// The block's rows are on their way while its threads find the places of its tokens.
template <int DT, int G, int LPR, int R, bool PAGED>
__global__ void __launch_bounds__(kHeadThreads) head_rope_kernel(HeadArgs a) {
  constexpr int kRows = kHeadThreads / LPR * R, kTokens = kRows / 2 + 2;
  __shared__ int64_t k_place[PAGED ? kTokens : 1], v_place[PAGED ? kTokens : 1];  // -1: none
  __shared__ int position[kTokens];                                             // -1: behind
  const uint32_t slots = a.slots, first = blockIdx.x * static_cast<uint32_t>(kRows);
  const uint32_t t0 = first / slots, slot0 = first - t0 * slots;
  const int lane = threadIdx.x % LPR;
  const uint32_t row0 = slot0 + threadIdx.x / LPR * R;  // from the block's first token's
  const uint32_t tokens = static_cast<uint32_t>(a.sq.rows) - t0;
  const uint32_t token0 = row0 / slots;
  // where this lane's two groups start, and whether they are turned
  int ga, gb, angle;
  bool turned;
  if (a.interleaved) {
    ga = 2 * G * lane, gb = ga + G;
    turned = ga >= a.offset && ga < a.offset + a.rotary;
    angle = (ga - a.offset) / 2;
  } else {
    turned = 2 * G * lane < a.rotary;
    ga = turned ? a.offset + G * lane : 2 * G * lane - a.rotary;
    if (!turned && ga >= a.offset) ga += a.rotary;
    gb = turned ? ga + a.rotary / 2 : ga + G;
    angle = G * lane;
  }
  const bool in_head = 2 * G * lane < a.d, in_value = PAGED && 2 * G * lane < a.d_v;
  Group<DT, G> xa[R], xb[R];
  {
    uint32_t token = token0, slot = row0 - token0 * slots;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t t = t0 + token;
      const bool is_q = static_cast<int>(slot) < a.heads;
      const bool is_v = PAGED && static_cast<int>(slot) >= a.heads + a.kv_heads;
      if (token < tokens && (is_v ? in_value : in_head)) {
        const int head = static_cast<int>(slot) - (is_q ? 0 : a.heads) - (is_v ? a.kv_heads : 0);
        const void* const from = is_q ? a.q : (is_v ? a.v : a.k);
        const int64_t at = is_q ? t * a.q_row + head * a.q_head
                                : (is_v ? t * a.v_row + head * a.v_head : t * a.k_row + head * a.k_head);
        xa[r] = load_group<DT, G>(from, at + (is_v ? 2 * G * lane : ga));
        xb[r] = load_group<DT, G>(from, at + (is_v ? 2 * G * lane + G : gb));
      }
      if (++slot == slots) slot = 0, ++token;
    }
  }
  const uint32_t last = slot0 + kRows - 1 < tokens * slots ? (slot0 + kRows - 1) / slots : tokens - 1;
  if constexpr (PAGED) {
    int s = find_sequence(a.sq, t0);  // by whole waves, of the block's first token
    for (uint32_t i = threadIdx.x; i <= last; i += kHeadThreads) {
      const int64_t t = static_cast<int64_t>(t0) + i;
      while (s < a.sq.count && sequence_rows(a.sq, s).end <= t) ++s;
      const RowRange rows = sequence_rows(a.sq, s);
      int pos = -1;
      int64_t kp = -1, vp = -1;
      if (s < a.sq.count && t >= rows.begin && t < rows.end) {
        const int64_t at = positions_before(a.table, s, rows.end - rows.begin) + (t - rows.begin);
        pos = at < 0 ? 0 : static_cast<int>(at);
        if (at >= 0 && at < static_cast<int64_t>(a.table.width) * a.table.page_rows) {
          const uint32_t block = static_cast<uint32_t>(pos) / static_cast<uint32_t>(a.table.page_rows);
          const int64_t page = a.table.pages_of[s * a.table.stride + block];
          const int64_t row = pos - static_cast<int64_t>(block) * a.table.page_rows;
          if (page >= 0 && page < a.table.pages) {
            kp = page * a.k_page + row * a.k_page_row;
            vp = page * a.v_page + row * a.v_page_row;
          }
        }
      }
      position[i] = pos, k_place[i] = kp, v_place[i] = vp;
    }
  } else {
    for (uint32_t i = threadIdx.x; i <= last; i += kHeadThreads) {
      const int64_t t = static_cast<int64_t>(t0) + i;
      int64_t pos = a.rotary == 0 ? 0
                    : a.positions_64 ? static_cast<const int64_t*>(a.positions)[t]
                                     : static_cast<const int32_t*>(a.positions)[t];
      pos = pos < 0 ? 0 : (pos >= a.table_rows ? a.table_rows - 1 : pos);
      position[i] = static_cast<int>(pos);
    }
  }
  __syncthreads();
  float c[G], s[G];
#pragma unroll
  for (int i = 0; i < G; ++i) c[i] = 1.f, s[i] = 0.f;
  uint32_t token = token0, slot = row0 - token0 * slots;
  int known = -1;  // the token that c and s are of
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (token < tokens) {
      const int64_t t = t0 + token;
      const int pos = position[token];
      const bool is_q = static_cast<int>(slot) < a.heads;
      const bool is_v = PAGED && static_cast<int>(slot) >= a.heads + a.kv_heads;
      const int head = static_cast<int>(slot) - (is_q ? 0 : a.heads) - (is_v ? a.kv_heads : 0);
      if (is_v) {  // as it is
        if (PAGED && in_value && v_place[token] >= 0) {
          const int64_t to = v_place[token] + head * a.v_page_head + 2 * G * lane;
          store_group<DT, G, (R > 1)>(a.v_out, to, xa[r]);
          store_group<DT, G, (R > 1)>(a.v_out, to + G, xb[r]);
        }
      } else {
        if (turned && known != static_cast<int>(token)) {
          known = static_cast<int>(token);
          const int row = pos < 0 ? 0 : (pos < a.table_rows ? pos : static_cast<int>(a.table_rows) - 1);
          const float* const angles = a.cos_sin + static_cast<int64_t>(row) * a.rotary + angle;
          unpack<LK_DTYPE_F32, G>(load_group<LK_DTYPE_F32, G>(angles, 0), c);
          unpack<LK_DTYPE_F32, G>(load_group<LK_DTYPE_F32, G>(angles, a.rotary / 2), s);
        }
        const void* const weight = is_q ? a.q_weight : a.k_weight;
        if (weight || a.rotary) {
          float x[G], y[G];
          if (in_head) {
            unpack<DT, G>(xa[r], x);
            unpack<DT, G>(xb[r], y);
          } else {
#pragma unroll
            for (int i = 0; i < G; ++i) x[i] = y[i] = 0.f;
          }
          if (weight) {
            float sq = 0.f;
#pragma unroll
            for (int i = 0; i < G; ++i) sq = fmaf(x[i], x[i], sq);
#pragma unroll
            for (int i = 0; i < G; ++i) sq = fmaf(y[i], y[i], sq);
            const float inv = 1.0f / sqrtf(lanes_sum<LPR>(sq) / static_cast<float>(a.d) + a.eps);
            if (in_head) {
              float w[G], u[G];
              load_weights<G>(weight, ga, a.weight_dtype, w);
              load_weights<G>(weight, gb, a.weight_dtype, u);
#pragma unroll
              for (int i = 0; i < G; ++i) x[i] = x[i] * inv * w[i], y[i] = y[i] * inv * u[i];
            }
          }
          if (turned) {
            // interleaved: pair i lies at values 2 i and 2 i + 1 of the two groups
            float p[G], q[G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
              const float first_of = a.interleaved ? (2 * i < G ? x[2 * i % G] : y[2 * i % G]) : x[i];
              const float second = a.interleaved ? (2 * i < G ? x[2 * i % G + 1] : y[2 * i % G + 1]) : y[i];
              p[i] = first_of * c[i] - second * s[i];
              q[i] = second * c[i] + first_of * s[i];
            }
#pragma unroll
            for (int i = 0; i < G; ++i) {
              x[i] = a.interleaved ? (i % 2 ? q[i / 2] : p[i / 2]) : p[i];
              y[i] = a.interleaved ? (i % 2 ? q[(i + G) / 2] : p[(i + G) / 2]) : q[i];
            }
          }
          xa[r] = pack<DT, G>(x);
          xb[r] = pack<DT, G>(y);
        }
        if (in_head && (!PAGED || is_q || k_place[token] >= 0)) {
          if (PAGED && is_q && pos < 0) xa[r] = xb[r] = Group<DT, G>{};
          int64_t to = (t * (is_q ? a.heads : a.kv_heads) + head) * a.d;
          if (PAGED && !is_q) to = k_place[token] + head * a.k_page_head;
          store_group<DT, G, (R > 1)>(is_q ? a.q_out : a.k_out, to + ga, xa[r]);
          store_group<DT, G, (R > 1)>(is_q ? a.q_out : a.k_out, to + gb, xb[r]);
        }
      }
    }
    if (++slot == slots) slot = 0, ++token;
  }
}

// Large calls (kHeadFill blocks at least) take two rows a lane group, and their
// outputs go past the caches. Both by 8192 tokens x 40 heads of 128 / 4096 packed tokens x
// 96 heads of 192 and 128: 36 / 55 us (4.8 and 4.9 TB/s; a large copy moves 5.1), with
// ordinary stores 37 / 63, of those with three rows 36 / 70, four 37 / 63, eight 40 / 64; loads
// past the caches 45 / 71 (a row's two halves share its lines).
constexpr int kHeadRun = 2;
constexpr int kHeadFill = 512;

template <int DT, int G, bool PAGED>
int launch_heads(const HeadArgs& a, const char* name, hipStream_t s) {
  const int width = PAGED && a.d_v > a.d ? a.d_v : a.d, need = (width + 2 * G - 1) / (2 * G);
  const int lanes = need <= 32 / G ? 32 / G : (need <= 64 / G ? 64 / G : 128 / G);
  const int64_t rows = a.sq.rows * a.slots, one = kHeadThreads / lanes;  // of a block at R = 1
  const bool large = rows >= one * kHeadRun * kHeadFill;
  const int64_t blocks = (rows + one * (large ? kHeadRun : 1) - 1) / (one * (large ? kHeadRun : 1));
  LK_REQUIRE(grid_fits(blocks, kHeadThreads) && rows < (int64_t{1} << 32),
             "too many rows and heads for one call");
  const dim3 grid(static_cast<unsigned>(blocks));
#define LK_HEADS(L)                                                                        \
  if (lanes == L) {                                                                        \
    if (large) head_rope_kernel<DT, G, L, kHeadRun, PAGED><<<grid, kHeadThreads, 0, s>>>(a); \
    else head_rope_kernel<DT, G, L, 1, PAGED><<<grid, kHeadThreads, 0, s>>>(a);            \
  }
  LK_HEADS(32 / G)
  LK_HEADS(64 / G)
  LK_HEADS(128 / G)
#undef LK_HEADS
  return check_launch(name);
}

// Groups of eight 16-bit values (16 bytes) where the widths and the slice divide.
template <int DT, bool PAGED>
int launch_heads(const HeadArgs& a, const char* name, hipStream_t s) {
  if constexpr (DT != LK_DTYPE_F32)
    if ((a.d | a.rotary | a.offset | (PAGED ? a.d_v : 0)) % 16 == 0)
      return launch_heads<DT, 8, PAGED>(a, name, s);
  return launch_heads<DT, 4, PAGED>(a, name, s);
}

bool on_16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// What both entry points ask of heads, widths, weights and the table of angles.
int check_heads(int64_t rows, int64_t heads, int64_t kv_heads, int64_t d, int64_t rotary,
                int64_t offset, int64_t table_rows, float eps, const void* q_weight,
                const void* k_weight, bool with_q, const float* cos_sin, int weight_dtype) {
  LK_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31), "rows must be in 0 .. 2^31 - 1");
  LK_REQUIRE(heads >= 0 && kv_heads > 0 && heads <= 65535 && kv_heads <= 65535,
             "heads must be in 1 .. 65535");
  LK_REQUIRE(d > 0 && d % 8 == 0 && d <= kHeadMaxDim,
             "the head dimension must be a multiple of 8 up to %d, got %lld", kHeadMaxDim,
             (long long)d);
  LK_REQUIRE(rotary >= 0 && rotary % 8 == 0 && offset >= 0 && offset % 8 == 0 && rotary <= d &&
                 offset <= d - rotary,
             "the rotated slice must lie within the head, in multiples of 8");
  LK_REQUIRE(rotary == 0 || (cos_sin && on_16(cos_sin) && table_rows > 0 &&
                             table_rows < (int64_t{1} << 31)),
             "a rotation needs a table of angles of 1 .. 2^31 - 1 rows on a 16-byte boundary");
  LK_REQUIRE(!with_q || (q_weight == nullptr) == (k_weight == nullptr),
             "both norm weights must be given, or neither");
  LK_REQUIRE(on_16(q_weight) && on_16(k_weight), "norm weights must start on a 16-byte boundary");
  LK_REQUIRE(weight_dtype >= LK_DTYPE_F32 && weight_dtype <= LK_DTYPE_BF16,
             "unknown norm weight dtype %d", weight_dtype);
  LK_REQUIRE(eps >= 0.f, "eps must be non-negative");
  return LK_OK;
}

// Whether no two places of a cache share memory, as far as steps that go up tell: each dimension's
// step takes it past all that the smaller ones reach.
bool places_apart(int64_t d, int64_t pages, int64_t page, int64_t rows, int64_t row, int64_t heads,
                  int64_t head) {
  struct Dim {
    int64_t step, count;
  } dims[3] = {{page, pages}, {row, rows}, {head, heads}};
  std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.step < y.step; });
  int64_t reach = d;
  for (const Dim& x : dims) {
    if (x.count <= 1) continue;
    if (x.step < reach) return false;
    reach += x.step * (x.count - 1);
  }
  return true;
}

// ---------------------------------------------------------------------------
// Copies of pages

constexpr int kCopyThreads = 256;
constexpr int kCopyPairs = 192;    // of a launch whose lists travel as its arguments
constexpr int kCopyTensors = 64;   // of a launch

struct CopyArgs {
  char* tensor[kCopyTensors];
  int64_t stride[kCopyTensors];
  int32_t chunks[kCopyTensors];  // of 16 bytes a page
  const int32_t *src_of, *dst_of;  // lists in device memory, else null and here:
  int32_t src[kCopyPairs], dst[kCopyPairs];
  int32_t pairs;
};
static_assert(sizeof(CopyArgs) <= 4096, "kernel arguments");

// 16 bytes a thread. Bound by HBM (1100 pages of 128 KB in 4 tensors, 1.15 GB: 201 us, 5.7 TB/s; in
// six launches, the lists in their arguments, 217). PACKED: pages smaller than a block's threads
// follow one another in a block. IDLE: the lists pair a page with itself, which stores nothing, since
// another pair may write the page (other lists are spared the comparison, which every block waits
// for: 1100 pages 200.7 us without it, 201.8 with it; as six launches of a graph 217 and 221).
template <bool PACKED, bool IDLE>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(CopyArgs a) {
  const int z = blockIdx.z, chunks = a.chunks[z];
  uint32_t i = blockIdx.x * kCopyThreads + threadIdx.x, pair = blockIdx.y;
  if constexpr (PACKED) {
    if (chunks == 0) return;
    pair = i / static_cast<uint32_t>(chunks);
    i -= pair * chunks;
  }
  if (pair >= static_cast<uint32_t>(a.pairs) || i >= static_cast<uint32_t>(chunks)) return;
  const int64_t src = a.src_of ? a.src_of[pair] : a.src[pair];
  const int64_t dst = a.dst_of ? a.dst_of[pair] : a.dst[pair];
  if (IDLE && src == dst) return;
  reinterpret_cast<uint4*>(a.tensor[z] + dst * a.stride[z])[i] =
      reinterpret_cast<const uint4*>(a.tensor[z] + src * a.stride[z])[i];
}

// A page is written once, and is no other pair's source: what a launch reads it
// does not write. Pairs of a page with itself (`idle`: there are any) count for neither.
int check_pairs(const int32_t* src, const int32_t* dst, int64_t pairs, int64_t pages, bool* idle) {
  for (int64_t i = 0; i < pairs; ++i)
    LK_REQUIRE(src[i] >= 0 && src[i] < pages && dst[i] >= 0 && dst[i] < pages,
               "pair %lld copies page %d to %d of a cache of %lld", (long long)i, src[i], dst[i],
               (long long)pages);
  uint8_t* const written = static_cast<uint8_t*>(std::calloc(pages / 8 + 1, 1));  // a bit a page
  LK_REQUIRE(written, "no memory for the list of pages");
  int32_t twice = -1, both = -1;
  *idle = false;
  for (int64_t i = 0; i < pairs; ++i) {
    if (src[i] == dst[i]) {
      *idle = true;
      continue;
    }
    if (written[dst[i] / 8] >> dst[i] % 8 & 1) twice = dst[i];
    written[dst[i] / 8] |= static_cast<uint8_t>(1u << dst[i] % 8);
  }
  for (int64_t i = 0; i < pairs; ++i)
    if (src[i] != dst[i] && written[src[i] / 8] >> src[i] % 8 & 1) both = src[i];
  std::free(written);
  LK_REQUIRE(twice < 0, "page %d is written twice", twice);
  LK_REQUIRE(both < 0, "page %d is both read and written", both);
  return LK_OK;
}

}  // namespace
}  // namespace lk

using namespace lk;

extern "C" {

int lk_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight,
                    const float* cos_sin, const void* positions, void* q_out, void* k_out,
                    int64_t rows, int64_t heads, int64_t kv_heads, int64_t d,
                    int64_t q_row_stride, int64_t q_head_stride, int64_t k_row_stride,
                    int64_t k_head_stride, int64_t rotary, int64_t offset, int interleaved,
                    int64_t table_rows, int positions_64, float eps, int dtype, int weight_dtype,
                    void* stream) {
  if (const int st = check_heads(rows, heads, kv_heads, d, rotary, offset, table_rows, eps,
                                 q_weight, k_weight, true, cos_sin, weight_dtype))
    return st;
  LK_REQUIRE(heads > 0, "heads must be in 1 .. 65535");
  for (const int64_t stride : {q_row_stride, q_head_stride, k_row_stride, k_head_stride})
    LK_REQUIRE(stride >= 0 && stride % 8 == 0, "strides must be multiples of 8 elements, not negative");
  LK_REQUIRE(dtype >= LK_DTYPE_F32 && dtype <= LK_DTYPE_BF16, "unknown dtype %d", dtype);
  if (rows == 0) return LK_OK;
  LK_REQUIRE(q && k && q_out && k_out && (positions || rotary == 0), "null pointer argument");
  LK_REQUIRE(on_16(q) && on_16(k) && on_16(q_out) && on_16(k_out),
             "queries and keys must start on a 16-byte boundary");
  HeadArgs a{};
  a.q = q, a.k = k, a.q_weight = q_weight, a.k_weight = k_weight;
  a.cos_sin = cos_sin, a.positions = positions, a.q_out = q_out, a.k_out = k_out;
  a.q_row = q_row_stride, a.q_head = q_head_stride, a.k_row = k_row_stride, a.k_head = k_head_stride;
  a.table_rows = table_rows, a.positions_64 = positions_64 != 0;
  a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
  a.d = static_cast<int>(d), a.rotary = static_cast<int>(rotary), a.offset = static_cast<int>(offset);
  a.slots = a.heads + a.kv_heads;
  a.sq.rows = rows;
  a.eps = eps, a.interleaved = interleaved != 0, a.weight_dtype = weight_dtype;
  const hipStream_t s = as_stream(stream);
  constexpr const char* kName = "lk_qk_norm_rope";
  if (dtype == LK_DTYPE_F32) return launch_heads<LK_DTYPE_F32, false>(a, kName, s);
  if (dtype == LK_DTYPE_F16) return launch_heads<LK_DTYPE_F16, false>(a, kName, s);
  return launch_heads<LK_DTYPE_BF16, false>(a, kName, s);
}

int lk_paged_append(const void* q, const void* k, const void* v, const void* q_weight,
                    const void* k_weight, const float* cos_sin, const int32_t* page_table,
                    const int32_t* lengths, const int32_t* cu, void* q_out, void* k_pages,
                    void* v_pages, int64_t sequences, int64_t rows, int64_t heads,
                    int64_t kv_heads, int64_t d_qk, int64_t d_v, int64_t q_row_stride,
                    int64_t q_head_stride, int64_t k_row_stride, int64_t k_head_stride,
                    int64_t v_row_stride, int64_t v_head_stride, int64_t pages, int64_t page_rows,
                    int64_t table_width, int64_t table_stride, int64_t k_page, int64_t k_page_row,
                    int64_t k_page_head, int64_t v_page, int64_t v_page_row, int64_t v_page_head,
                    int64_t rotary, int64_t offset, int interleaved, int64_t table_rows, float eps,
                    int dtype, int weight_dtype, void* stream) {
  if (const int st = check_heads(rows, heads, kv_heads, d_qk, rotary, offset, table_rows, eps,
                                 heads ? q_weight : nullptr, k_weight, heads > 0, cos_sin,
                                 weight_dtype))
    return st;
  LK_REQUIRE(d_v > 0 && d_v % 8 == 0 && d_v <= kHeadMaxDim,
             "the value dimension must be a multiple of 8 up to %d, got %lld", kHeadMaxDim,
             (long long)d_v);
  LK_REQUIRE(dtype == LK_DTYPE_F16 || dtype == LK_DTYPE_BF16, "cached values must be fp16 or bf16");
  for (const int64_t stride : {q_row_stride, q_head_stride, k_row_stride, k_head_stride,
                               v_row_stride, v_head_stride})
    LK_REQUIRE(stride >= 0 && stride % 8 == 0, "strides must be multiples of 8 elements, not negative");
  if (const int st = check_pages(sequences, rows, cu != nullptr, pages, page_rows, table_width,
                                 table_stride, {k_page, k_page_row, k_page_head, v_page, v_page_row,
                                                v_page_head}))
    return st;
  LK_REQUIRE(places_apart(d_qk, pages, k_page, page_rows, k_page_row, kv_heads, k_page_head) &&
                 places_apart(d_v, pages, v_page, page_rows, v_page_row, kv_heads, v_page_head),
             "the places of a cache that is written must not overlap");
  LK_REQUIRE(k_pages != v_pages || !k_pages, "keys and values must have pages of their own");
  if (rows == 0) return LK_OK;
  LK_REQUIRE(k && v && lengths && (table_width == 0 || page_table) && (pages == 0 || (k_pages && v_pages)) &&
                 (heads == 0 || (q && q_out)),
             "null pointer argument");
  LK_REQUIRE(on_16(k) && on_16(v) && on_16(k_pages) && on_16(v_pages) &&
                 (heads == 0 || (on_16(q) && on_16(q_out))),
             "queries, keys, values and pages must start on a 16-byte boundary");
  HeadArgs a{};
  a.q = q, a.k = k, a.v = v, a.q_weight = q_weight, a.k_weight = k_weight;
  a.cos_sin = cos_sin, a.q_out = q_out, a.k_out = k_pages, a.v_out = v_pages;
  a.q_row = q_row_stride, a.q_head = q_head_stride, a.k_row = k_row_stride, a.k_head = k_head_stride;
  a.v_row = v_row_stride, a.v_head = v_head_stride;
  a.k_page = k_page, a.k_page_row = k_page_row, a.k_page_head = k_page_head;
  a.v_page = v_page, a.v_page_row = v_page_row, a.v_page_head = v_page_head;
  a.table = PageTable{page_table, lengths, table_stride, pages, static_cast<int>(table_width),
                      static_cast<int>(page_rows)};
  a.sq = Sequences{cu, rows, rows / sequences, static_cast<int>(sequences)};
  a.table_rows = table_rows;
  a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
  a.d = static_cast<int>(d_qk), a.d_v = static_cast<int>(d_v);
  a.rotary = static_cast<int>(rotary), a.offset = static_cast<int>(offset);
  a.slots = a.heads + 2 * a.kv_heads;
  a.eps = eps, a.interleaved = interleaved != 0, a.weight_dtype = weight_dtype;
  const hipStream_t s = as_stream(stream);
  constexpr const char* kName = "lk_paged_append";
  if (dtype == LK_DTYPE_F16) return launch_heads<LK_DTYPE_F16, true>(a, kName, s);
  return launch_heads<LK_DTYPE_BF16, true>(a, kName, s);
}

int lk_copy_pages(void* const* tensors, const int64_t* page_strides, const int64_t* page_bytes,
                  int64_t count, const int32_t* src, const int32_t* dst, int64_t pairs,
                  int64_t pages, const int32_t* lists, void* stream) {
  LK_REQUIRE(count >= 0 && pairs >= 0 && pages >= 0 && pages < (int64_t{1} << 31) &&
                 pairs < (int64_t{1} << 31),
             "tensors, pairs and pages must be in 0 .. 2^31 - 1");
  if (count == 0 || pairs == 0) return LK_OK;
  LK_REQUIRE(tensors && page_strides && page_bytes && src && dst, "null pointer argument");
  int64_t most = 0;
  for (int64_t i = 0; i < count; ++i) {
    LK_REQUIRE(tensors[i], "null pointer argument");
    LK_REQUIRE(on_16(tensors[i]) && page_strides[i] % 16 == 0 && page_bytes[i] % 16 == 0,
               "pages must start on 16-byte boundaries and be a multiple of 16 bytes");
    LK_REQUIRE(page_bytes[i] >= 0 && page_bytes[i] <= page_strides[i] &&
                   page_bytes[i] < (int64_t{1} << 31),
               "pages must not overlap, and be below 2^31 bytes");
    most = std::max(most, page_bytes[i]);
  }
  bool idle = false;
  if (const int st = check_pairs(src, dst, pairs, pages, &idle)) return st;
  if (most == 0) return LK_OK;
  const hipStream_t s = as_stream(stream);
  const int64_t chunks = most / 16;
  const bool packed = chunks < kCopyThreads;
  // of a launch: what its arguments hold, or a grid takes
  const int64_t step = lists ? (packed ? (int64_t{1} << 30) / chunks : 65535) : kCopyPairs;
  for (int64_t z0 = 0; z0 < count; z0 += kCopyTensors)
    for (int64_t p0 = 0; p0 < pairs; p0 += step) {
      CopyArgs a{};
      const int z = static_cast<int>(std::min<int64_t>(kCopyTensors, count - z0));
      const int64_t n = std::min<int64_t>(step, pairs - p0);
      for (int i = 0; i < z; ++i) {
        a.tensor[i] = static_cast<char*>(tensors[z0 + i]);
        a.stride[i] = page_strides[z0 + i];
        a.chunks[i] = static_cast<int32_t>(page_bytes[z0 + i] / 16);
      }
      a.pairs = static_cast<int32_t>(n);
      if (lists) {
        a.src_of = lists + p0, a.dst_of = lists + pairs + p0;
      } else {
        std::copy(src + p0, src + p0 + n, a.src);
        std::copy(dst + p0, dst + p0 + n, a.dst);
      }
      const int64_t blocks = ((packed ? n : 1) * chunks + kCopyThreads - 1) / kCopyThreads;
      const dim3 grid(static_cast<unsigned>(blocks), packed ? 1u : static_cast<unsigned>(n),
                      static_cast<unsigned>(z));
      if (packed && idle) copy_pages_kernel<true, true><<<grid, kCopyThreads, 0, s>>>(a);
      else if (packed) copy_pages_kernel<true, false><<<grid, kCopyThreads, 0, s>>>(a);
      else if (idle) copy_pages_kernel<false, true><<<grid, kCopyThreads, 0, s>>>(a);
      else copy_pages_kernel<false, false><<<grid, kCopyThreads, 0, s>>>(a);
      if (const int st = check_launch("lk_copy_pages")) return st;
    }
  return LK_OK;
}

}  // extern "C"
