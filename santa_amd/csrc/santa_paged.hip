// santa_paged.hip -- a paged KV cache that sequences share
// (santa_amd/paged.py): page copies and block table edits, RoPE of new tokens
// with their write into pages, and the exact attention over pages, in which
// a prefix that sequences have in common is read once for all of them.  No
// counterpart in the reference, whose caches are contiguous and one per sequence
// (tutorial_code/runtime_common.py:340-397).
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "santa_amd.h"
#include "santa_attn_device.h"
#include "santa_internal.h"
#include "santa_paged.h"

namespace santa {
namespace paged {

using attn::f32x16;
using attn::kLowest;
using attn::mfma32;
using attn::other_half;
using attn::pack8;
using attn::read_tr8;
using attn::u32x4;

// ------------------------------------------------------------------- pages
// Lists travel in the kernel arguments: nothing is uploaded, and a captured
// launch holds its own.
constexpr int kPoolsPerLaunch = 64;
constexpr int kPairsPerLaunch = 384;
constexpr int kEditsPerLaunch = 240;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;

struct CopyArgs {
  char* pool[kPoolsPerLaunch];
  PageCopy pair[kPairsPerLaunch];
  long long stride;
  uint32_t vecs;  // 16-byte pieces of a page
};
struct EditArgs {
  TableEdit edit[kEditsPerLaunch];
  int* table;
  long long stride;
};
struct RemapArgs {
  PageCopy pair[kPairsPerLaunch];
  int* table;
  long long entries;
  int n;
};

// Workgroup (piece of the page, pair, pool): 16 KiB in flight per workgroup, all
// pairs and up to 64 pools of a launch at once.  Bound by HBM: 5.0 TB/s read and
// written together where half of a batch's pages are closed up (898 MB in 180 us;
// a plain copy of 2 GiB reaches 4.8 TB/s).
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(CopyArgs a) {
  char* const pool = a.pool[blockIdx.z];
  const PageCopy c = a.pair[blockIdx.y];
  const u32x4* src = reinterpret_cast<const u32x4*>(pool + c.src * a.stride);
  u32x4* dst = reinterpret_cast<u32x4*>(pool + c.dst * a.stride);
  const uint32_t i0 = blockIdx.x * (kCopyThreads * kCopyUnroll) + threadIdx.x;
  u32x4 v[kCopyUnroll];
#pragma unroll
  for (int k = 0; k < kCopyUnroll; ++k)
    if (i0 + k * kCopyThreads < a.vecs) v[k] = src[i0 + k * kCopyThreads];
#pragma unroll
  for (int k = 0; k < kCopyUnroll; ++k)
    if (i0 + k * kCopyThreads < a.vecs) dst[i0 + k * kCopyThreads] = v[k];
}

// A workgroup per edit; a few us whatever it holds (64 rows of 2048 entries 3.7).
__global__ __launch_bounds__(256) void edit_table_kernel(EditArgs a) {
  const TableEdit e = a.edit[blockIdx.x];
  int* dst = a.table + e.row * a.stride + e.col;
  const int* src = a.table + (-1 - static_cast<long long>(e.value)) * a.stride + e.col;
  for (int i = threadIdx.x; i < e.count; i += 256) dst[i] = e.value < 0 ? src[i] : e.value + i;
}

// Entries that are a pair's source become its destination; the pairs are in
// ascending order of their sources, and no destination is a source.
__global__ __launch_bounds__(256) void remap_table_kernel(RemapArgs a) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.entries) return;
  const int page = a.table[i];
  int lo = 0, hi = a.n;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.pair[mid].src < page) lo = mid + 1;
    else hi = mid;
  }
  if (lo < a.n && a.pair[lo].src == page) a.table[i] = a.pair[lo].dst;
}

hipError_t launch_copies(const void* const* pools, int n_pools, long long bytes, long long stride,
                         const PageCopy* pairs, int n, hipStream_t stream) {
  CopyArgs a;
  a.stride = stride;
  a.vecs = static_cast<uint32_t>(bytes / 16);
  const unsigned pieces = (a.vecs + kCopyThreads * kCopyUnroll - 1) / (kCopyThreads * kCopyUnroll);
  for (int i = 0; i < n; i += kPairsPerLaunch) {
    const int k = std::min(kPairsPerLaunch, n - i);
    std::copy(pairs + i, pairs + i + k, a.pair);
    for (int j = 0; j < n_pools; j += kPoolsPerLaunch) {
      const int m = std::min(kPoolsPerLaunch, n_pools - j);
      for (int p = 0; p < m; ++p) a.pool[p] = static_cast<char*>(const_cast<void*>(pools[j + p]));
      hipLaunchKernelGGL(copy_pages_kernel, dim3(pieces, static_cast<unsigned>(k), static_cast<unsigned>(m)),
                         dim3(kCopyThreads), 0, stream, a);
    }
  }
  return hipGetLastError();
}

// Pools a launch can address.
int check_pools(const void* const* pools, int n_pools, long long bytes, long long stride) {
  if (n_pools < 0 || (n_pools > 0 && !pools)) return set_error(SANTA_ERR_INVALID, "null pointer argument");
  if (bytes <= 0 || stride < bytes || bytes % 16 != 0 || stride % 16 != 0 || bytes / 16 > (1LL << 30))
    return set_error(SANTA_ERR_INVALID, "pages must be whole 16-byte pieces, up to 16 GiB, that do not overlap");
  for (int i = 0; i < n_pools; ++i)
    if (!pools[i] || reinterpret_cast<uintptr_t>(pools[i]) % 16 != 0)
      return set_error(SANTA_ERR_INVALID, "page pools must be 16-byte aligned");
  return SANTA_OK;
}

// -------------------------------------------------------------------- append
// Strides in elements of a pool: pages, rows, heads.
struct PoolStrides {
  long long page, row, head;
};

struct Pages {
  const int* table;
  long long stride;  // entries per row
  int shift, num_pages;
};

__device__ __forceinline__ int in_pool(const Pages& pg, int page) { return min(max(page, 0), pg.num_pages - 1); }

// y_d = x_d cos_d - x_{d + D/2} sin_d and y_{d + D/2} = x_{d + D/2} cos_{d + D/2}
// + x_d sin_{d + D/2}: a thread takes dims d .. d + 7 and d + D/2 .. d + D/2 + 7
// of one head of one token, the two pieces that the formula combines, so that qkv
// is read and q, k and v are written once, in 16-byte pieces.  Bound by HBM: 27
// thousand tokens of 32 + 2 x 8 heads of 128 in 69 us, 5.7 TB/s read and written;
// one token for each of 64 sequences is latency (3.7 us).
template <bool BF16>
__global__ __launch_bounds__(256) void rope_append_kernel(const uint16_t* __restrict__ qkv,
                                                          const uint16_t* __restrict__ cos_,
                                                          const uint16_t* __restrict__ sin_,
                                                          uint16_t* __restrict__ q_out, uint16_t* __restrict__ k_pages,
                                                          uint16_t* __restrict__ v_pages, int H, int KVH, int D,
                                                          PoolStrides sk, PoolStrides sv, Pages pg,
                                                          const int2* __restrict__ pos, uint32_t total) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= total) return;
  const uint32_t per = static_cast<uint32_t>(D) / 16, heads = static_cast<uint32_t>(H + 2 * KVH);
  const int d = 8 * static_cast<int>(i % per), half = D / 2;
  const int hh = static_cast<int>(i / per % heads);
  const uint32_t t = i / per / heads;
  const uint16_t* src = qkv + (static_cast<size_t>(t) * heads + hh) * D + d;
  u32x4 x0 = *reinterpret_cast<const u32x4*>(src), x1 = *reinterpret_cast<const u32x4*>(src + half);
  uint16_t* dst;
  if (hh < H) {
    dst = q_out + (static_cast<size_t>(t) * H + hh) * D + d;
  } else {
    const int2 at = pos[t];
    if (at.x < 0 || (at.x >> pg.shift) >= pg.stride) return;
    const long long page = in_pool(pg, pg.table[at.y * pg.stride + (at.x >> pg.shift)]);
    const long long row = at.x & ((1 << pg.shift) - 1);
    dst = hh < H + KVH ? k_pages + page * sk.page + row * sk.row + (hh - H) * sk.head + d
                       : v_pages + page * sv.page + row * sv.row + (hh - H - KVH) * sv.head + d;
  }
  if (hh < H + KVH) {
    const uint16_t *cp = cos_ + static_cast<size_t>(t) * D + d, *sp = sin_ + static_cast<size_t>(t) * D + d;
    const u32x4 c0 = *reinterpret_cast<const u32x4*>(cp), c1 = *reinterpret_cast<const u32x4*>(cp + half);
    const u32x4 s0 = *reinterpret_cast<const u32x4*>(sp), s1 = *reinterpret_cast<const u32x4*>(sp + half);
    float y0[8], y1[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      auto at = [k](u32x4 v) { return k & 1 ? hi16_to_f32<BF16>(v[k >> 1]) : lo16_to_f32<BF16>(v[k >> 1]); };
      // one rounding each, to the 16-bit type at the end
      y0[k] = fmaf(at(x0), at(c0), -(at(x1) * at(s0)));
      y1[k] = fmaf(at(x1), at(c1), at(x0) * at(s1));
    }
    x0 = pack8<BF16>(y0);
    x1 = pack8<BF16>(y1);
  }
  *reinterpret_cast<u32x4*>(dst) = x0;
  *reinterpret_cast<u32x4*>(dst + half) = x1;
}

// ----------------------------------------------------------------- attention
// out = sum_n p_n v_n / sum_n p_n over the tokens n <= the row's position, p_n =
// exp(scale q k_n - m), m a running reference near the largest score: one pass
// over K and V.  A row is a (token, query head); the rows of a KV head that read
// the same tokens form a block of up to 256, and read each tile of 64 tokens once:
// the new tokens of a sequence or, over a prefix that sequences have in common,
// those of all of them.  S^T = K Q^T and O^T += V^T P^T by 32x32x16 products, a
// lane holding one row throughout, so that the softmax needs one exchange (with
// the other half of the wave) and P^T never leaves the registers.
//
// One workgroup of 8 waves per compute unit, with a ring of tiles in LDS (128
// KiB: 4 of K and V at D 128, 8 at D 64) that asynchronous loads fill ahead of
// their use and across items.  The plan gives every workgroup a run of items of
// about the same cost, one resident round; long blocks are cut between
// workgroups, and their parts (sum, mass, reference) joined by merge_kernel.
// KV head h's workgroups are those of numbers h modulo the KV heads, so that with
// 8 of them an XCD's L2 holds one head (16 unshared sequences: 280 us, against
// 294 with whole sequences side by side).
//
// The probabilities are rounded to the 16-bit type for the second product in
// batches with several new tokens and more than 32 rows per sequence (a prefill),
// as the prefill over contiguous caches does.  Elsewhere they enter it as two
// values of that type, with a product each, so that a decode step has the values of
// float32 probabilities, however many sequences read the same pages: free up to
// 32 rows, up to a third more time above (both sides in santa_paged_plan.cpp).
//
// What bounds it, at D 128 in bf16.  Few rows: HBM, 5.6 TB/s over 16-token pages
// (16 sequences of 1000 to 40 000 tokens, 32 query and 8 KV heads, 1.55 GB:
// 277 us; half the ring, or two workgroups of half the waves per compute unit,
// change nothing).  256 rows: issue, of the products (0.42 of a SIMD's cycles), of
// the softmax's vector work (about as many) and of the steps between them, which
// hardly overlap: 984 TFLOP/s behind shared prompts (six sequences of 4000 shared,
// 100 to 1300 own and 1300 new tokens, 295 us, and 314 with the join), where a plain
// product of 8192^3 reaches 1202.  Counted cycles of that kernel, 664 thousand as it is: the two
// waves of a SIMD half a tile apart, products of one beside the softmax of the
// other, 685; loads issued between the products 711; steps without bookkeeping
// 667; first products as soon as their first operand is there 661.  A batch behind
// a long prompt has both: 64 sequences behind 32k tokens 114 us, 32 with 64 query and
// 8 KV heads behind 128k 262 us (106 and 215 with rounded probabilities).  Little work: latency, about 10 us for the first
// loads, one tile, the join of the waves and the output.
constexpr int kWaves = 8;
// Above this a row's reference in log2 units is subtracted from the scores before
// they are scaled: fma(score, scale, -round(m * scale)) is off by half an ulp of
// the product, up to here 2^-15, a factor common to the row's probabilities that
// hardly moves what they are rounded to.
constexpr float kExactMax = 512.0f;
constexpr int kBufWord3 = 0x00020000;  // raw buffer descriptor, gfx9 family

typedef int i32x4 __attribute__((ext_vector_type(4)));

// 16 bytes per lane from rs + off (this lane's byte offset) to LDS, 1 KiB from
// byte `at` on in lane order.  As asm, because with the builtin the compiler
// makes the next read of LDS wait for it, whatever it reads; it has no result in
// registers, and the waits are the tile loop's own.
__device__ __forceinline__ void load_lds16(i32x4 rs, uint32_t at, uint32_t off) {
  uint32_t m0;  // kept as it was; the pause is the one that scalars written by the vector unit need before a load
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
               "s_mov_b32 m0, %0"
               : "=&s"(m0)
               : "s"(at), "v"(off), "s"(rs)
               : "memory");
}

template <int D>
struct Geometry {
  static constexpr int kRow = 2 * D;                   // bytes
  static constexpr int kLanes = D / 8;                 // lanes per row
  static constexpr int kRows = 64 / kLanes;            // rows per load instruction
  static constexpr int kLoads = 8 / kRows;             // load instructions per wave, tile and tensor
  static constexpr int kVecs = kTile * kLanes;         // 16-byte pieces per K or V tile
  static constexpr int kStages = 512 / D;              // tiles in LDS, 128 KiB of them
  static constexpr int kStage = 2 * kVecs;             // pieces per stage: the K tile, the V tile
};

// Waits until at most N of this wave's loads are in flight (they land in order;
// loads and stores the compiler has issued since only make it wait for more).
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// How far a row's largest score may exceed the one that its sums are relative to
// before they are rescaled: with none, new maxima among 32 rows rescale most
// tiles (a quarter more vector work); probabilities up to 2^8 round as well as
// those up to 1.
constexpr float kHeadroom = 8.0f;
// Probabilities are held 2^kLift times as large, a factor common to a row's sum and
// mass in every wave and part.  bf16 has float32's exponents.  f16 ends at 2^-24:
// held as they are, probabilities below 2^-25 of the reference would be lost, 0.4 %
// of a row with 131 thousand of them.  Lifted to the type's upper end (2^7 and the
// headroom: 2^15), the limit is 2^-32, and n tokens lose at most n of it.
template <bool BF16>
constexpr float kLift = BF16 ? 0.0f : 7.0f;

template <bool BF16>
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
  return make_uint2(f32_to_h16<BF16>(a) | static_cast<uint32_t>(f32_to_h16<BF16>(b)) << 16,
                    f32_to_h16<BF16>(c) | static_cast<uint32_t>(f32_to_h16<BF16>(d)) << 16);
}

// acc + the eight 16-bit values of v.
template <bool BF16>
__device__ __forceinline__ float sum8(u32x4 v, float acc) {
  typedef typename attn::Half8<BF16>::T H8;
  const H8 x = __builtin_bit_cast(H8, v);
  constexpr uint32_t kOnes = BF16 ? 0x3f803f80u : 0x3c003c00u;
  const H8 one = __builtin_bit_cast(H8, u32x4{kOnes, kOnes, kOnes, kOnes});
  if constexpr (BF16) {
    acc = __builtin_amdgcn_fdot2_f32_bf16(x.s01, one.s01, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(x.s23, one.s01, acc, false);
    acc = __builtin_amdgcn_fdot2_f32_bf16(x.s45, one.s01, acc, false);
    return __builtin_amdgcn_fdot2_f32_bf16(x.s67, one.s01, acc, false);
  } else {
    acc = __builtin_amdgcn_fdot2(x.s01, one.s01, acc, false);
    acc = __builtin_amdgcn_fdot2(x.s23, one.s01, acc, false);
    acc = __builtin_amdgcn_fdot2(x.s45, one.s01, acc, false);
    return __builtin_amdgcn_fdot2(x.s67, one.s01, acc, false);
  }
}

template <class T>
using Const = const __attribute__((address_space(4))) T;  // read through the scalar cache

struct AttnArgs {
  const uint16_t* q;
  const char *k, *v;
  uint16_t* out;
  float *part, *part_ml;  // sums [records, D]; (maximum, mass) [records]
  const Item* items;
  const int* list;
  Pages pg;
  long long sq_t, sq_h;              // elements
  long long sk_h, sv_h;              // bytes
  uint32_t sk_p, sk_r, sv_p, sv_r;
  int KVH, GH;
  float scale_log2;
};

// Where a workgroup's loads are: tile t of an item (in scalar registers), and
// where this wave's eight tokens of 64 tiles lie in K and V, one tile a lane:
// looked up tile by tile as scalars they would be waited for with the loop's
// reads of LDS, and their addresses be formed by every wave.
struct Cursor {
  int begin, end, row, next;      // of the item
  int begin2, end2, row2, next2;  // of the next one
  int t, tiles;                   // of the item
  int left;                       // tokens from this wave's first one of the tile to the end
  uint32_t k_lo, k_hi, v_lo, v_hi;
  bool more;                      // there is a tile
};

struct Loader {
  const char *k, *v;      // this KV head in the pools
  Const<Item>* items;
  const int* table;
  long long stride;
  int shift, num_pages, limit;  // limit: tokens a block table row can name
  uint32_t sk_p, sk_r, sv_p, sv_r;
  uint32_t stages;  // LDS byte address of this wave's part of the first stage
  int wave;
};

__device__ __forceinline__ int tiles_of(int begin, int end) { return (end - begin + kTile - 1) / kTile; }

__device__ __forceinline__ void look_up(const Loader& w, Cursor& c) {
  const int n = min(c.begin + (c.t + static_cast<int>(threadIdx.x & 63)) * kTile + 8 * w.wave, min(c.end, w.limit) - 1);
  const uint32_t page = min(max(w.table[c.row * w.stride + (n >> w.shift)], 0), w.num_pages - 1);
  const uint32_t r = n & ((1 << w.shift) - 1) & ~7;
  const uint64_t p64 = page, r64 = r;
  const uint64_t k = reinterpret_cast<uint64_t>(w.k) + p64 * w.sk_p + r64 * w.sk_r;
  const uint64_t v = reinterpret_cast<uint64_t>(w.v) + p64 * w.sv_p + r64 * w.sv_r;
  c.k_lo = static_cast<uint32_t>(k), c.k_hi = static_cast<uint32_t>(k >> 32) & 0xffff;
  c.v_lo = static_cast<uint32_t>(v), c.v_hi = static_cast<uint32_t>(v >> 32) & 0xffff;
  // waited for here, once in 64 tiles, and not at every use
  asm volatile("" : "+v"(c.k_lo), "+v"(c.k_hi), "+v"(c.v_lo), "+v"(c.v_hi));
}
__device__ __forceinline__ void read_next(const Loader& w, Cursor& c) {
  if (c.next < 0) return;
  Const<Item>* it = w.items + c.next;
  c.begin2 = it->begin, c.end2 = it->end, c.row2 = it->row, c.next2 = it->next;
}
// To the first tile of the next item that has one.
__device__ __forceinline__ void enter_next(const Loader& w, Cursor& c) {
  c.more = false;
  while (c.next >= 0) {
    c.begin = c.begin2, c.end = c.end2, c.row = c.row2, c.next = c.next2;
    read_next(w, c);
    if (c.end > c.begin) {
      c.t = 0;
      c.tiles = tiles_of(c.begin, c.end);
      c.left = c.end - c.begin - 8 * w.wave;
      c.more = true;
      look_up(w, c);
      return;
    }
  }
}

// Issues this wave's loads of the cursor's tile into a stage (tokens 8 wave ..
// 8 wave + 7 of it, which lie in one page, so that their address is a scalar's)
// and moves the cursor on; nothing waits for them here.  Rows past the end read
// as zeros.  A row's 16-byte pieces are swizzled so that the reads of both
// tiles are without bank conflicts.
template <int D>
__device__ __forceinline__ void load_tile(const Loader& w, Cursor& c, uint32_t stage, const uint32_t (&ko)[2],
                                          const uint32_t (&vo)[2]) {
  using G = Geometry<D>;
  const int lane = c.t & 63;
  int k_bytes = 7 * w.sk_r + 2 * D, v_bytes = 7 * w.sv_r + 2 * D;
  if (c.left < 8) {
    k_bytes = c.left > 0 ? (c.left - 1) * w.sk_r + 2 * D : 0;
    v_bytes = c.left > 0 ? (c.left - 1) * w.sv_r + 2 * D : 0;
  }
  const i32x4 rk{static_cast<int>(__builtin_amdgcn_readlane(c.k_lo, lane)),
                 static_cast<int>(__builtin_amdgcn_readlane(c.k_hi, lane)), k_bytes, kBufWord3};
  const i32x4 rv{static_cast<int>(__builtin_amdgcn_readlane(c.v_lo, lane)),
                 static_cast<int>(__builtin_amdgcn_readlane(c.v_hi, lane)), v_bytes, kBufWord3};
  const uint32_t at = w.stages + 16 * G::kStage * stage;
#pragma unroll
  for (int i = 0; i < G::kLoads; ++i) {
    load_lds16(rk, at + 1024 * i, ko[i]);
    load_lds16(rv, at + 1024 * i + 16 * G::kVecs, vo[i]);
  }
  c.left -= kTile;
  if (++c.t == c.tiles) enter_next(w, c);
  else if ((c.t & 63) == 0) look_up(w, c);
}

// How probabilities enter the second product.
enum class Parts {
  kOne,    // rounded to the 16-bit type
  kTwo,    // as the sum of two 16-bit values, each with a product of its own
  kLanes,  // likewise, the second values in lanes that up to 16 rows leave free
  kLanesOfTwo,  // likewise, in a kernel whose other items are kTwo
};

// Probabilities of kTwo are 1 + kMore times as large (cut8); those of kLanesOfTwo,
// whose sums are joined with theirs, have the factor in their exponent.
template <bool BF16>
constexpr float kMore = BF16 ? 0x1p-20f : 0x1p-10f;
template <bool BF16>
constexpr float kMoreLog2 = BF16 ? 1.3758605e-6f : 1.4081944e-3f;  // log2(1 + kMore)

// e cut off to the 16-bit type, and in low what that leaves of e (1 + kMore), as
// 16-bit values.  low has the sign of e and is not 0 where e is not (in f16, where
// e is a normal number): an infinite value of a token keeps its sign in both
// products, where the remainder of a rounding, of either sign or 0, would make it
// NaN.  The factor is common to sum and mass.
template <bool BF16>
__device__ __forceinline__ u32x4 cut8(const float (&e)[8], u32x4& low) {
  u32x4 p;
  float rest[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (BF16) {
      p[j] = __builtin_amdgcn_perm(__float_as_uint(e[2 * j + 1]), __float_as_uint(e[2 * j]), 0x07060302);
    } else {
      p[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(e[2 * j], e[2 * j + 1]));
    }
    rest[2 * j] = fmaf(e[2 * j], 1.0f + kMore<BF16>, -lo16_to_f32<BF16>(p[j]));
    rest[2 * j + 1] = fmaf(e[2 * j + 1], 1.0f + kMore<BF16>, -hi16_to_f32<BF16>(p[j]));
  }
  low = pack8<BF16>(rest);
  return p;
}

// Running softmax of a wave's rows (one per lane of each half): the sum of MB x
// 32 dims and the mass of this half's tokens, relative to m, a score that the
// row's largest exceeds by less than kHeadroom (log2 units).  mc: m in log2
// units; grows: the score above which m moves up; exact: some row's mc is too
// large to scale the scores before m is subtracted (kExactMax).
template <int MB>
struct State {
  f32x16 o[MB];
  float m, l, mc, grows;
  bool exact;
};

// Scores S^T = K Q^T of a tile's 32 KB tokens x 32 rows.  The first fragments of
// K are all asked for before the first product, the rest one by one beside the
// products: left to itself the compiler reads, waits and multiplies in turn.
template <bool BF16, int D, int KB>
__device__ __forceinline__ void scores(const char* buf, const u32x4 (&qf)[D / 16], uint32_t ko, f32x16 (&s)[KB]) {
  asm volatile("" : "+v"(ko));  // its parts are formed here and not kept over the loop
  u32x4 k[KB][D / 16];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      k[kb][c] = *reinterpret_cast<const u32x4*>(buf + (ko ^ (32 * c)) + 32 * Geometry<D>::kRow * kb);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) s[kb] = mfma32<BF16>(k[kb][c], qf[c], s[kb]);
  }
  __builtin_amdgcn_sched_group_barrier(0x100, D / 16, 0);  // LDS reads
#pragma unroll
  for (int i = 0; i < D / 16 * (KB - 1); ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix products
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, D / 16, 0);
}

// Their softmax: P^T in the 16-bit type, the running state moved on.  kMasked:
// the lane's row attends to the first lim + 1 of the tokens.
template <bool BF16, int KB, int MB, bool kMasked, Parts kParts>
__device__ __forceinline__ void softmax(f32x16 (&s)[KB], u32x4 (&p)[2 * KB], u32x4 (&low)[2 * KB], int lim,
                                        float scale_log2, State<MB>& st) {
  const int lane = threadIdx.x & 63;
  if constexpr (kMasked) {
    const int left = lim - 4 * (lane >> 5);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (32 * kb + 8 * (e >> 2) + (e & 3) > left) s[kb][e] = -__builtin_inff();
  }
  float mx = s[0][0];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
  mx = fmaxf(mx, other_half(mx));
  const bool up = mx > st.grows;
  if (__any(up)) {
    const float m = up ? fmaxf(st.m, mx) : st.m;
    const float w = __builtin_amdgcn_exp2f((st.m - m) * scale_log2);
    st.l *= w;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[mb][e] *= w;
    st.m = m;
    st.mc = m * scale_log2;
    if (up) st.grows = m + kHeadroom / scale_log2;
    st.exact = __any(fabsf(st.mc) > kExactMax);
  }
  constexpr bool kLanes = kParts == Parts::kLanes || kParts == Parts::kLanesOfTwo;
  constexpr float kUp = kLift<BF16> + (kParts == Parts::kLanesOfTwo ? kMoreLog2<BF16> : 0.0f);
  float mc = st.mc - kUp;
  if (st.exact) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] -= st.m;
    mc = -kUp;
  }
#pragma unroll
  for (int kc = 0; kc < 2 * KB; ++kc) {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(s[kc >> 1][8 * (kc & 1) + j], scale_log2, -mc));
    if constexpr (kParts == Parts::kTwo) {
      p[kc] = cut8<BF16>(e, low[kc]);
      st.l = sum8<BF16>(low[kc], st.l);
    } else {
      p[kc] = pack8<BF16>(e);
    }
    // up to 16 rows leave lanes 16 .. 31 of the wave free: they hold the same
    // rows again, and carry what rounding took from their probabilities
    if constexpr (kLanes) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        e[j] -= lo16_to_f32<BF16>(p[kc][j >> 1]);
        e[j + 1] -= hi16_to_f32<BF16>(p[kc][j >> 1]);
      }
      const u32x4 rest = pack8<BF16>(e);
      if (lane & 16) p[kc] = rest;
    }
    // the mass of the probabilities as rounded: a row's weights sum to 1, and one
    // that attends to one token gives its value
    st.l = sum8<BF16>(p[kc], st.l);
  }
}

// O^T += V^T P^T over MB x 32 dims; the reads of V run ahead of the products as
// those of K do.
template <bool BF16, int D, int KB, int MB, Parts kParts>
__device__ __forceinline__ void sums(const char* buf, uint32_t vo, const u32x4 (&p)[2 * KB],
                                     const u32x4 (&low)[2 * KB], State<MB>& st) {
  asm volatile("" : "+v"(vo));
  using G = Geometry<D>;
  constexpr int N = 2 * KB * MB, kAhead = N < 4 ? N : 4, kProducts = kParts == Parts::kTwo ? 2 : 1;
  u32x4 v[2 * KB][MB];
#pragma unroll
  for (int kc = 0; kc < 2 * KB; ++kc)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) v[kc][mb] = read_tr8<G::kRow>(buf + (vo ^ (64 * mb)) + 16 * G::kRow * kc);
#pragma unroll
  for (int kc = 0; kc < 2 * KB; ++kc) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) st.o[mb] = mfma32<BF16>(v[kc][mb], p[kc], st.o[mb]);
    if constexpr (kParts == Parts::kTwo) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) st.o[mb] = mfma32<BF16>(v[kc][mb], low[kc], st.o[mb]);
    }
  }
  __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);  // LDS reads
#pragma unroll
  for (int i = 0; i < N - kAhead; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, kProducts, 0);  // matrix products
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, kProducts * kAhead, 0);
}

// Whether 32 KB rows of a V tile hold an infinity or a NaN.
template <bool BF16, int D, int KB>
__device__ __forceinline__ bool not_finite(const char* rows) {
  constexpr uint32_t kStep = BF16 ? 0x00800080 : 0x04000400;  // carries an exponent of all ones into the sign's bit
  uint32_t bad = 0;
#pragma unroll 4
  for (int i = 0; i < 32 * KB * Geometry<D>::kRow / 1024; ++i) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(rows + 1024 * i + 16 * (threadIdx.x & 63));
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= (v[j] & 0x7fff7fff) + kStep;
  }
  return __any((bad & 0x80008000) != 0);
}

// sums() for a tile of which some rows do not attend to all tokens.  Where a
// value there is not finite (apart), and would not vanish with a probability of
// 0: for one last token after the other, the values behind it left out, and the
// result kept by the rows that end there.
template <bool BF16, int D, int KB, int MB, Parts kParts>
__device__ __forceinline__ void sums_masked(const char* buf, uint32_t vo, const u32x4 (&p)[2 * KB],
                                            const u32x4 (&low)[2 * KB], int n0, int last, int lim, int lim_lo,
                                            int lim_hi, bool apart, State<MB>& st) {
  using G = Geometry<D>;
  const int most = apart ? min(lim_hi, last) : last;
  for (int end = apart ? max(lim_lo, n0) : last; end <= most; ++end) {
    const int left = end - n0 - 4 * (static_cast<int>(threadIdx.x & 63) >> 5);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      u32x4 v[2 * KB];
#pragma unroll
      for (int kc = 0; kc < 2 * KB; ++kc) v[kc] = read_tr8<G::kRow>(buf + (vo ^ (64 * mb)) + 16 * G::kRow * kc);
      if (!apart) {
#pragma unroll
        for (int kc = 0; kc < 2 * KB; ++kc) {
          st.o[mb] = mfma32<BF16>(v[kc], p[kc], st.o[mb]);
          if constexpr (kParts == Parts::kTwo) st.o[mb] = mfma32<BF16>(v[kc], low[kc], st.o[mb]);
        }
      } else {
        f32x16 o = st.o[mb];
#pragma unroll
        for (int kc = 0; kc < 2 * KB; ++kc) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int n = 16 * kc + 8 * (j >> 1) + 2 * (j & 1);  // of the dword's first value
            v[kc][j] = n < left ? v[kc][j] : n == left ? v[kc][j] & 0xffff : 0;
          }
          o = mfma32<BF16>(v[kc], p[kc], o);
          if constexpr (kParts == Parts::kTwo) o = mfma32<BF16>(v[kc], low[kc], o);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) st.o[mb][e] = min(lim, last) == end ? o[e] : st.o[mb][e];
      }
    }
  }
}

// The workgroup's barrier alone: no wave waits for its loads here.
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// LDS beside the stages, for what the waves of the same rows and dims hold of
// different tokens.
struct Shares {
  float4 o[24][64];
  float m[kWaves][64], l[kWaves][64];
};

// One item.  Its rows are RG groups of 32, each held by 8 / RG waves.  RG 8: one
// wave has all of a tile.  4: two waves, each a half of its tokens.  2: four
// waves, each a half of its tokens and of the dims.  1: eight waves, each a half
// of the dims and a quarter of the tokens of two tiles (with four waves to a
// tile, its latency, not HBM, would bound the pass).  tile: the number of the
// item's first tile, loaded: that of the next one to be loaded, counted over the
// workgroup's items.
template <bool BF16, int D, int RG, Parts kParts>
__device__ __forceinline__ void attend(const AttnArgs& a, const Item& it, int kv, const Loader& w, Cursor& cur,
                                       const uint32_t (&lk)[2], const uint32_t (&lv)[2], uint32_t& tile,
                                       uint32_t& loaded, u32x4* stages, Shares* x) {
  using G = Geometry<D>;
  constexpr int KB = RG == 8 ? 2 : 1;                       // 32s of a tile's tokens that a wave takes
  constexpr int DH = RG >= 4 ? 1 : 2, MB = D / 32 / DH;     // parts of the dims, 32s of them in each
  constexpr int TG = RG == 8 ? 1 : RG == 1 ? 4 : 2;         // parts of the tokens
  constexpr int kStep = RG == 1 ? 2 : 1;                    // tiles at once
  // opaque, so that what depends on it is formed here: the offsets of all four
  // forms, kept over all items, would not fit the registers
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  const int half = lane >> 5, ql = lane & 31;
  const int wave = w.wave;
  const int dh = DH == 1 ? 0 : wave & 1, tg = wave / DH % TG, rg = wave / (DH * TG);
  const int kh = TG == 1 ? 0 : tg & 1;                      // half of a tile
  constexpr bool dup = kParts == Parts::kLanes || kParts == Parts::kLanesOfTwo;

  // this lane's row
  const int r = dup ? ql & 15 : 32 * rg + ql;
  const int rc = min(r, it.rows - 1);
  const int i = rc / a.GH, h = kv * a.GH + (rc - i * a.GH);
  const int tok = it.flags & kFromList ? a.list[it.tok0 + i] : it.tok0 + i;
  const int pos = it.pos0 + i;
  const int lim = min(it.end - 1, pos);  // last position this row attends to here
  const int lim_lo = __builtin_amdgcn_readlane(lim, 0), lim_hi = __builtin_amdgcn_readlane(lim, 31);
  const bool any = 32 * rg < it.rows;

  // Q fragments: dims 16c + 8 half .. + 7 of this lane's row
  u32x4 qf[D / 16];
  {
    const uint16_t* qr = a.q + tok * a.sq_t + h * a.sq_h + 8 * half;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = *reinterpret_cast<const u32x4*>(qr + 16 * c);
  }
  // LDS byte offsets inside a stage of this lane's first fragments; those of
  // further dims lie at these numbers with some bits flipped (the swizzle)
  const uint32_t ko = (ql + 32 * kh) * G::kRow + 16 * (half ^ (D == 128 ? ql & 15 : (ql >> 1) & 7));
  const int r3 = (lane & 15) >> 2, piece = 4 * MB * dh + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t vo = 16 * G::kVecs + (4 * half + r3 + 32 * kh) * G::kRow +
                      16 * (piece ^ (D == 128 ? 4 * r3 : 4 * (r3 >> 1))) + 8 * (lane & 1);

  State<MB> st;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int e = 0; e < 16; ++e) st.o[mb][e] = 0.0f;
  st.m = kLowest;
  st.l = st.mc = 0.0f;
  st.grows = -__builtin_inff();
  st.exact = false;
  // Q has landed: known here, it is not waited for in every tile
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) alone
  const int nt = tiles_of(it.begin, it.end);
  const int mine = kStep == 1 ? 0 : tg >> 1, first = it.begin + 32 * kh;  // tile of the step, token of the tile 0
  // tiles in which a row of this wave attends to a token; and those of them in
  // which all rows attend to all
  const int busy = any && lim_hi >= it.begin ? min(nt, (lim_hi - it.begin) / kTile + 1) : 0;
  const int whole = min(busy, (max(lim_lo + 1 - first - 32 * KB, -kTile) + kTile) / kTile);
  // To the step of tile t: this wave's loads of its tiles have landed (those of
  // newer ones need not have), then all waves' have, and no wave reads the tiles
  // before any more, whose places are loaded anew.
  auto enter = [&](int t) {
    const int newer = static_cast<int>(loaded - tile) - min(kStep, nt - t);
    constexpr int kMost = G::kStages - 1 - kStep, kSome = kMost / 2;
    if (newer >= kMost) wait_loads<2 * G::kLoads * kMost>();
    else if (newer >= kSome) wait_loads<2 * G::kLoads * kSome>();
    else wait_loads<0>();
    barrier();
    while (cur.more && loaded - tile < G::kStages)
      load_tile<D>(w, cur, loaded++ % G::kStages, lk, lv);
    const uint32_t at = tile + mine;
    tile += min(kStep, nt - t);
    return reinterpret_cast<const char*>(stages + (at % G::kStages) * G::kStage);
  };
  int t = 0;
  for (; t + mine < whole; t += kStep) {
    const char* stage = enter(t);
    f32x16 s[KB];
    u32x4 p[2 * KB], low[2 * KB];
    scores<BF16, D, KB>(stage, qf, ko, s);
    softmax<BF16, KB, MB, false, kParts>(s, p, low, 0, a.scale_log2, st);
    sums<BF16, D, KB, MB, kParts>(stage, vo, p, low, st);
  }
  for (; t < nt; t += kStep) {  // a loop of its own, or both would run short of registers
    const char* stage = enter(t);
    if (t + mine >= busy) continue;
    f32x16 s[KB];
    u32x4 p[2 * KB], low[2 * KB];
    const int n0 = first + (t + mine) * kTile, last = min(it.end, n0 + 32 * KB) - 1;
    scores<BF16, D, KB>(stage, qf, ko, s);
    softmax<BF16, KB, MB, true, kParts>(s, p, low, lim - n0, a.scale_log2, st);
    const bool apart = last > lim_lo && not_finite<BF16, D, KB>(stage + 16 * G::kVecs + 32 * kh * G::kRow);
    sums_masked<BF16, D, KB, MB, kParts>(stage, vo, p, low, n0, last, lim, lim_lo, lim_hi, apart, st);
  }
  float m = st.m, l = st.l + other_half(st.l);
  f32x16(&o)[MB] = st.o;
  if constexpr (dup) {  // an infinite value is whole in the first part, and times 0 or less in the second
    l += fxor<16>(l, lane);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float low = fxor<16>(o[mb][e], lane);
        o[mb][e] += fabsf(low) < __builtin_inff() ? low : 0.0f;
      }
  }
  // The parts of the tokens, each wave joining a share of the dims: EP of the
  // four pieces that it has of every 32 of them.
  constexpr int EP = 4 / TG;
  float4 res[MB][EP];
  if constexpr (TG == 1) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int k = 0; k < EP; ++k)
        res[mb][k] = make_float4(o[mb][4 * k], o[mb][4 * k + 1], o[mb][4 * k + 2], o[mb][4 * k + 3]);
  } else {
    const int team = TG * (wave % DH + DH * rg);  // its waves' number: team + tg
    auto place = [&](int to, int from, int k) {
      return x->o[((team + to) * (TG - 1) + (from < to ? from : from - 1)) * EP + k] + lane;
    };
    x->m[team + tg][lane] = m;
    x->l[team + tg][lane] = l;
    float own = 0.0f, weight[TG - 1];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
      for (int to = 0; to < TG; ++to)
#pragma unroll
        for (int k = 0; k < EP; ++k) {
          const int e = 4 * (to * EP + k);
          const float4 v = make_float4(o[mb][e], o[mb][e + 1], o[mb][e + 2], o[mb][e + 3]);
          if (to == tg) res[mb][k] = v;
          else *place(to, tg, k) = v;
        }
      __syncthreads();
      if (mb == 0) {
        float top = m;
#pragma unroll
        for (int i = 0; i < TG; ++i) top = fmaxf(top, x->m[team + i][lane]);
        own = __builtin_amdgcn_exp2f((m - top) * a.scale_log2);
        l *= own;
        m = top;
#pragma unroll
        for (int i = 0; i < TG - 1; ++i) {
          const int from = team + (i < tg ? i : i + 1);
          weight[i] = __builtin_amdgcn_exp2f((x->m[from][lane] - top) * a.scale_log2);
          l = fmaf(x->l[from][lane], weight[i], l);
        }
      }
#pragma unroll
      for (int k = 0; k < EP; ++k) {
        float4& c = res[mb][k];
        c.x *= own, c.y *= own, c.z *= own, c.w *= own;
#pragma unroll
        for (int i = 0; i < TG - 1; ++i) {
          const float4 v = *place(tg, i < tg ? i : i + 1, k);
          c.x = fmaf(v.x, weight[i], c.x), c.y = fmaf(v.y, weight[i], c.y);
          c.z = fmaf(v.z, weight[i], c.z), c.w = fmaf(v.w, weight[i], c.w);
        }
      }
      __syncthreads();
    }
    if (dup && (ql & 16)) return;
  }
  if (!any || r >= it.rows) return;
  const int d0 = 32 * MB * dh + (TG == 1 ? 0 : 8 * EP * tg) + 4 * half;  // of the first piece
  if (it.flags & kDirect) {
    const float inv = pos < 0 ? 0.0f : 1.0f / l;
    uint16_t* orow = a.out + (static_cast<size_t>(tok) * (a.KVH * a.GH) + h) * D + d0;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int k = 0; k < EP; ++k) {
        const float4& c = res[mb][k];
        *reinterpret_cast<uint2*>(orow + 32 * mb + 8 * k) = pack4<BF16>(c.x * inv, c.y * inv, c.z * inv, c.w * inv);
      }
    return;
  }
  const size_t rec = static_cast<size_t>(it.base) + static_cast<size_t>(kv) * it.rows + r;
  float* prow = a.part + rec * D + d0;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int k = 0; k < EP; ++k) *reinterpret_cast<float4*>(prow + 32 * mb + 8 * k) = res[mb][k];
  if (dh == 0 && tg == 0 && half == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * rec) = make_float2(m, l);
}

__device__ __forceinline__ Item read_item(const Loader& w, int i) {
  Const<Item>* p = w.items + i;
  Item it;
  it.flags = p->flags, it.row = p->row, it.begin = p->begin, it.end = p->end, it.tok0 = p->tok0, it.rows = p->rows;
  it.pos0 = p->pos0, it.base = p->base, it.next = p->next;
  return it;
}

template <bool BF16, int D, Parts kParts>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_attention_kernel(AttnArgs a) {
  using G = Geometry<D>;
  __shared__ u32x4 stages[G::kStages * G::kStage];
  __shared__ Shares shares;
  constexpr Parts kLanes = kParts == Parts::kTwo ? Parts::kLanesOfTwo : Parts::kLanes;
  const int kv = blockIdx.x % a.KVH, group = blockIdx.x / a.KVH;
  const int lane = threadIdx.x & 63;
  Loader w;
  w.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  w.k = a.k + kv * a.sk_h;
  w.v = a.v + kv * a.sv_h;
  w.items = (Const<Item>*)a.items;
  w.table = a.pg.table;
  w.stride = a.pg.stride;
  w.shift = a.pg.shift;
  w.num_pages = a.pg.num_pages;
  w.limit = static_cast<int>(min(a.pg.stride << a.pg.shift, 0x7fffffffLL));
  w.sk_p = a.sk_p, w.sk_r = a.sk_r, w.sv_p = a.sv_p, w.sv_r = a.sv_r;
  w.stages = __builtin_amdgcn_readfirstlane(
                 static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)stages))) +
             1024 * G::kLoads * w.wave;
  uint32_t lk[2], lv[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = G::kRows * i + lane / G::kLanes, slot = lane % G::kLanes;
    const int pr = 8 * w.wave + row;  // row of the tile
    lk[i] = row * a.sk_r + 16 * (slot ^ (D == 128 ? pr & 15 : (pr >> 1) & 7));
    lv[i] = row * a.sv_r + 16 * (slot ^ (D == 128 ? 4 * (pr & 3) : 4 * ((pr >> 1) & 1)));
  }
  Cursor c;
  c.next = group;
  const int item = c.next;
  uint32_t tile = 0, loaded = 0;
  read_next(w, c);
  enter_next(w, c);
  for (; loaded < G::kStages - 1 && c.more; ++loaded)
    load_tile<D>(w, c, loaded, lk, lv);
  Item it = read_item(w, item);
  for (bool last = false; !last && it.rows > 0;) {
    const Item now = it;
    last = now.next < 0;
    if (!last) it = read_item(w, now.next);  // while this one is worked on
    if (now.rows <= 16) attend<BF16, D, 1, kLanes>(a, now, kv, w, c, lk, lv, tile, loaded, stages, &shares);
    else if (now.rows <= 32) attend<BF16, D, 1, kParts>(a, now, kv, w, c, lk, lv, tile, loaded, stages, &shares);
    else if (now.rows <= 64) attend<BF16, D, 2, kParts>(a, now, kv, w, c, lk, lv, tile, loaded, stages, &shares);
    else if (now.rows <= 128) attend<BF16, D, 4, kParts>(a, now, kv, w, c, lk, lv, tile, loaded, stages, &shares);
    else attend<BF16, D, 8, kParts>(a, now, kv, w, c, lk, lv, tile, loaded, stages, &shares);
  }
}

// Joins the parts of a (token, head): D / 4 lanes, a team, hold four dims each of
// every part that they take, in one pass with a running maximum.  kOne: the teams
// of a workgroup take the parts of one row in turn; otherwise each has a row of its
// own.  Parts come in fixed order, so that the same call gives the same bits.
// Latency bound with few rows (128 rows 3.7 us, 2048 of about 14 parts 6.6); 58
// thousand rows of two parts, 75 MB: 19 us, 3.9 TB/s.
template <bool BF16, int D, bool kOne>
__global__ __launch_bounds__(256) void merge_kernel(const float* __restrict__ part, const float2* __restrict__ part_ml,
                                                    const int* __restrict__ tokens, const int4* __restrict__ parts,
                                                    const int2* __restrict__ pos, int first_row, int rows, int H,
                                                    int KVH, float scale_log2, uint16_t* __restrict__ out) {
  constexpr int kTeam = D / 4, kTeams = 256 / kTeam, kStep = kOne ? kTeams : 1, kBatch = 4;
  __shared__ float s_m[kTeams], s_z[kTeams];
  __shared__ float4 s_o[kTeams][kTeam];
  const int team = threadIdx.x / kTeam, d4 = threadIdx.x % kTeam;
  const int row = kOne ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x) * kTeams + team;
  if (row >= rows) return;  // of all the workgroup or, without a barrier below, of some teams
  const int tok = tokens[(first_row + row) / H], h = (first_row + row) % H;
  if (tok < 0) return;
  const int4 pa = parts[2 * tok], pb = parts[2 * tok + 1];  // base, rows, local, splits
  if (pb.w <= 0) return;                                    // written by its item
  const bool blind = pos[tok].x < 0;
  const int n = pa.w + pb.w, kv = h / (H / KVH), g = h % (H / KVH);
  auto record = [&](int j) {
    const bool first = j < pa.w;
    return static_cast<size_t>(first ? pa.x : pb.x) +
           (static_cast<size_t>(first ? j : j - pa.w) * KVH + kv) * (first ? pa.y : pb.y) + (first ? pa.z : pb.z) + g;
  };
  float m = kLowest, z = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float mj, float zj, const float4& o) {
    const float e = __builtin_amdgcn_exp2f((mj - m) * scale_log2);
    z = fmaf(e, zj, z);
    acc.x = fmaf(e, o.x, acc.x), acc.y = fmaf(e, o.y, acc.y);
    acc.z = fmaf(e, o.z, acc.z), acc.w = fmaf(e, o.w, acc.w);
  };
  for (int j0 = kOne ? team : 0; j0 < n; j0 += kBatch * kStep) {
    float2 ml[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const size_t rec = record(min(j0 + b * kStep, n - 1));
      ml[b] = part_ml[rec];
      v[b] = *reinterpret_cast<const float4*>(part + rec * D + 4 * d4);
    }
    float top = m;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) top = fmaxf(top, ml[b].x);  // the last part stands for those past the end
    const float w = __builtin_amdgcn_exp2f((m - top) * scale_log2);
    z *= w, acc.x *= w, acc.y *= w, acc.z *= w, acc.w *= w;
    m = top;
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (j0 + b * kStep < n) add(ml[b].x, ml[b].y, v[b]);
  }
  if constexpr (kOne) {
    if (d4 == 0) s_m[team] = m, s_z[team] = z;
    s_o[team][d4] = acc;
    __syncthreads();
    if (team > 0) return;
#pragma unroll
    for (int t = 1; t < kTeams; ++t) m = fmaxf(m, s_m[t]);
    z = 0.0f;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int t = 0; t < kTeams; ++t) add(s_m[t], s_z[t], s_o[t][d4]);
  }
  const float inv = blind ? 0.0f : 1.0f / z;
  *reinterpret_cast<uint2*>(out + (static_cast<size_t>(tok) * H + h) * D + 4 * d4) =
      pack4<BF16>(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
}

// A block table, pools and plan that belong together.
int check_paged(const void* q, const void* k, const void* v, const void* out, int dtype, int num_pages, int page_size,
                const long long* strides, int n_strides, const int* table, long long table_stride, int table_rows,
                const santa_paged_plan_info* info, const int* plan, const char* what, Pages* pg) {
  if (!q || !k || !v || !out || !strides || !table || !info || !plan || (dtype != SANTA_BF16 && dtype != SANTA_F16) ||
      info->kv_heads <= 0 || info->heads % info->kv_heads != 0 || info->heads <= 0)
    return set_error(SANTA_ERR_INVALID, "bad %s arguments", what);
  const int rc = check_page_size(page_size);
  if (rc != SANTA_OK) return rc;
  if (num_pages <= 0) return set_error(SANTA_ERR_INVALID, "num_pages must be > 0; got %d", num_pages);
  if (info->max_row >= table_rows)
    return set_error(SANTA_ERR_INVALID, "the plan names block table row %d of %d", info->max_row, table_rows);
  const long long need = (static_cast<long long>(info->max_len) + page_size - 1) / page_size;
  if (table_stride < std::max(1LL, need))
    return set_error(SANTA_ERR_INVALID, "block table too narrow: %lld entries per sequence, %lld needed for %d tokens",
                     table_stride, need, info->max_len);
  bool ok = true;
  for (int i = 0; i < n_strides; ++i) ok = ok && strides[i] >= 0 && strides[i] % 8 == 0;
  for (const void* p : {q, k, v, out}) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  if (!ok || reinterpret_cast<uintptr_t>(plan) % 16 != 0)
    return set_error(SANTA_ERR_INVALID, "%s: strides must be multiples of 8 elements and the tensors 16-byte aligned",
                     what);
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  *pg = Pages{table, table_stride, shift, num_pages};
  return SANTA_OK;
}

}  // namespace paged
}  // namespace santa

using namespace santa;

extern "C" int santa_paged_copy(const void* const* pools, int n_pools, long long page_bytes, long long page_stride,
                                int num_pages, const int* pairs, int n, hipStream_t stream) {
  if (n < 0 || (n > 0 && !pairs)) return set_error(SANTA_ERR_INVALID, "null pointer argument");
  const int rc = paged::check_pools(pools, n_pools, page_bytes, page_stride);
  if (rc != SANTA_OK) return rc;
  try {
    std::vector<int> dst(static_cast<size_t>(n));
    for (int i = 0; i < n; ++i) {
      if (pairs[2 * i] < 0 || pairs[2 * i] >= num_pages || pairs[2 * i + 1] < 0 || pairs[2 * i + 1] >= num_pages)
        return set_error(SANTA_ERR_INVALID, "no page %d or %d in a pool of %d", pairs[2 * i], pairs[2 * i + 1],
                         num_pages);
      dst[i] = pairs[2 * i + 1];
    }
    std::sort(dst.begin(), dst.end());
    const auto twice = std::adjacent_find(dst.begin(), dst.end());
    if (twice != dst.end()) return set_error(SANTA_ERR_INVALID, "page %d is written twice", *twice);
    for (int i = 0; i < n; ++i)
      if (std::binary_search(dst.begin(), dst.end(), pairs[2 * i]))
        return set_error(SANTA_ERR_INVALID, "page %d is both read and written", pairs[2 * i]);
  } catch (const std::bad_alloc&) {
    return set_error(SANTA_ERR_INVALID, "out of host memory");
  }
  const hipError_t e = paged::launch_copies(pools, n_pools, page_bytes, page_stride,
                                            reinterpret_cast<const PageCopy*>(pairs), n, stream);
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "page copy launch failed: %s", hipGetErrorString(e));
  return clear_error();
}

extern "C" int santa_pages_apply(const santa_pages* p, const void* const* pools, int n_pools, long long page_bytes,
                                 long long page_stride, int* table, long long table_stride, int max_seqs,
                                 hipStream_t stream) {
  const int *copies, *edits;
  int n_copies, n_edits, remap;
  if (!p || !table) return set_error(SANTA_ERR_INVALID, "null pointer argument");
  int rc = paged::check_pools(pools, n_pools, page_bytes, page_stride);
  if (rc != SANTA_OK) return rc;
  rc = santa_pages_changes(p, &copies, &n_copies, &edits, &n_edits, &remap);
  if (rc != SANTA_OK) return rc;
  const PageCopy* pairs = reinterpret_cast<const PageCopy*>(copies);
  hipError_t e = paged::launch_copies(pools, n_pools, page_bytes, page_stride, pairs, n_copies, stream);
  if (n_edits > 0) {
    paged::EditArgs a;
    a.table = table;
    a.stride = table_stride;
    for (int i = 0; i < n_edits; i += paged::kEditsPerLaunch) {
      const int k = std::min(paged::kEditsPerLaunch, n_edits - i);
      const TableEdit* from = reinterpret_cast<const TableEdit*>(edits) + i;
      std::copy(from, from + k, a.edit);
      hipLaunchKernelGGL(paged::edit_table_kernel, dim3(static_cast<unsigned>(k)), dim3(256), 0, stream, a);
    }
  }
  if (remap) {
    paged::RemapArgs a;
    a.table = table;
    a.entries = table_stride * max_seqs;
    for (int i = 0; i < n_copies; i += paged::kPairsPerLaunch) {
      a.n = std::min(paged::kPairsPerLaunch, n_copies - i);
      std::copy(pairs + i, pairs + i + a.n, a.pair);
      hipLaunchKernelGGL(paged::remap_table_kernel, dim3(static_cast<unsigned>((a.entries + 255) / 256)), dim3(256), 0,
                         stream, a);
    }
  }
  if (e == hipSuccess) e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "page update launch failed: %s", hipGetErrorString(e));
  return clear_error();
}

extern "C" int santa_paged_rope_append(const void* qkv, const void* cos_, const void* sin_, void* q_out, void* k_pages,
                                       void* v_pages, int dtype, int D, int num_pages, int page_size,
                                       const long long* strides, const int* table, long long table_stride,
                                       int table_rows, const santa_paged_plan_info* info, const int* plan,
                                       hipStream_t stream) {
  paged::Pages pg;
  const int rc = paged::check_paged(qkv, k_pages, v_pages, q_out, dtype, num_pages, page_size, strides, 6, table,
                                    table_stride, table_rows, info, plan, "rope_append", &pg);
  if (rc != SANTA_OK) return rc;
  if (!cos_ || !sin_ || (reinterpret_cast<uintptr_t>(cos_) | reinterpret_cast<uintptr_t>(sin_)) % 16 != 0)
    return set_error(SANTA_ERR_INVALID, "rope_append: cos and sin must be 16-byte aligned");
  if (D <= 0 || D % 16 != 0)
    return set_error(SANTA_ERR_UNSUPPORTED, "rope_append: D must be a multiple of 16. Got D=%d", D);
  const int H = info->heads, KVH = info->kv_heads;
  const long long total = static_cast<long long>(info->tokens) * (H + 2LL * KVH) * (D / 16);
  if (total >= 0x7fffff00LL) return set_error(SANTA_ERR_INVALID, "too many new tokens");
  if (total > 0) {
    const paged::PoolStrides sk{strides[0], strides[1], strides[2]}, sv{strides[3], strides[4], strides[5]};
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0, stream,
                         static_cast<const uint16_t*>(qkv), static_cast<const uint16_t*>(cos_),
                         static_cast<const uint16_t*>(sin_), static_cast<uint16_t*>(q_out),
                         static_cast<uint16_t*>(k_pages), static_cast<uint16_t*>(v_pages), H, KVH, D, sk, sv, pg,
                         reinterpret_cast<const int2*>(plan + info->pos_at), static_cast<uint32_t>(total));
    };
    if (dtype == SANTA_BF16) launch(paged::rope_append_kernel<true>);
    else launch(paged::rope_append_kernel<false>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "rope_append launch failed: %s", hipGetErrorString(e));
  return clear_error();
}

extern "C" size_t santa_paged_workspace_size(const santa_paged_plan_info* info, int D) {
  if (!info || info->records < 0 || D <= 0) return 0;
  return static_cast<size_t>(info->records) * (static_cast<size_t>(D) + 2) * sizeof(float);
}

extern "C" int santa_paged_attention(const void* q, const void* k_pages, const void* v_pages, void* out, int dtype,
                                     int D, int num_pages, int page_size, const long long* strides, const int* table,
                                     long long table_stride, int table_rows, const santa_paged_plan_info* info,
                                     const int* plan, float scale, void* workspace, size_t workspace_bytes,
                                     hipStream_t stream) {
  using namespace paged;
  Pages pg;
  const int rc = check_paged(q, k_pages, v_pages, out, dtype, num_pages, page_size, strides, 8, table, table_stride,
                             table_rows, info, plan, "paged_attention", &pg);
  if (rc != SANTA_OK) return rc;
  if (D != 64 && D != 128)
    return set_error(SANTA_ERR_UNSUPPORTED, "paged_attention: D must be 64 or 128. Got D=%d", D);
  if (info->records > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0))
    return set_error(SANTA_ERR_INVALID, "paged_attention: the workspace must be 16-byte aligned");
  if (workspace_bytes < santa_paged_workspace_size(info, D))
    return set_error(SANTA_ERR_WORKSPACE, "paged_attention: workspace too small");
  const int H = info->heads, KVH = info->kv_heads;
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const char*>(k_pages);
  a.v = static_cast<const char*>(v_pages);
  a.out = static_cast<uint16_t*>(out);
  a.part = static_cast<float*>(workspace);
  a.part_ml = a.part + static_cast<size_t>(info->records) * D;
  a.items = reinterpret_cast<const Item*>(plan);
  a.list = plan + info->list_at;
  a.pg = pg;
  a.sq_t = strides[0], a.sq_h = strides[1];
  if (strides[2] >= 1LL << 31 || strides[5] >= 1LL << 31)
    return set_error(SANTA_ERR_UNSUPPORTED, "paged_attention: pages must lie less than 4 GiB apart");
  // rows past the end are told by their offset from the first of eight
  if (strides[3] < D || strides[6] < D || strides[3] >= 1LL << 26 || strides[6] >= 1LL << 26)
    return set_error(SANTA_ERR_UNSUPPORTED,
                     "paged_attention: the rows of a page must lie at least D and less than 2^26 elements apart");
  a.sk_p = static_cast<uint32_t>(2 * strides[2]), a.sk_r = static_cast<uint32_t>(2 * strides[3]);
  a.sv_p = static_cast<uint32_t>(2 * strides[5]), a.sv_r = static_cast<uint32_t>(2 * strides[6]);
  a.sk_h = 2 * strides[4], a.sv_h = 2 * strides[7];
  a.KVH = KVH;
  a.GH = H / KVH;
  a.scale_log2 = 1.44269504088896340736f * scale;
  // maxima are those of the raw scores, and kHeadroom is divided by the scale
  if (!(scale > 0.0f) || !std::isnormal(scale) || !std::isnormal(a.scale_log2))
    return set_error(SANTA_ERR_INVALID, "paged_attention: scale must be positive and finite. Got scale=%g",
                     static_cast<double>(scale));
  auto run = [&](auto bf, auto dim) {
    constexpr bool BF16 = decltype(bf)::value;
    constexpr int kD = decltype(dim)::value;
    auto attend = [&](auto kernel) {  // one resident round
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(info->groups) * KVH), dim3(64 * kWaves), 0, stream, a);
    };
    if (info->groups > 0) {
      if (info->rounded) attend(paged_attention_kernel<BF16, kD, Parts::kOne>);
      else attend(paged_attention_kernel<BF16, kD, Parts::kTwo>);
    }
    const long long rows = static_cast<long long>(info->merge_tokens) * H;
    // a workgroup per row up to one resident round of them (2048 rows of 14 parts
    // 6.6 us, against 7.6 with a team each, and of 24 parts 8.9 against 11.4); above
    // it the rows have few parts (58 thousand of two 57 us, against 19.5)
    const bool wide = rows <= 2048;
    for (long long r = 0; r < rows; r += 1 << 22) {  // a launch holds fewer than 2^32 threads
      const int n = static_cast<int>(std::min<long long>(rows - r, 1 << 22));
      auto merge = [&](auto kernel, int wgs) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(wgs)), dim3(256), 0, stream, a.part,
                           reinterpret_cast<const float2*>(a.part_ml), plan + info->merge_at,
                           reinterpret_cast<const int4*>(plan + info->parts_at),
                           reinterpret_cast<const int2*>(plan + info->pos_at), static_cast<int>(r), n, H, KVH,
                           a.scale_log2, a.out);
      };
      constexpr int kTeams = 1024 / kD;
      if (wide) merge(merge_kernel<BF16, kD, true>, n);
      else merge(merge_kernel<BF16, kD, false>, (n + kTeams - 1) / kTeams);
    }
  };
  if (dtype == SANTA_BF16) {
    if (D == 128) run(std::true_type{}, std::integral_constant<int, 128>{});
    else run(std::true_type{}, std::integral_constant<int, 64>{});
  } else {
    if (D == 128) run(std::false_type{}, std::integral_constant<int, 128>{});
    else run(std::false_type{}, std::integral_constant<int, 64>{});
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "paged_attention launch failed: %s", hipGetErrorString(e));
  return clear_error();
}
