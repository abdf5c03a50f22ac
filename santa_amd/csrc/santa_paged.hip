// santa_paged.hip -- a paged KV cache that sequences share
// (santa_amd/paged.py): page copies and block table edits, RoPE of new tokens
// with their write into pages, and the exact attention over pages, in which
// a prefix that sequences have in common is read once for all of them.  No
// counterpart in the reference, whose caches are contiguous and one per sequence
// (tutorial_code/runtime_common.py:340-397).
#include <algorithm>
#include <climits>
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

// Workgroup (piece of the page, pair, pool).
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

// A thread takes dims d .. d + 7 and d + D/2 .. d + D/2 + 7 of one head of one
// token, the two pieces that rotate-half combines.
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
constexpr int kWaves = 4;
// Above this a maximum in log2 units is subtracted from the scores before they
// are scaled: fma(score, scale, -round(max * scale)) is off by half an ulp of
// the product, a factor common to a row's probabilities that up to here (2^-15)
// leaves the largest of them 1 in either 16-bit type.
constexpr float kExactMax = 512.0f;
constexpr int kWaitVmem = 0x0f70;  // s_waitcnt vmcnt(0) alone

// What invalid rows of a tile are read from.
__device__ u32x4 g_zero_row[16];

template <int D>
struct Geometry {
  static constexpr int kRow = 2 * D;               // bytes
  static constexpr int kLanes = D / 8;             // lanes per row
  static constexpr int kRows = 64 / kLanes;        // rows per load instruction
  static constexpr int kGroups = kTile / kRows;    // load instructions per tile
  static constexpr int kVecs = kTile * kLanes;     // 16-byte pieces per tile
};

struct AttnArgs {
  const uint16_t* q;
  const char *k, *v;
  uint16_t* out;
  float *part, *part_ml;  // sums [records, D]; (maximum, mass) [records]
  const Item* items;
  const int* list;
  Pages pg;
  long long sq_t, sq_h;                  // elements
  long long sk_p, sk_r, sk_h, sv_p, sv_r, sv_h;  // bytes
  int KVH, GH;
  float scale_log2;
};

// What a lane loads of a tile: its piece of the rows n, n + 1, ... from the
// tile's row0 on, one per load instruction.
struct TileLoad {
  const char *k, *v;         // this KV head in the pools
  const int* table;          // the block table row
  int row0, lrow, lslot;
  int begin, end, last;
};

// Issues the loads of tile t into dst; nothing waits for them here.  A row's
// 16-byte pieces are swizzled so that the reads of both tiles are without bank
// conflicts.  Eight tokens from a multiple of eight on lie in one page.
template <int D>
__device__ __forceinline__ void load_tile(const AttnArgs& a, const TileLoad& w, u32x4* __restrict__ dst, int wave, int t,
                                          int page) {
  using G = Geometry<D>;
  constexpr int GPW = G::kGroups / kWaves;
  const int n = w.begin + t * kTile + w.row0;
  page = in_pool(a.pg, page);
  const int in_page = n & ((1 << a.pg.shift) - 1);
  const char* kp = w.k + page * a.sk_p + in_page * a.sk_r;
  const char* vp = w.v + page * a.sv_p + in_page * a.sv_r;
#pragma unroll
  for (int c = 0; c < GPW; ++c) {
    const int g = GPW * wave + c;
    const int pr = G::kRows * g + w.lrow;  // row of the tile in LDS
    const int ks = 16 * (w.lslot ^ (D == 128 ? pr & 15 : (pr >> 1) & 7));
    const int vs = 16 * (w.lslot ^ (D == 128 ? 4 * (pr & 3) : 4 * ((pr >> 1) & 1)));
    const bool in = n + c < w.end;
    const char* zero = reinterpret_cast<const char*>(g_zero_row);
    const char* ka = in ? kp + c * a.sk_r + ks : zero + ks;
    const char* va = in ? vp + c * a.sv_r + vs : zero + vs;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)ka,
                                     (__attribute__((address_space(3))) void*)(dst + 64 * g), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)va,
                                     (__attribute__((address_space(3))) void*)(dst + G::kVecs + 64 * g), 16, 0, 0);
  }
}

// Running softmax of a wave's rows (one per lane of each half): the sum of
// MB x 32 dims, the maximum of the raw scores and the mass of this half's
// tokens.  mc: the maximum in log2 units, or 0 where the scores have it
// subtracted (kExactMax); grows: the maximum, or -inf there, so that every tile's
// scores pass that way.
template <int MB>
struct State {
  f32x16 o[MB];
  float m, l, mc, grows;
};

// One tile: scores S^T = K Q^T of 32 KB tokens x 32 rows, softmax, and
// O^T += V^T P^T.  n0 and lim: the tile's first token and the last one that the
// lane's row attends to.
template <bool BF16, int D, int KB, int MB>
__device__ __forceinline__ void attend_tile(const char* __restrict__ buf, const u32x4 (&qf)[D / 16],
                                            const uint32_t (&ko)[D / 16], const uint32_t (&vo)[MB], int kh, int n0,
                                            int lim, int lim_lo, bool dup, float scale_log2, State<MB>& st) {
  using G = Geometry<D>;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  f32x16 s[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[kb][e] = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      s[kb] = mfma32<BF16>(*reinterpret_cast<const u32x4*>(buf + ko[c] + 32 * G::kRow * kb), qf[c], s[kb]);
  }
  if (n0 + kTile - 1 > lim_lo) {  // tokens that some row does not attend to
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int pr = 32 * (kh + kb) + 8 * (e >> 2) + 4 * half + (e & 3);
        const int n = n0 + G::kGroups * (pr % G::kRows) + pr / G::kRows;
        if (n > lim) s[kb][e] = -__builtin_inff();
      }
  }
  float mx = s[0][0];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
  mx = fmaxf(mx, other_half(mx));
  const float m_new = fmaxf(st.m, mx);
  if (__any(m_new > st.grows)) {
    const float w = __builtin_amdgcn_exp2f((st.m - m_new) * scale_log2);
    st.l *= w;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[mb][e] *= w;
    st.grows = st.m = m_new;
    st.mc = st.m * scale_log2;
    if (__any(fabsf(st.mc) > kExactMax)) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] -= st.m;
      st.mc = 0.0f;
      st.grows = -__builtin_inff();
    }
  }
  u32x4 p[2 * KB];
#pragma unroll
  for (int kc = 0; kc < 2 * KB; ++kc) {
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      e[j] = __builtin_amdgcn_exp2f(fmaf(s[kc >> 1][8 * (kc & 1) + j], scale_log2, -st.mc));
      st.l += e[j];
    }
    p[kc] = pack8<BF16>(e);
    // up to 16 rows leave lanes 16 .. 31 of the wave free: they hold the same
    // rows again, and carry what rounding took from their probabilities
    if (dup) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        e[j] -= lo16_to_f32<BF16>(p[kc][j >> 1]);
        e[j + 1] -= hi16_to_f32<BF16>(p[kc][j >> 1]);
      }
      const u32x4 low = pack8<BF16>(e);
      if (lane & 16) p[kc] = low;
    }
  }
#pragma unroll
  for (int kc = 0; kc < 2 * KB; ++kc)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
      st.o[mb] = mfma32<BF16>(read_tr8<G::kRow>(buf + vo[mb] + 16 * G::kRow * kc), p[kc], st.o[mb]);
}

// The next tile's loads and this tile's work.  The buffers are told apart by
// their restrict qualifiers: without them the compiler makes the first read of
// this tile wait for the loads of the next.
template <bool BF16, int D, int KB, int MB>
__device__ __forceinline__ void step(const char* __restrict__ cur, u32x4* __restrict__ next, bool more,
                                     const AttnArgs& a, const TileLoad& w, int wave, int t, int& page, bool busy,
                                     const u32x4 (&qf)[D / 16], const uint32_t (&ko)[D / 16], const uint32_t (&vo)[MB],
                                     int kh, int lim, int lim_lo, bool dup, State<MB>& st) {
  if (more) {
    load_tile<D>(a, w, next, wave, t + 1, page);
    page = w.table[min(w.begin + (t + 2) * kTile + w.row0, w.last) >> a.pg.shift];
  }
  if (busy)
    attend_tile<BF16, D, KB, MB>(cur, qf, ko, vo, kh, w.begin + t * kTile, lim, lim_lo, dup, a.scale_log2, st);
}

// The passes of one wave over its item's tiles, and its output.  SPLIT: the four
// waves hold the same rows (up to 32) and take two halves of each tile's
// tokens times two halves of the dims; else each has its own 32 rows.
template <bool BF16, int D, bool SPLIT>
__device__ __forceinline__ void attend(const AttnArgs& a, const Item& it, int kv,
                                       u32x4 (*s_kv)[2 * Geometry<D>::kVecs]) {
  using G = Geometry<D>;
  constexpr int KB = SPLIT ? 1 : 2;
  constexpr int MB = SPLIT ? D / 64 : D / 32;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, ql = lane & 31;
  const int kh = SPLIT ? wave & 1 : 0, dh = SPLIT ? wave >> 1 : 0;
  const bool dup = SPLIT && it.rows <= 16;

  // this lane's row
  const int r = dup ? ql & 15 : SPLIT ? ql : 32 * wave + ql;
  const bool active = r < it.rows;
  const int rc = min(r, it.rows - 1);
  const int i = rc / a.GH, h = kv * a.GH + (rc - i * a.GH);
  const int tok = it.flags & kFromList ? a.list[it.tok0 + i] : it.tok0 + i;
  const int pos = it.pos0 + i;
  const int lim = min(it.end - 1, pos);  // last position this row attends to here
  const int lim_lo = __builtin_amdgcn_readlane(lim, 0), lim_hi = __builtin_amdgcn_readlane(lim, 31);
  const bool any = SPLIT || 32 * wave < it.rows;

  TileLoad w;
  w.k = a.k + kv * a.sk_h;
  w.v = a.v + kv * a.sv_h;
  w.table = a.pg.table + it.row * a.pg.stride;
  w.lrow = lane / G::kLanes;
  w.lslot = lane % G::kLanes;
  w.row0 = G::kGroups * w.lrow + G::kGroups / kWaves * wave;
  w.begin = it.begin;
  w.end = it.end;
  w.last = static_cast<int>(min(static_cast<long long>(it.end), a.pg.stride << a.pg.shift)) - 1;
  const int nt = (it.end - it.begin + kTile - 1) / kTile;
  int page = 0;
  if (nt > 0) {
    page = w.table[min(w.begin + w.row0, w.last) >> a.pg.shift];
    load_tile<D>(a, w, s_kv[0], wave, 0, page);
    page = w.table[min(w.begin + kTile + w.row0, w.last) >> a.pg.shift];
  }

  // Q fragments: dims 16c + 8 half .. + 7 of this lane's row
  u32x4 qf[D / 16];
  {
    const uint16_t* qr = a.q + tok * a.sq_t + h * a.sq_h + 8 * half;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = *reinterpret_cast<const u32x4*>(qr + 16 * c);
  }
  // LDS byte offsets of this lane's fragments inside a buffer
  uint32_t ko[D / 16], vo[MB];
#pragma unroll
  for (int c = 0; c < D / 16; ++c)
    ko[c] = (ql + 32 * kh) * G::kRow + 16 * ((2 * c + half) ^ (D == 128 ? ql & 15 : (ql >> 1) & 7));
  const int r3 = (lane & 15) >> 2;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int piece = 4 * (mb + MB * dh) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    vo[mb] = 16 * G::kVecs + (4 * half + r3 + 32 * kh) * G::kRow +
             16 * (piece ^ (D == 128 ? 4 * r3 : 4 * (r3 >> 1))) + 8 * (lane & 1);
  }

  State<MB> st;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int e = 0; e < 16; ++e) st.o[mb][e] = 0.0f;
  st.m = kLowest;
  st.l = st.mc = 0.0f;
  st.grows = -__builtin_inff();
  for (int t = 0; t < nt; ++t) {
    __builtin_amdgcn_s_waitcnt(kWaitVmem);
    __syncthreads();  // tile t is in LDS, and no wave reads the other buffer any more
    step<BF16, D, KB, MB>(reinterpret_cast<const char*>(s_kv[t & 1]), s_kv[(t + 1) & 1], t + 1 < nt, a, w, wave, t,
                          page, any && w.begin + t * kTile <= lim_hi, qf, ko, vo, kh, lim, lim_lo, dup, st);
  }
  float m = st.m, l = st.l + other_half(st.l);
  f32x16(&o)[MB] = st.o;
  if constexpr (SPLIT) {
    if (dup) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[mb][e] += fxor<16>(o[mb][e], lane);
    }
    // the two halves of the tokens
    float* const x = reinterpret_cast<float*>(s_kv) + dh * (16 * MB + 2) * 64 + lane;
    __syncthreads();  // no wave reads a tile any more
    if (kh == 1) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[(16 * mb + e) * 64] = o[mb][e];
      x[16 * MB * 64] = m;
      x[(16 * MB + 1) * 64] = l;
    }
    __syncthreads();
    if (kh == 1) return;
    const float m2 = x[16 * MB * 64], top = fmaxf(m, m2);
    const float w1 = __builtin_amdgcn_exp2f((m - top) * a.scale_log2), w2 = __builtin_amdgcn_exp2f((m2 - top) * a.scale_log2);
    m = top;
    l = l * w1 + x[(16 * MB + 1) * 64] * w2;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[mb][e] = o[mb][e] * w1 + x[(16 * mb + e) * 64] * w2;
    if (dup && (ql & 16)) return;
  }
  if (!active) return;
  if (it.flags & kDirect) {
    const float inv = pos < 0 ? 0.0f : 1.0f / l;
    uint16_t* orow = a.out + (static_cast<size_t>(tok) * (a.KVH * a.GH) + h) * D + 32 * MB * dh;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        uint2 w;
        w.x = f32_to_h16<BF16>(o[mb][e] * inv) | (static_cast<uint32_t>(f32_to_h16<BF16>(o[mb][e + 1] * inv)) << 16);
        w.y = f32_to_h16<BF16>(o[mb][e + 2] * inv) | (static_cast<uint32_t>(f32_to_h16<BF16>(o[mb][e + 3] * inv)) << 16);
        *reinterpret_cast<uint2*>(orow + 32 * mb + 2 * e + 4 * half) = w;
      }
    return;
  }
  const size_t rec = static_cast<size_t>(it.base) + static_cast<size_t>(kv) * it.rows + r;
  float* prow = a.part + rec * D + 32 * MB * dh;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<float4*>(prow + 32 * mb + 2 * e + 4 * half) =
          make_float4(o[mb][e], o[mb][e + 1], o[mb][e + 2], o[mb][e + 3]);
  if (dh == 0 && half == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * rec) = make_float2(m, l);
}

template <bool BF16, int D>
__global__ __launch_bounds__(256, 2) void paged_attention_kernel(AttnArgs a, int first_item) {
  __shared__ u32x4 s_kv[2][2 * Geometry<D>::kVecs];  // per buffer: the K tile, the V tile
  const int kv = blockIdx.x % a.KVH;
  const Item it = a.items[first_item + blockIdx.x / a.KVH];
  if (it.rows <= 0) return;
  if (it.rows <= 32)
    attend<BF16, D, true>(a, it, kv, s_kv);
  else
    attend<BF16, D, false>(a, it, kv, s_kv);
}

// Joins the parts of one (token, head): 256 threads, the parts spread over
// them for the maximum and the weights, then 256 / (D / 2) groups of D / 2
// threads, two dims each, over the parts in turn.
constexpr int kMergeThreads = 256;

template <bool BF16, int D>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const float* __restrict__ part,
                                                              const float2* __restrict__ part_ml,
                                                              const int* __restrict__ tokens,
                                                              const int4* __restrict__ parts,
                                                              const int2* __restrict__ pos, int first_token, int H,
                                                              int KVH, float scale_log2, uint16_t* __restrict__ out) {
  constexpr int kThreads = D / 2, kTeams = kMergeThreads / kThreads;
  __shared__ float s_w[kMergeThreads];
  __shared__ float s_red[2][4];
  __shared__ float2 s_o[kTeams][kThreads];
  const int tok = tokens[first_token + blockIdx.x / H];
  if (tok < 0) return;
  const int h = blockIdx.x % H, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int kv = h / (H / KVH), g = h % (H / KVH);
  const int4 pa = parts[2 * tok], pb = parts[2 * tok + 1];  // base, rows, local, splits
  const int n = pb.w > 0 ? pa.w + pb.w : 0;
  if (n == 0) return;  // written by its item
  auto record = [&](int j) {
    const int4 p = j < pa.w ? pa : pb;
    return static_cast<size_t>(p.x) + (static_cast<size_t>(j < pa.w ? j : j - pa.w) * KVH + kv) * p.y + p.z + g;
  };
  float mx = kLowest;
  for (int j = tid; j < n; j += kMergeThreads) mx = fmaxf(mx, part_ml[record(j)].x);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
  if (lane == 0) s_red[0][wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  const int team = tid / kThreads, d2 = tid % kThreads;
  float z = 0.0f;
  float2 acc = make_float2(0.0f, 0.0f);
  for (int j0 = 0; j0 < n; j0 += kMergeThreads) {
    __syncthreads();  // the weights of the parts before are used up
    if (j0 + tid < n) {
      const float2 ml = part_ml[record(j0 + tid)];
      const float w = __builtin_amdgcn_exp2f((ml.x - mx) * scale_log2);
      s_w[tid] = w;
      z = fmaf(w, ml.y, z);
    }
    __syncthreads();
    const int k = min(kMergeThreads, n - j0);
#pragma unroll 8
    for (int j = team; j < k; j += kTeams) {
      const float2 v = *reinterpret_cast<const float2*>(part + record(j0 + j) * D + 2 * d2);
      acc.x = fmaf(s_w[j], v.x, acc.x);
      acc.y = fmaf(s_w[j], v.y, acc.y);
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) z += __shfl_xor(z, d, 64);
  if (lane == 0) s_red[1][wave] = z;
  s_o[team][d2] = acc;
  __syncthreads();
  if (team > 0) return;
  z = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
#pragma unroll
  for (int k = 1; k < kTeams; ++k) acc.x += s_o[k][d2].x, acc.y += s_o[k][d2].y;
  const float inv = pos[tok].x < 0 ? 0.0f : 1.0f / z;
  const uint32_t w = f32_to_h16<BF16>(acc.x * inv) | (static_cast<uint32_t>(f32_to_h16<BF16>(acc.y * inv)) << 16);
  *reinterpret_cast<uint32_t*>(out + (static_cast<size_t>(tok) * H + h) * D + 2 * d2) = w;
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
  if (D <= 0 || D % 16 != 0) return set_error(SANTA_ERR_UNSUPPORTED, "rope_append: D must be a multiple of 16. Got D=%d", D);
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
  a.sk_p = 2 * strides[2], a.sk_r = 2 * strides[3], a.sk_h = 2 * strides[4];
  a.sv_p = 2 * strides[5], a.sv_r = 2 * strides[6], a.sv_h = 2 * strides[7];
  a.KVH = KVH;
  a.GH = H / KVH;
  a.scale_log2 = 1.44269504088896340736f * scale;
  auto run = [&](auto attention, auto merge) {
    // a launch holds fewer than 2^32 threads
    const int step = (1 << 23) / std::max(H, KVH);
    for (int i = 0; i < info->items; i += step)
      hipLaunchKernelGGL(attention, dim3(static_cast<unsigned>(std::min(step, info->items - i) * KVH)), dim3(256), 0,
                         stream, a, i);
    for (int t = 0; t < info->merge_tokens; t += step)
      hipLaunchKernelGGL(merge, dim3(static_cast<unsigned>(std::min(step, info->merge_tokens - t) * H)),
                         dim3(kMergeThreads), 0, stream, a.part, reinterpret_cast<const float2*>(a.part_ml),
                         plan + info->merge_at, reinterpret_cast<const int4*>(plan + info->parts_at),
                         reinterpret_cast<const int2*>(plan + info->pos_at), t, H, KVH, a.scale_log2, a.out);
  };
  if (dtype == SANTA_BF16) {
    if (D == 128) run(paged_attention_kernel<true, 128>, merge_kernel<true, 128>);
    else run(paged_attention_kernel<true, 64>, merge_kernel<true, 64>);
  } else {
    if (D == 128) run(paged_attention_kernel<false, 128>, merge_kernel<false, 128>);
    else run(paged_attention_kernel<false, 64>, merge_kernel<false, 64>);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "paged_attention launch failed: %s", hipGetErrorString(e));
  return clear_error();
}
