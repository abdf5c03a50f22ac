// santa_rotary.hip -- rotary positions for shared paged caches
// (santa_amd/paged.py): tables of cos and sin in either layout, and the norms of q
// and k heads with their rotation, wholly or in part, and the write into pages.
// No counterpart in the reference, whose models rotate and norm in torch
// (tutorial_code/runtime_common.py:501-571).
#include <algorithm>
#include <cmath>

#include "santa_amd.h"
#include "santa_attn_device.h"
#include "santa_internal.h"
#include "santa_paged.h"

namespace santa {
namespace paged {

using attn::pack8;
using attn::u32x4;

// -------------------------------------------------------------------- tables
constexpr int kMostPairs = 256;

struct Frequencies {
  double turns[kMostPairs];  // per position
  float magnitude;
};

template <class T>
__device__ __forceinline__ T rounded(float x);
template <>
__device__ __forceinline__ float rounded<float>(float x) { return x; }
template <>
__device__ __forceinline__ __bf16 rounded<__bf16>(float x) { return static_cast<__bf16>(x); }
template <>
__device__ __forceinline__ _Float16 rounded<_Float16>(float x) { return static_cast<_Float16>(x); }

// cos and sin of pos x f for every (position, pair), kMore pairs to a thread (4 where
// their number allows it: stores of up to 16 bytes).  The angle is taken in turns,
// in float64, of which the whole ones leave nothing.  What remains, r, is a float32 h
// and what that leaves, l, of at most 2^-26 turns: with e = 2 pi l, cos(2 pi r) = cos(2
// pi h) - e sin(2 pi h), sin(2 pi r) = sin(2 pi h) + e cos(2 pi h), up to e^2 / 2 < 2^-47.
// Bound by sincospif's vector work beside the stores: 27 thousand positions of 64 pairs
// in float32, 28 MB, 9.9 us (9.8 without l, 10.3 with a pair a thread); 64 positions are
// the launch (2.6 us).
template <class T, int kMore, bool kInterleaved>
__global__ __launch_bounds__(256) void rope_tables_kernel(const void* __restrict__ positions, int wide,
                                                          long long stride, Frequencies f, int pairs,
                                                          T* __restrict__ cos_, T* __restrict__ sin_, uint32_t n) {
  typedef T Vec __attribute__((ext_vector_type(kMore)));
  const uint32_t per = static_cast<uint32_t>(pairs / kMore), rows = 256u / per;  // positions of a workgroup at once
  if (threadIdx.x >= per * rows) return;
  const int p = kMore * static_cast<int>(threadIdx.x % per);
  double f_[kMore];
#pragma unroll
  for (int k = 0; k < kMore; ++k) f_[k] = f.turns[p + k];
  for (uint32_t row = blockIdx.x * rows + threadIdx.x / per; row < n; row += gridDim.x * rows) {
    const long long at = static_cast<long long>(row) * stride;
    const double pos = wide ? static_cast<double>(static_cast<const long long*>(positions)[at])
                            : static_cast<double>(static_cast<const int*>(positions)[at]);
    T c[kMore], s[kMore];
#pragma unroll
    for (int k = 0; k < kMore; ++k) {
      const double turns = pos * f_[k], r = turns - rint(turns);
      const float h = static_cast<float>(r), e = 6.28318531f * static_cast<float>(r - h);
      float sh, ch;
      sincospif(2.0f * h, &sh, &ch);
      c[k] = rounded<T>(fmaf(-e, sh, ch) * f.magnitude), s[k] = rounded<T>(fmaf(e, ch, sh) * f.magnitude);
    }
    const size_t base = static_cast<size_t>(row) * (2 * pairs);
    // the kMore values of a pair's first dims, then of the second ones; or both in turn
    Vec c0, c1, s0, s1;
#pragma unroll
    for (int k = 0; k < kMore; ++k) {
      const int a = kInterleaved ? k / 2 : k, b = kInterleaved ? (kMore + k) / 2 : k;
      c0[k] = c[a], s0[k] = s[a], c1[k] = c[b], s1[k] = s[b];
    }
    const size_t first = base + (kInterleaved ? 2 * p : p), second = kInterleaved ? first + kMore : first + pairs;
    *reinterpret_cast<Vec*>(cos_ + first) = c0;
    *reinterpret_cast<Vec*>(cos_ + second) = c1;
    *reinterpret_cast<Vec*>(sin_ + first) = s0;
    *reinterpret_cast<Vec*>(sin_ + second) = s1;
  }
}

// --------------------------------------------------------------------- heads
enum class Layout {
  kHalf,   // dims d and d + R/2, R a multiple of 16
  kFours,  // the same, R a multiple of 8
  kPairs,  // dims 2d and 2d + 1, R a multiple of 8
  kAny     // either, R even
};

struct HeadArgs {
  const uint16_t *qkv, *cos_, *sin_;
  const uint16_t *q_norm, *k_norm;  // NULL: none
  long long q_norm_row, k_norm_row; // elements from head to head
  uint16_t *q_out, *k_pages, *v_pages;
  int H, KVH, D, R, interleaved;
  float eps, inv_d;
  PoolStrides sk, sv;
  Pages pg;
  const int2* pos;
  uint32_t total;  // heads of all tokens
};

template <bool BF16>
__device__ __forceinline__ float half_of(u32x4 v, int k) {
  return k & 1 ? hi16_to_f32<BF16>(v[k >> 1]) : lo16_to_f32<BF16>(v[k >> 1]);
}

// y = x / sqrt(mean(x^2) + eps) * w over a head, then a rotation of its first R
// dims; float32, rounded once.  A team of kTeam lanes has a head, a lane two pieces of
// 8 dims: with rotate-half those that the rotation combines.  Bound by HBM: 14 thousand
// tokens of 32 + 2 x 8 heads of 128, normed, 351 MB, in 64 us over whole heads in halves
// (5.6 TB/s; 61 without norms) and 67 over half of each in pairs; halves that are no
// whole pieces 85 to 93 (163 to 261 where they were read value by value).  64 drafts are
// latency (3.9 us).
template <bool BF16, Layout kLayout, int kTeam>
__global__ __launch_bounds__(256) void heads_append_kernel(HeadArgs a) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const int lane = static_cast<int>(i % kTeam);
  const uint32_t head = i / kTeam, heads = static_cast<uint32_t>(a.H + 2 * a.KVH);
  const bool on = head < a.total && 16 * lane < a.D;  // other lanes take part in the exchange
  const uint32_t t = on ? head / heads : 0;
  const int h = on ? static_cast<int>(head % heads) : 0;
  const int turned = a.R / 16;  // lanes with pieces to rotate
  int d0 = 16 * lane, d1 = d0 + 8;
  if (kLayout == Layout::kHalf && lane < turned) d0 = 8 * lane, d1 = d0 + a.R / 2;
  const uint16_t* src = a.qkv + (static_cast<size_t>(t) * heads + h) * a.D;
  u32x4 x0{}, x1{};
  if (on) {
    x0 = *reinterpret_cast<const u32x4*>(src + d0);
    x1 = *reinterpret_cast<const u32x4*>(src + d1);
  }
  const bool is_v = h >= a.H + a.KVH, is_q = h < a.H;
  const uint16_t* w = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
  if (w) w += is_q ? h * a.q_norm_row : (h - a.H) * a.k_norm_row;
  float y0[8], y1[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y0[k] = half_of<BF16>(x0, k), y1[k] = half_of<BF16>(x1, k);
  float scale = 1.0f;
  if (a.q_norm || a.k_norm) {
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fmaf(y0[k], y0[k], fmaf(y1[k], y1[k], ss));
#pragma unroll
    for (int m = kTeam / 2; m > 0; m >>= 1) ss += __shfl_xor(ss, m, 64);
    scale = 1.0f / sqrtf(fmaf(ss, a.inv_d, a.eps));
  }
  if (!on) return;
  uint16_t* dst;
  if (is_q) {
    dst = a.q_out + (static_cast<size_t>(t) * a.H + h) * a.D;
  } else {
    const int2 at = a.pos[t];
    if (at.x < 0 || (at.x >> a.pg.shift) >= a.pg.stride) return;
    const int page_id = a.pg.table[at.y * a.pg.stride + (at.x >> a.pg.shift)];
    const long long page = min(max(page_id, 0), a.pg.num_pages - 1), row = at.x & ((1 << a.pg.shift) - 1);
    dst = is_v ? a.v_pages + page * a.sv.page + row * a.sv.row + (h - a.H - a.KVH) * a.sv.head
               : a.k_pages + page * a.sk.page + row * a.sk.row + (h - a.H) * a.sk.head;
  }
  if (!is_v) {
    if (w) {
      const u32x4 w0 = *reinterpret_cast<const u32x4*>(w + d0), w1 = *reinterpret_cast<const u32x4*>(w + d1);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        y0[k] *= scale * half_of<BF16>(w0, k);
        y1[k] *= scale * half_of<BF16>(w1, k);
      }
    }
    const uint16_t *cp = a.cos_ + static_cast<size_t>(t) * a.R, *sp = a.sin_ + static_cast<size_t>(t) * a.R;
    if constexpr (kLayout == Layout::kHalf) {
      if (lane < turned) {
        const u32x4 c0 = *reinterpret_cast<const u32x4*>(cp + d0), c1 = *reinterpret_cast<const u32x4*>(cp + d1);
        const u32x4 s0 = *reinterpret_cast<const u32x4*>(sp + d0), s1 = *reinterpret_cast<const u32x4*>(sp + d1);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float u = y0[k], v = y1[k];
          y0[k] = fmaf(u, half_of<BF16>(c0, k), -(v * half_of<BF16>(s0, k)));
          y1[k] = fmaf(v, half_of<BF16>(c1, k), u * half_of<BF16>(s1, k));
        }
      }
    } else if constexpr (kLayout == Layout::kFours) {
      // four dims lie in one half, and those that belong to them in the other: read
      // again, 8 bytes at a time
      auto turn = [&](float(&y)[8], int d) {
        if (d >= a.R) return;
        const u32x4 c = *reinterpret_cast<const u32x4*>(cp + d), s = *reinterpret_cast<const u32x4*>(sp + d);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool first = d + 4 * j < a.R / 2;
          const int o = first ? d + 4 * j + a.R / 2 : d + 4 * j - a.R / 2;
          const uint2 x = *reinterpret_cast<const uint2*>(src + o);
          float other[4] = {lo16_to_f32<BF16>(x.x), hi16_to_f32<BF16>(x.x), lo16_to_f32<BF16>(x.y), hi16_to_f32<BF16>(x.y)};
          if (w) {
            const uint2 v = *reinterpret_cast<const uint2*>(w + o);
            other[0] *= scale * lo16_to_f32<BF16>(v.x), other[1] *= scale * hi16_to_f32<BF16>(v.x);
            other[2] *= scale * lo16_to_f32<BF16>(v.y), other[3] *= scale * hi16_to_f32<BF16>(v.y);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float o = other[k] * half_of<BF16>(s, 4 * j + k);
            y[4 * j + k] = fmaf(y[4 * j + k], half_of<BF16>(c, 4 * j + k), first ? -o : o);
          }
        }
      };
      turn(y0, d0);
      turn(y1, d1);
    } else if constexpr (kLayout == Layout::kPairs) {
      auto turn = [&](float(&y)[8], int d) {
        if (d >= a.R) return;
        const u32x4 c = *reinterpret_cast<const u32x4*>(cp + d), s = *reinterpret_cast<const u32x4*>(sp + d);
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          const float u = y[k], v = y[k + 1];
          y[k] = fmaf(u, half_of<BF16>(c, k), -(v * half_of<BF16>(s, k)));
          y[k + 1] = fmaf(v, half_of<BF16>(c, k + 1), u * half_of<BF16>(s, k + 1));
        }
      };
      turn(y0, d0);
      turn(y1, d1);
    } else {
      auto turn = [&](float(&y)[8], int d) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int e = d + k;
          if (e >= a.R) return;
          const bool first = a.interleaved ? !(e & 1) : e < a.R / 2;
          const int o = a.interleaved ? e ^ 1 : first ? e + a.R / 2 : e - a.R / 2;
          float other = h16_to_f32<BF16>(src[o]);
          if (w) other *= scale * h16_to_f32<BF16>(w[o]);
          const float c = h16_to_f32<BF16>(cp[e]), s = h16_to_f32<BF16>(sp[e]);
          y[k] = fmaf(y[k], c, first ? -(other * s) : other * s);
        }
      };
      turn(y0, d0);
      turn(y1, d1);
    }
    x0 = pack8<BF16>(y0);
    x1 = pack8<BF16>(y1);
  }
  *reinterpret_cast<u32x4*>(dst + d0) = x0;
  *reinterpret_cast<u32x4*>(dst + d1) = x1;
}

template <bool BF16, Layout kLayout>
void launch_heads(const HeadArgs& a, hipStream_t stream) {
  auto launch = [&](auto kernel, int team) {
    const unsigned grid = static_cast<unsigned>((static_cast<unsigned long long>(a.total) * team + 255) / 256);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, stream, a);
  };
  if (a.D <= 32) launch(heads_append_kernel<BF16, kLayout, 2>, 2);
  else if (a.D <= 64) launch(heads_append_kernel<BF16, kLayout, 4>, 4);
  else if (a.D <= 128) launch(heads_append_kernel<BF16, kLayout, 8>, 8);
  else if (a.D <= 256) launch(heads_append_kernel<BF16, kLayout, 16>, 16);
  else launch(heads_append_kernel<BF16, kLayout, 32>, 32);
}

}  // namespace paged
}  // namespace santa

using namespace santa;

extern "C" int santa_rope_tables(const void* positions, int wide, long long stride, long long n, const double* turns,
                                 int pairs, float magnitude, int interleaved, int dtype, void* cos_, void* sin_,
                                 hipStream_t stream) {
  if (n < 0 || !turns || pairs <= 0 || (n > 0 && (!positions || !cos_ || !sin_)))
    return set_error(SANTA_ERR_INVALID, "bad rope_tables arguments");
  if (dtype != SANTA_BF16 && dtype != SANTA_F16 && dtype != SANTA_F32)
    return set_error(SANTA_ERR_UNSUPPORTED, "rope_tables: the tables are bf16, f16 or float32");
  if (pairs > paged::kMostPairs)
    return set_error(SANTA_ERR_UNSUPPORTED, "rope_tables: up to %d dims. Got %d", 2 * paged::kMostPairs, 2 * pairs);
  if (n > 0x7fffff00LL / pairs) return set_error(SANTA_ERR_INVALID, "too many positions");
  if (n == 0) return clear_error();
  paged::Frequencies f;
  for (int i = 0; i < pairs; ++i) f.turns[i] = turns[i];
  f.magnitude = magnitude;
  if ((reinterpret_cast<uintptr_t>(cos_) | reinterpret_cast<uintptr_t>(sin_)) % 16 != 0)
    return set_error(SANTA_ERR_INVALID, "rope_tables: the tables must be 16-byte aligned");
  auto run = [&](auto* c, auto* s) {
    using T = std::remove_reference_t<decltype(*c)>;
    auto launch = [&](auto kernel, int more) {
      const long long rows = 256 / (pairs / more), wgs = (n + rows - 1) / rows;
      // a few rounds of positions to a workgroup, for one look at the frequencies
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min(wgs, 1024LL))), dim3(256), 0, stream, positions,
                         wide, stride, f, pairs, c, s, static_cast<uint32_t>(n));
    };
    if (pairs % 4 == 0)
      interleaved ? launch(paged::rope_tables_kernel<T, 4, true>, 4) : launch(paged::rope_tables_kernel<T, 4, false>, 4);
    else
      interleaved ? launch(paged::rope_tables_kernel<T, 1, true>, 1) : launch(paged::rope_tables_kernel<T, 1, false>, 1);
  };
  if (dtype == SANTA_F32) run(static_cast<float*>(cos_), static_cast<float*>(sin_));
  else if (dtype == SANTA_BF16) run(static_cast<__bf16*>(cos_), static_cast<__bf16*>(sin_));
  else run(static_cast<_Float16*>(cos_), static_cast<_Float16*>(sin_));
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "rope_tables launch failed: %s", hipGetErrorString(e));
  return clear_error();
}

extern "C" int santa_paged_heads_append(const void* qkv, const void* cos_, const void* sin_, int R, int interleaved,
                                        const void* q_norm, int q_norm_heads, const void* k_norm, int k_norm_heads,
                                        float eps, void* q_out, void* k_pages, void* v_pages, int dtype, int D,
                                        int num_pages, int page_size, const long long* strides, const int* table,
                                        long long table_stride, int table_rows, const santa_paged_plan_info* info,
                                        const int* plan, hipStream_t stream) {
  using namespace paged;
  HeadArgs a{};
  const int rc = check_paged(qkv, k_pages, v_pages, q_out, dtype, num_pages, page_size, strides, 6, table,
                             table_stride, table_rows, info, plan, "heads_append", &a.pg);
  if (rc != SANTA_OK) return rc;
  for (const void* p : {cos_, sin_, q_norm, k_norm})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0)
      return set_error(SANTA_ERR_INVALID, "heads_append: cos, sin and norms must be 16-byte aligned");
  if (!cos_ || !sin_) return set_error(SANTA_ERR_INVALID, "bad heads_append arguments");
  if (D <= 0 || D % 16 != 0 || D > 512)
    return set_error(SANTA_ERR_UNSUPPORTED, "heads_append: D must be a multiple of 16 up to 512. Got D=%d", D);
  if (R <= 0 || R > D || R % 2 != 0)
    return set_error(SANTA_ERR_INVALID, "heads_append: an even number of dims up to D=%d is rotated. Got %d", D, R);
  if ((q_norm && q_norm_heads != 1 && q_norm_heads != info->heads) ||
      (k_norm && k_norm_heads != 1 && k_norm_heads != info->kv_heads))
    return set_error(SANTA_ERR_INVALID, "heads_append: norms have one row, or one per head");
  if (!(eps >= 0.0f)) return set_error(SANTA_ERR_INVALID, "heads_append: eps must be at least 0");
  const long long heads = static_cast<long long>(info->tokens) * (info->heads + 2LL * info->kv_heads);
  if (heads * (D <= 256 ? 16 : 32) >= 0x7fffff00LL) return set_error(SANTA_ERR_INVALID, "too many new tokens");
  if (heads == 0) return clear_error();
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.cos_ = static_cast<const uint16_t*>(cos_);
  a.sin_ = static_cast<const uint16_t*>(sin_);
  a.q_norm = static_cast<const uint16_t*>(q_norm);
  a.k_norm = static_cast<const uint16_t*>(k_norm);
  a.q_norm_row = q_norm_heads > 1 ? D : 0;
  a.k_norm_row = k_norm_heads > 1 ? D : 0;
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_pages = static_cast<uint16_t*>(k_pages);
  a.v_pages = static_cast<uint16_t*>(v_pages);
  a.H = info->heads, a.KVH = info->kv_heads, a.D = D, a.R = R, a.interleaved = interleaved;
  a.eps = eps;
  a.inv_d = 1.0f / static_cast<float>(D);
  a.sk = PoolStrides{strides[0], strides[1], strides[2]};
  a.sv = PoolStrides{strides[3], strides[4], strides[5]};
  a.pos = reinterpret_cast<const int2*>(plan + info->pos_at);
  a.total = static_cast<uint32_t>(heads);
  auto run = [&](auto bf) {
    constexpr bool BF16 = decltype(bf)::value;
    if (R % 8 != 0) launch_heads<BF16, Layout::kAny>(a, stream);
    else if (interleaved) launch_heads<BF16, Layout::kPairs>(a, stream);
    else if (R % 16 != 0) launch_heads<BF16, Layout::kFours>(a, stream);
    else launch_heads<BF16, Layout::kHalf>(a, stream);
  };
  if (dtype == SANTA_BF16) run(std::true_type{});
  else run(std::false_type{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "heads_append launch failed: %s", hipGetErrorString(e));
  return clear_error();
}
