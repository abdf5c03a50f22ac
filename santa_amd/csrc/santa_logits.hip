// santa_logits.hip -- rules on a model's logits before a token is chosen
// (santa_amd/logits.py): penalties for tokens that a sequence holds, biases and
// grammar masks, for single tokens and for the nodes of drafted trees.  No
// counterpart in the reference, which takes the logits' argmax
// (tutorial_code/runtime_common.py:574-675).
#include <algorithm>
#include <cstdint>

#include "santa_amd.h"
#include "santa_device.h"
#include "santa_internal.h"
#include "santa_paged.h"

namespace santa {
namespace logits {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512;
constexpr int kLeastSlice = 4 * kThreads;
constexpr int kMostSlice = 7 * kLeastSlice;  // 56 KiB of LDS: two workgroups per compute unit

// What a slice's word says of a token.
constexpr uint32_t kCount = 0xfffffu;       // how often it is in the answer
constexpr uint32_t kInPrompt = 0x100000u;   // whether it is in the prompt
constexpr int kBiasShift = 21;              // above: its bias's number, and one
constexpr int kMostBiases = 2046;
constexpr int kMostTokens = 0xfffff;

struct Args {
  const void* x;
  long long stride;
  int V, N, rows, slice, slices;  // rows: of a workgroup
  const void* tokens;
  int wide;
  long long tokens_stride;
  const int* prompts;
  const float *repetition, *frequency, *presence;
  float repetition_all, frequency_all, presence_all;
  const int* bias_ids;
  const float* bias;
  int biases;
  long long bias_stride;
  const uint32_t* allowed;
  long long allowed_stride;
  const int2* pos;   // NULL: no plan; row n has nothing seen and is sequence n
  const int* tree;   // records of tree_ints ints
  int tree_ints;
  float* out;
  unsigned long long* best;  // [N, slices]
};

// Larger for larger values, NaN above all, -0 as 0; among equal ones for smaller
// indices.
__device__ __forceinline__ unsigned long long order_key(float v, int index) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t up = v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
  return static_cast<unsigned long long>(up) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

__device__ __forceinline__ unsigned long long most(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

__device__ __forceinline__ unsigned long long wave_most(unsigned long long v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v = most(v, __shfl_xor(v, m, 64));
  return v;
}

struct Rules {
  float repetition, frequency, presence;
  const float* bias;
};

__device__ __forceinline__ float apply(float x, uint32_t word, const Rules& r) {
  if (word & (kCount | kInPrompt)) x = x > 0.0f ? x / r.repetition : x * r.repetition;
  const uint32_t count = word & kCount;
  x = x - r.frequency * static_cast<float>(count);
  if (count) x = x - r.presence;
  if (word >> kBiasShift) x = x + r.bias[(word >> kBiasShift) - 1];
  return x;
}

template <int kType, int kVec>
__device__ __forceinline__ void load(const void* x, long long at, float (&v)[kVec]) {
  if constexpr (kType == SANTA_F32) {
    const float* p = static_cast<const float*>(x) + at;
    if constexpr (kVec == 4) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = w[k];
    } else {
      v[0] = *p;
    }
  } else {
    constexpr bool BF16 = kType == SANTA_BF16;
    const uint16_t* p = static_cast<const uint16_t*>(x) + at;
    if constexpr (kVec == 4) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p);
      v[0] = lo16_to_f32<BF16>(w[0]), v[1] = hi16_to_f32<BF16>(w[0]);
      v[2] = lo16_to_f32<BF16>(w[1]), v[3] = hi16_to_f32<BF16>(w[1]);
    } else {
      v[0] = h16_to_f32<BF16>(*p);
    }
  }
}

// Workgroup (slice of the vocabulary, rows): counts what the row has seen of its
// slice in LDS, with integers, whose order does not matter, then passes over the
// logits once.  Rows of one sequence follow one another (a plan's tokens): the next
// one adds the tokens that it sees beyond the row before, and a drafted token's path
// is added for its row alone.
template <int kType, int kVec, bool kGreedy>
__global__ __launch_bounds__(kThreads) void adjust_kernel(Args a) {
  extern __shared__ uint32_t words[];
  __shared__ unsigned long long s_best[kThreads / 64];
  const int tid = static_cast<int>(threadIdx.x);
  const int lo = static_cast<int>(blockIdx.x) * a.slice, n = min(a.slice, a.V - lo);
  const int first = static_cast<int>(blockIdx.y) * a.rows, end = min(first + a.rows, a.N);
  int held = -1, upto = 0;  // the words are those of this sequence's first tokens
  auto token = [&](const void* row, int at) {
    return a.wide ? static_cast<const long long*>(row)[at] : static_cast<long long>(static_cast<const int*>(row)[at]);
  };
  for (int r = first; r < end; ++r) {
    int seq = r, context = 0;
    const int* record = nullptr;
    if (a.pos) {
      const int2 at = a.pos[r];
      seq = at.y;
      context = at.x + 1;
      if (a.tree) record = a.tree + static_cast<long long>(r) * a.tree_ints, context = record[0];
    }
    if (!a.tokens) context = 0, record = nullptr;
    const void* row = static_cast<const char*>(a.tokens) + seq * a.tokens_stride * (a.wide ? 8 : 4);
    const int prompt = a.prompts ? a.prompts[seq] : 0;
    if (seq != held || context < upto) {
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) words[i] = 0;
      __syncthreads();
      for (int i = tid; i < a.biases; i += kThreads) {  // the last of a token's
        const uint32_t at = static_cast<uint32_t>(a.bias_ids[seq * a.bias_stride + i]) - static_cast<uint32_t>(lo);
        if (at < static_cast<uint32_t>(n)) atomicMax(words + at, static_cast<uint32_t>(i + 1) << kBiasShift);
      }
      held = seq;
      upto = 0;
    }
    __syncthreads();
    for (int i = upto + tid; i < context; i += kThreads) {
      const long long at = token(row, i) - lo;
      if (at < 0 || at >= n) continue;
      if (i < prompt) atomicOr(words + at, kInPrompt);
      else atomicAdd(words + at, 1u);
    }
    upto = context;
    auto drafted = [&](uint32_t by) {
      if (!record) return;
      const int base = context & ~63;
      for (int i = tid; i < 32 * (a.tree_ints - paged::kTreeWords); i += kThreads) {
        if (base + i < context || !(static_cast<uint32_t>(record[paged::kTreeWords + (i >> 5)]) >> (i & 31) & 1)) continue;
        const long long at = token(row, base + i) - lo;
        if (at >= 0 && at < n) atomicAdd(words + at, by);
      }
    };
    drafted(1u);
    __syncthreads();
    Rules rules;
    rules.repetition = a.repetition ? a.repetition[seq] : a.repetition_all;
    rules.frequency = a.frequency ? a.frequency[seq] : a.frequency_all;
    rules.presence = a.presence ? a.presence[seq] : a.presence_all;
    rules.bias = a.bias + seq * a.bias_stride;
    const long long at = r * a.stride + lo;
    const uint32_t* allowed = a.allowed ? a.allowed + r * a.allowed_stride + lo / 32 : nullptr;
    float* out = kGreedy ? nullptr : a.out + static_cast<long long>(r) * a.V + lo;
    unsigned long long best = 0;
    for (int i = tid * kVec; i < n; i += kThreads * kVec) {
      float v[kVec];
      load<kType, kVec>(a.x, at + i, v);
      const uint32_t bits = allowed ? allowed[i >> 5] >> (i & 31) : 0xffffffffu;
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const uint32_t word = words[i + k];
        if (word) v[k] = apply(v[k], word, rules);
        if (!(bits >> k & 1)) v[k] = -__builtin_inff();
        if constexpr (kGreedy) best = most(best, order_key(v[k], lo + i + k));
      }
      if constexpr (!kGreedy) {
        if constexpr (kVec == 4) *reinterpret_cast<f32x4*>(out + i) = f32x4{v[0], v[1], v[2], v[3]};
        else out[i] = v[0];
      }
    }
    if constexpr (kGreedy) {
      best = wave_most(best);
      if ((tid & 63) == 0) s_best[tid >> 6] = best;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < kThreads / 64; ++w) best = most(best, s_best[w]);
        a.best[static_cast<long long>(r) * a.slices + blockIdx.x] = best;
      }
    }
    __syncthreads();
    drafted(0xffffffffu);
  }
}

// A wave per row: the best of its slices.
__global__ __launch_bounds__(64) void choose_kernel(const unsigned long long* __restrict__ best, int slices,
                                                    long long* __restrict__ token) {
  const unsigned long long* row = best + static_cast<long long>(blockIdx.x) * slices;
  unsigned long long b = 0;
  for (int i = static_cast<int>(threadIdx.x); i < slices; i += 64) b = most(b, row[i]);
  b = wave_most(b);
  if (threadIdx.x == 0) token[blockIdx.x] = 0xffffffffu - static_cast<uint32_t>(b);
}

// How N rows of V logits are cut up: slices of the vocabulary, a multiple of 2048
// tokens, and rows to a workgroup.
void cut(int N, int V, int* slice, int* rows) {
  const long long wgs = 512;
  long long s = (static_cast<long long>(N) * V / wgs + kLeastSlice - 1) / kLeastSlice * kLeastSlice;
  s = std::min<long long>(std::max<long long>(s, kLeastSlice), kMostSlice);
  const long long slices = (V + s - 1) / s;
  *slice = static_cast<int>(s);
  *rows = static_cast<int>(std::min<long long>(std::max<long long>(1, N * slices / (2 * wgs)), 16));
}

}  // namespace logits
}  // namespace santa

using namespace santa;

extern "C" size_t santa_adjust_logits_workspace_size(int N, int V) {
  if (N <= 0 || V <= 0) return 0;
  int slice, rows;
  logits::cut(N, V, &slice, &rows);
  return static_cast<size_t>(N) * static_cast<size_t>((V + slice - 1) / slice) * 8;
}

extern "C" int santa_adjust_logits(const void* x, int dtype, long long stride, int N, int V,
                                   const santa_logit_rules* rules, const santa_paged_plan_info* info, const int* plan,
                                   float* out, long long* token, void* workspace, size_t workspace_bytes,
                                   hipStream_t stream) {
  using namespace logits;
  if (!x || !rules || N < 0 || V <= 0 || V > 1 << 30 || stride < V || (!out) == (!token) || (info && !plan))
    return set_error(SANTA_ERR_INVALID, "bad adjust_logits arguments");
  if (dtype != SANTA_BF16 && dtype != SANTA_F16 && dtype != SANTA_F32)
    return set_error(SANTA_ERR_UNSUPPORTED, "adjust_logits: logits are bf16, f16 or float32");
  if (info && info->tokens != N)
    return set_error(SANTA_ERR_INVALID, "adjust_logits: the plan is for %d rows; got %d", info->tokens, N);
  if (rules->tokens) {
    if (!info) return set_error(SANTA_ERR_INVALID, "adjust_logits: a plan says which tokens a row has seen");
    if (info->max_row >= rules->tokens_rows || info->max_len > rules->tokens_len)
      return set_error(SANTA_ERR_INVALID, "adjust_logits: the plan names token %d of row %d; there are %d rows of %d",
                       info->max_len - 1, info->max_row, rules->tokens_rows, rules->tokens_len);
    if (info->max_len > kMostTokens)
      return set_error(SANTA_ERR_UNSUPPORTED, "adjust_logits counts up to %d tokens. Got %d", kMostTokens, info->max_len);
    if (reinterpret_cast<uintptr_t>(rules->tokens) % (rules->tokens_wide ? 8 : 4) != 0)
      return set_error(SANTA_ERR_INVALID, "adjust_logits: tokens must be aligned");
  }
  if (rules->biases < 0 || (rules->biases > 0 && (!rules->bias_ids || !rules->bias)))
    return set_error(SANTA_ERR_INVALID, "bad adjust_logits arguments");
  if (rules->biases > kMostBiases)
    return set_error(SANTA_ERR_UNSUPPORTED, "adjust_logits: up to %d biases for a row. Got %d", kMostBiases,
                     rules->biases);
  if (N == 0) return clear_error();
  if (token && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8 != 0 ||
                workspace_bytes < santa_adjust_logits_workspace_size(N, V)))
    return set_error(SANTA_ERR_WORKSPACE, "adjust_logits: workspace too small");
  Args a{};
  a.x = x;
  a.stride = stride;
  a.V = V, a.N = N;
  cut(N, V, &a.slice, &a.rows);
  a.slices = (V + a.slice - 1) / a.slice;
  a.tokens = rules->tokens;
  a.wide = rules->tokens_wide;
  a.tokens_stride = rules->tokens_stride;
  a.prompts = rules->prompts;
  a.repetition = rules->repetition, a.frequency = rules->frequency, a.presence = rules->presence;
  a.repetition_all = rules->repetition_all, a.frequency_all = rules->frequency_all;
  a.presence_all = rules->presence_all;
  a.bias_ids = rules->bias_ids, a.bias = rules->bias, a.biases = rules->biases, a.bias_stride = rules->bias_stride;
  a.allowed = reinterpret_cast<const uint32_t*>(rules->allowed);
  a.allowed_stride = rules->allowed_stride;
  if (info) {
    a.pos = reinterpret_cast<const int2*>(plan + info->pos_at);
    if (info->tree_ints > 0) a.tree = plan + info->tree_at, a.tree_ints = info->tree_ints;
  }
  a.out = out;
  a.best = static_cast<unsigned long long*>(workspace);
  const int group = (N + a.rows - 1) / a.rows;
  if (group > 65535) return set_error(SANTA_ERR_INVALID, "adjust_logits: too many rows");
  const int size = dtype == SANTA_F32 ? 4 : 2;
  // four logits at a time where every row's are aligned
  const bool vec = V % 4 == 0 && stride % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * size) == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.slices), static_cast<unsigned>(group)), dim3(kThreads),
                       static_cast<unsigned>(std::min(a.slice, (V + 3) / 4 * 4)) * 4, stream, a);
  };
  auto run = [&](auto type) {
    constexpr int kType = decltype(type)::value;
    if (token) vec ? launch(adjust_kernel<kType, 4, true>) : launch(adjust_kernel<kType, 1, true>);
    else vec ? launch(adjust_kernel<kType, 4, false>) : launch(adjust_kernel<kType, 1, false>);
  };
  if (dtype == SANTA_F32) run(std::integral_constant<int, SANTA_F32>{});
  else if (dtype == SANTA_BF16) run(std::integral_constant<int, SANTA_BF16>{});
  else run(std::integral_constant<int, SANTA_F16>{});
  if (token)
    hipLaunchKernelGGL(choose_kernel, dim3(static_cast<unsigned>(N)), dim3(64), 0, stream, a.best, a.slices, token);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "adjust_logits launch failed: %s", hipGetErrorString(e));
  return clear_error();
}
