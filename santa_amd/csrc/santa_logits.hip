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
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kLeastSlice = 4 * kThreads;
constexpr int kMostSteps = 3;  // of that size in a slice: 68 KiB of LDS, two workgroups per compute unit

// What a slice's word says of a token.
constexpr uint32_t kCount = 0x7ffffu;       // how often it is in the answer
constexpr uint32_t kInPrompt = 0x80000u;    // whether it is in the prompt
constexpr uint32_t kDrafted = 0x100000u;    // whether it is a drafted token, of this row's path or not
constexpr int kBiasShift = 21;              // above: its bias's number, and one
constexpr int kMostBiases = 2046;
constexpr int kMostTokens = 0x7ffff;
constexpr uint32_t kUntouched = 0x7fc0feedu;  // a NaN; a result with these bits is written as another one

struct Args {
  const void* x;
  long long stride;
  int V, N, rows;  // rows: of a workgroup
  const void* tokens;
  int wide, tokens_len;
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
  unsigned long long* best;  // [N, slices, waves]
};

// Larger for larger values, NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
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
  if (count) x = x - r.frequency * static_cast<float>(count) - r.presence;  // of others not even 0 times an infinity
  if (word >> kBiasShift) x = x + r.bias[(word >> kBiasShift) - 1];
  return x;
}

// Four logits as they lie in memory.
template <int kType>
struct Four {
  u32x4 raw;
};
template <>
struct Four<SANTA_BF16> {
  u32x2 raw;
};
template <>
struct Four<SANTA_F16> {
  u32x2 raw;
};

// Four logits from x[at] on, which need no more than their own alignment; at the end
// of a row those that there are.
template <int kType>
__device__ __forceinline__ Four<kType> load4(const void* x, long long at, int left) {
  Four<kType> v;
  if constexpr (kType == SANTA_F32) {
    typedef u32x4 Loose __attribute__((aligned(4)));
    const uint32_t* p = static_cast<const uint32_t*>(x) + at;
    if (left >= 4) {
      v.raw = *reinterpret_cast<const Loose*>(p);
    } else {
      v.raw = u32x4{p[0], left > 1 ? p[1] : 0, left > 2 ? p[2] : 0, 0};
    }
  } else {
    typedef u32x2 Loose __attribute__((aligned(2)));
    const uint16_t* p = static_cast<const uint16_t*>(x) + at;
    if (left >= 4) {
      v.raw = *reinterpret_cast<const Loose*>(p);
    } else {
      v.raw = u32x2{p[0] | (left > 1 ? static_cast<uint32_t>(p[1]) << 16 : 0), left > 2 ? p[2] : 0u};
    }
  }
  return v;
}
template <int kType>
__device__ __forceinline__ float value(const Four<kType>& v, int k) {
  if constexpr (kType == SANTA_F32) return __uint_as_float(v.raw[k]);
  else return k & 1 ? hi16_to_f32<kType == SANTA_BF16>(v.raw[k >> 1]) : lo16_to_f32<kType == SANTA_BF16>(v.raw[k >> 1]);
}

__device__ __forceinline__ int token_at(const Args& a, const void* row, int i) {
  if (!a.wide) return static_cast<const int*>(row)[i];
  const long long v = static_cast<const long long*>(row)[i];
  return v < 0 || v > 0x7fffffff ? -1 : static_cast<int>(v);
}

// Tokens of the places from i0 on, before end, four a lane and step: 16 a lane.
constexpr int kTokenSteps = 4, kTokens = 4 * kThreads * kTokenSteps;
__device__ __forceinline__ void ask_tokens(const Args& a, const void* row, int i0, int end,
                                           int (&id)[kTokenSteps][4]) {
  typedef i32x4 Four __attribute__((aligned(4)));
#pragma unroll
  for (int k = 0; k < kTokenSteps; ++k) {
    const int i = i0 + 4 * (static_cast<int>(threadIdx.x) + k * kThreads);
    if (!a.wide && i + 3 < end) {
      const i32x4 v = *reinterpret_cast<const Four*>(static_cast<const int*>(row) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) id[k][j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) id[k][j] = i + j < end ? token_at(a, row, i + j) : -1;
    }
  }
}

// What is asked for of a row ahead of its turn, as it lies in memory: anything done
// with it there would wait for it.
template <int kType, int kSteps>
struct Ahead {
  Four<kType> x[kSteps];
  uint32_t bits[kSteps];
  int2 at = {-1, 0};  // position, sequence
  int2 head = {0, -1};  // of its record
  uint32_t path = 0;    // the record's bits of 32 places, this lane's among them
};

// Workgroup (slice of the vocabulary, rows): counts what a row has seen of its
// slice in LDS, with integers, whose order does not matter, and lists the tokens with
// a count or a bias.  For each row the listed tokens' logits are worked out first, a
// lane each, into LDS, and then the row passes once, with a select between a logit and
// what LDS has of it: few tokens of a vocabulary are listed, but most waves would have
// some at any place.  Bound by HBM, and by what a group of rows does before its first
// one: 400 rows of 128256 float32 logits, trees of 16 sequences of 1000 to 20000 tokens
// under all rules, 417 MB, 92 us, 4.5 TB/s (a copy of the logits alone 77 us; 129 with
// the penalties in the pass, whose vector work bounded it, and 112 where the rows
// ahead were converted as they were asked for).  Single rows are the first loads'
// latency: 64 of 10 000 tokens each 29.5 us, four with the token chosen 7 and 3.5.
// The rows of a sequence follow one another (a plan's tokens), so the next one only
// adds the tokens that it sees beyond the row before; of a tree's tokens every lane
// holds one, and adds or takes it away where the next row differs.  Two rows are on
// their way while one is worked on; workgroups of one row (not kMany) need half the
// registers, so that more of them hide each other's first loads.
template <int kType, int kSteps, bool kGreedy, bool kMany>
__global__ __launch_bounds__(kThreads, kMany || kSteps == kMostSteps ? 4 : 6) void adjust_kernel(Args a) {
  constexpr int kSlice = kLeastSlice * kSteps;
  __shared__ uint32_t words[kSlice];
  __shared__ u32x4 results4[kSlice / 4];
  __shared__ uint16_t list[kSlice];
  __shared__ float bias[kMostBiases + 2];
  __shared__ int listed;
  uint32_t* const results = reinterpret_cast<uint32_t*>(results4);
  const int tid = static_cast<int>(threadIdx.x);
  const int lo = static_cast<int>(blockIdx.x) * kSlice, n = min(kSlice, a.V - lo);
  const int first = static_cast<int>(blockIdx.y) * a.rows, end = min(first + a.rows, a.N);
  const bool ruled = a.tokens || a.biases > 0;
  const int drafts = a.tree ? 32 * (a.tree_ints - paged::kTreeWords) : 0;
  // The id's word, changed by `change`, is listed where it was 0 (only a draft's mark,
  // which stays, keeps a word that goes back to 0).
  auto touch = [&](int id, auto change) {
    const uint32_t at = static_cast<uint32_t>(id) - static_cast<uint32_t>(lo);
    if (at < static_cast<uint32_t>(n) && change(words + at) == 0) list[atomicAdd(&listed, 1)] = static_cast<uint16_t>(at);
  };
  auto logit = [&](int r, int at) {
    const long long i = r * a.stride + lo + at;
    if constexpr (kType == SANTA_F32) return static_cast<const float*>(a.x)[i];
    else return h16_to_f32<kType == SANTA_BF16>(static_cast<const uint16_t*>(a.x)[i]);
  };
  auto ask = [&](Ahead<kType, kSteps>& w, int r) {
    if (r >= end) return;
#pragma unroll
    for (int p = 0; p < kSteps; ++p) {
      const int i = (p * kThreads + tid) * 4;
      if (i >= n) continue;
      w.x[p] = load4<kType>(a.x, r * a.stride + lo + i, n - i);
      if (a.allowed) w.bits[p] = a.allowed[r * a.allowed_stride + ((lo + i) >> 5)];
    }
    if (a.pos) w.at = a.pos[r];
    if (a.tree) {
      const int* record = a.tree + static_cast<long long>(r) * a.tree_ints;
      w.head = *reinterpret_cast<const int2*>(record);
      if (tid < drafts) w.path = static_cast<uint32_t>(record[paged::kTreeWords + (tid >> 5)]);
    }
  };
  int held = -1, upto = 0;   // the words are those of this sequence's first tokens,
  bool added = false;        // this lane's drafted token where this is set,
  const int* far = nullptr;  // and those beyond the lanes that this record's token follows,
  int tree_base = -1;        // of the tree behind this place (-1: none are marked)
  int mine = -1;             // the drafted token
  int own = -1;                  // the listed token that this lane has the logit of, for the next row
  float own_logit = 0.0f;
  Rules rules{1.0f, 0.0f, 0.0f, bias};
  auto work_on = [&](Ahead<kType, kSteps>& w, int r) {
    const int seq = a.pos ? w.at.y : r, context = !a.tokens ? 0 : a.tree ? w.head.x : w.at.x + 1;
    // a tree's token lies behind the context that it sees, others are the last of theirs
    const bool drafted = a.tokens && a.tree && w.head.y >= 0 && context <= w.at.x;
    // a tree's token that is not in use has seen nothing; the words stay those of the rows around it
    const bool unused = a.tokens && a.tree && w.head.y < 0;
    int count = 0;
    if (ruled) {
      const void* row = static_cast<const char*>(a.tokens) + seq * a.tokens_stride * (a.wide ? 8 : 4);
      const int base = context & ~63;
      const bool anew = seq != held || (!unused && (context < upto || (tree_base >= 0 && !(drafted && base == tree_base &&
                                                                                           context == upto))));
      if (anew) upto = 0, tree_base = -1;
      // what is read here is asked for before any of it is used
      int id[kTokenSteps][4], bias_id = -1;
      float bias_value = 0.0f;
      if (anew && tid < a.biases) {
        bias_id = a.bias_ids[seq * a.bias_stride + tid];
        bias_value = a.bias[seq * a.bias_stride + tid];
      }
      if (context > upto) ask_tokens(a, row, upto, context, id);
      const bool plant = drafted && tree_base < 0;
      if (plant) {
        mine = tid < drafts && base + tid >= context && base + tid < a.tokens_len ? token_at(a, row, base + tid) : -1;
        tree_base = base;
      }
      if (anew) {
        rules.repetition = a.repetition ? a.repetition[seq] : a.repetition_all;
        rules.frequency = a.frequency ? a.frequency[seq] : a.frequency_all;
        rules.presence = a.presence ? a.presence[seq] : a.presence_all;
        __syncthreads();  // the row before has been worked on
#pragma unroll
        for (int p = 0; p < kSteps; ++p) {
          reinterpret_cast<u32x4*>(words)[p * kThreads + tid] = u32x4{0, 0, 0, 0};
          results4[p * kThreads + tid] = u32x4{kUntouched, kUntouched, kUntouched, kUntouched};
        }
        if (tid == 0) listed = 0;
        __syncthreads();
        for (int i = tid; i < a.biases; i += kThreads) {  // the last of a token's
          if (i != tid) {
            bias_id = a.bias_ids[seq * a.bias_stride + i];
            bias_value = a.bias[seq * a.bias_stride + i];
          }
          bias[i] = bias_value;
          touch(bias_id, [&](uint32_t* at) { return atomicMax(at, static_cast<uint32_t>(i + 1) << kBiasShift); });
        }
        __syncthreads();
        held = seq;
        added = false;
        far = nullptr;
        own = -1;
      }
      if (context > upto) {
        const int prompt = a.prompts ? a.prompts[seq] : 0;
        for (int i0 = upto; i0 < context; i0 += kTokens) {
          int now[kTokenSteps][4];
#pragma unroll
          for (int k = 0; k < kTokenSteps; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) now[k][j] = id[k][j];
          if (i0 + kTokens < context) ask_tokens(a, row, i0 + kTokens, context, id);
#pragma unroll
          for (int k = 0; k < kTokenSteps; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int i = i0 + 4 * (tid + k * kThreads) + j;
              if (i >= context) continue;
              touch(now[k][j], [&](uint32_t* at) { return i < prompt ? atomicOr(at, kInPrompt) : atomicAdd(at, 1u); });
            }
        }
        upto = context;
      }
      if (plant) {
        touch(mine, [](uint32_t* at) { return atomicOr(at, kDrafted); });
        for (int i = tid + kThreads; i < drafts && base + i < a.tokens_len; i += kThreads)  // all behind the context
          touch(token_at(a, row, base + i), [](uint32_t* at) { return atomicOr(at, kDrafted); });
      }
      if (drafted) {
        const bool want = (w.path >> (tid & 31) & 1) && base + tid >= context;
        const uint32_t by = want ? 1u : 0xffffffffu;
        if (want != added) touch(mine, [&](uint32_t* at) { return atomicAdd(at, by) | 1u; });
        added = want;
        const int* record = a.tree + static_cast<long long>(r) * a.tree_ints;
        for (int i = tid + kThreads; i < drafts; i += kThreads) {
          auto follows = [&](const int* of) {
            return (static_cast<uint32_t>(of[paged::kTreeWords + (i >> 5)]) >> (i & 31) & 1) != 0;
          };
          const bool had = far && follows(far), now = follows(record);
          const uint32_t far_by = now ? 1u : 0xffffffffu;
          if (had != now) touch(token_at(a, row, base + i), [&](uint32_t* at) { return atomicAdd(at, far_by) | 1u; });
        }
        far = record;
      }
      __syncthreads();
      count = listed;
      for (int i = tid; i < count; i += kThreads) {
        const int at = list[i];
        const float x = i == tid && at == own ? own_logit : logit(r, at);
        const uint32_t word = unused ? words[at] & ~(kCount | kInPrompt) : words[at];
        const uint32_t result = __float_as_uint(apply(x, word, rules));
        results[at] = result == kUntouched ? 0x7fc00000u : result;
      }
      __syncthreads();
    }
    Four<kType> x[kSteps];
    uint32_t bits[kSteps];
#pragma unroll
    for (int p = 0; p < kSteps; ++p) x[p] = w.x[p], bits[p] = w.bits[p];
    // before the rows ahead: loads are waited for in order
    if (kMany && r + 1 < end && tid < count) {
      own = list[tid];
      own_logit = logit(r + 1, own);
    }
    if (kMany) ask(w, r + 2);
    uint32_t best = 0;
    int best_at = 0;
#pragma unroll
    for (int p = 0; p < kSteps; ++p) {
      const int i = (p * kThreads + tid) * 4;
      if (i >= n) continue;
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = value<kType>(x[p], k);
      if (ruled) {
        const u32x4 result = results4[i / 4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (result[k] != kUntouched) v[k] = __uint_as_float(result[k]);
      }
      if (a.allowed) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t stays = static_cast<uint32_t>(__builtin_amdgcn_sbfe(bits[p] >> (i & 31), k, 1));
          v[k] = __uint_as_float((__float_as_uint(v[k]) & stays) | (0xff800000u & ~stays));
        }
      }
      if constexpr (kGreedy) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t key = order_key(v[k]);
          if (i + k < n && key > best) best = key, best_at = lo + i + k;
        }
      } else {
        typedef f32x4 Four __attribute__((aligned(4)));
        float* out = a.out + static_cast<long long>(r) * a.V + lo + i;
        if (n - i >= 4) {
          *reinterpret_cast<Four*>(out) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
          for (int k = 0; k < 3; ++k)
            if (i + k < n) out[k] = v[k];
        }
      }
    }
    if constexpr (kGreedy) {  // among equal values the first index
      const unsigned long long most = wave_most(static_cast<unsigned long long>(best) << 32 |
                                                (0xffffffffu - static_cast<uint32_t>(best_at)));
      if ((tid & 63) == 0)
        a.best[(static_cast<long long>(r) * gridDim.x + blockIdx.x) * kWaves + (tid >> 6)] = most;
    }
  };
  Ahead<kType, kSteps> even, odd;
  ask(even, first);
  if constexpr (!kMany) {
    work_on(even, first);
    return;
  }
  ask(odd, first + 1);
  for (int r = first; r < end; r += 2) {
    work_on(even, r);
    if (r + 1 < end) work_on(odd, r + 1);
  }
}

// A wave per row: the best of its parts.
__global__ __launch_bounds__(64) void choose_kernel(const unsigned long long* __restrict__ best, int parts,
                                                    long long* __restrict__ token) {
  const unsigned long long* row = best + static_cast<long long>(blockIdx.x) * parts;
  unsigned long long b = 0;
  for (int i0 = 0; i0 < parts; i0 += 64 * 8) {
    unsigned long long v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + 64 * k + static_cast<int>(threadIdx.x);
      v[k] = i < parts ? row[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) b = most(b, v[k]);
  }
  b = wave_most(b);
  if (threadIdx.x == 0) token[blockIdx.x] = 0xffffffffu - static_cast<uint32_t>(b);
}

// How N rows of V logits are cut up: rows to a workgroup, as many as a sequence has
// on average (each group of them counts its sequence's tokens once) while there are
// two workgroups for each compute unit; then the largest slices, by which a
// sequence's tokens are read the fewest times, that leave as many or, for single rows,
// of which more run at once, four times as many (64 rows of 10 000 tokens behind
// 128256 logits: 31.6 us with two, 29.5 with eight for each compute unit).
void cut(int N, int V, int sequences, int* steps, int* rows) {
  constexpr long long kWorkgroups = 512;
  const long long least = (V + kLeastSlice - 1) / kLeastSlice;
  const long long each = sequences > 0 ? (N + sequences - 1) / sequences : 1;
  *rows = static_cast<int>(std::max(1LL, std::min({each, 32LL, N * least / kWorkgroups})));
  const long long groups = (N + *rows - 1) / *rows, want = *rows > 1 ? kWorkgroups : 4 * kWorkgroups;
  *steps = 1;
  for (const int s : {2, kMostSteps})
    if ((V + s * kLeastSlice - 1) / (s * kLeastSlice) * groups >= want) *steps = s;
}

}  // namespace logits
}  // namespace santa

using namespace santa;

namespace {
// 8-byte parts of a row's maximum.
size_t parts_of(int V, int steps) {
  const int slice = steps * logits::kLeastSlice;
  return static_cast<size_t>((V + slice - 1) / slice) * logits::kWaves;
}
}  // namespace

extern "C" size_t santa_adjust_logits_workspace_size(int N, int V, int sequences) {
  if (N <= 0 || V <= 0) return 0;
  int steps, rows;
  logits::cut(N, V, sequences, &steps, &rows);
  return static_cast<size_t>(N) * parts_of(V, steps) * 8;
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
  // what the kernels read in one piece: pairs of the plan's, one element of all else
  const auto aligned = [](const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; };
  if (info && !aligned(plan, 16))
    return set_error(SANTA_ERR_INVALID, "adjust_logits: the plan must be 16-byte aligned");
  if (!aligned(x, dtype == SANTA_F32 ? 4 : 2) || !aligned(out, 4) || !aligned(token, 8))
    return set_error(SANTA_ERR_INVALID, "adjust_logits: logits and output must be aligned to their elements");
  for (const void* p : {static_cast<const void*>(rules->prompts), static_cast<const void*>(rules->repetition),
                        static_cast<const void*>(rules->frequency), static_cast<const void*>(rules->presence),
                        static_cast<const void*>(rules->bias_ids), static_cast<const void*>(rules->bias),
                        static_cast<const void*>(rules->allowed)})
    if (!aligned(p, 4))
      return set_error(SANTA_ERR_INVALID, "adjust_logits: the rules' arrays must be aligned to their elements");
  if (info && info->tokens != N)
    return set_error(SANTA_ERR_INVALID, "adjust_logits: the plan is for %d rows; got %d", info->tokens, N);
  if (rules->tokens) {
    if (!info) return set_error(SANTA_ERR_INVALID, "adjust_logits: a plan says which tokens a row has seen");
    if (info->max_row >= rules->tokens_rows || info->max_len > rules->tokens_len)
      return set_error(SANTA_ERR_INVALID, "adjust_logits: the plan names token %d of row %d; there are %d rows of %d",
                       info->max_len - 1, info->max_row, rules->tokens_rows, rules->tokens_len);
    if (info->max_len > kMostTokens)
      return set_error(SANTA_ERR_UNSUPPORTED, "adjust_logits counts up to %d tokens. Got %d", kMostTokens, info->max_len);
    if (!aligned(rules->tokens, rules->tokens_wide ? 8 : 4))
      return set_error(SANTA_ERR_INVALID, "adjust_logits: tokens must be aligned");
  }
  if (rules->biases < 0 || (rules->biases > 0 && (!rules->bias_ids || !rules->bias)))
    return set_error(SANTA_ERR_INVALID, "bad adjust_logits arguments");
  if (rules->biases > kMostBiases)
    return set_error(SANTA_ERR_UNSUPPORTED, "adjust_logits: up to %d biases for a row. Got %d", kMostBiases,
                     rules->biases);
  if (N == 0) return clear_error();
  if (token && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8 != 0 ||
                workspace_bytes < santa_adjust_logits_workspace_size(N, V, rules->sequences)))
    return set_error(SANTA_ERR_WORKSPACE, "adjust_logits: workspace too small");
  Args a{};
  a.x = x;
  a.stride = stride;
  a.V = V, a.N = N;
  int steps;
  cut(N, V, rules->sequences, &steps, &a.rows);
  a.tokens = rules->tokens;
  a.wide = rules->tokens_wide;
  a.tokens_len = rules->tokens_len;
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
  a.rows = std::max(a.rows, (N + 65534) / 65535);  // a grid's second dimension
  const int group = (N + a.rows - 1) / a.rows;
  const int parts = static_cast<int>(parts_of(V, steps));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(parts / kWaves), static_cast<unsigned>(group)),
                       dim3(kThreads), 0, stream, a);
  };
  auto run = [&](auto type) {
    constexpr int kType = decltype(type)::value;
    auto cut_to = [&](auto greedy, auto many) {
      constexpr bool kGreedy = decltype(greedy)::value, kMany = decltype(many)::value;
      if (steps == 1) launch(adjust_kernel<kType, 1, kGreedy, kMany>);
      else if (steps == 2) launch(adjust_kernel<kType, 2, kGreedy, kMany>);
      else launch(adjust_kernel<kType, kMostSteps, kGreedy, kMany>);
    };
    if (token) a.rows > 1 ? cut_to(std::true_type{}, std::true_type{}) : cut_to(std::true_type{}, std::false_type{});
    else a.rows > 1 ? cut_to(std::false_type{}, std::true_type{}) : cut_to(std::false_type{}, std::false_type{});
  };
  if (dtype == SANTA_F32) run(std::integral_constant<int, SANTA_F32>{});
  else if (dtype == SANTA_BF16) run(std::integral_constant<int, SANTA_BF16>{});
  else run(std::integral_constant<int, SANTA_F16>{});
  if (token)
    hipLaunchKernelGGL(choose_kernel, dim3(static_cast<unsigned>(N)), dim3(64), 0, stream, a.best, parts, token);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(SANTA_ERR_HIP, "adjust_logits launch failed: %s", hipGetErrorString(e));
  return clear_error();
}
