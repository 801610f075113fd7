// Router of the expert MLP: each token's k experts, their weights, and the
// plan that groups the tokens' rows by expert; and the weighted sum that
// brings the experts' rows back.
//
//   chosen[t, j]  j-th largest logit of token t (ties to the lower expert)
//   weights       exp(l - l_max) over its sum (selected, or all, experts)
//   offsets[e]    number of slots (t, j) with an expert below e
//   positions     offsets[expert] + number of earlier slots of that expert
//
// The plan is a stable counting sort of the tokens * k slots without atomics
// on memory, so it is the same on every run.  A workgroup takes a stretch of
// tokens, kPass at a time: each wave chooses for four tokens, finds the ranks
// of its slots among themselves by ballots over the bits of the expert, and
// the waves' counts are added up in LDS.  A second launch adds the counts of
// the workgroups before; a batch of up to 256 tokens (more than 256
// experts: 128) is one stretch and needs none.
//
// Choosing is what takes time, and it is a chain: k times a maximum over the
// experts.  Up to 256 experts lie on 16 lanes, so that a wave works on four
// tokens at once and a maximum is four row rotations in the VALU.  16384
// tokens, 128 experts, k = 8, bf16: 9.6 us and 7-8 for the second launch (one
// token a wave: 84 in all); one token: 4 us.
//
// The sum is bound by memory: 8192 tokens of 4 rows of 4096 in 66 us, 5.6
// TB/s.
#include "common.hpp"
#include "experts.hpp"
#include "kernels.hpp"

namespace kiosk {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kWaveTokens = 4;
constexpr int kPass = kWaves * kWaveTokens;     // 64 tokens
// one launch up to here: what fits 64 KiB of LDS with k = 32
template <int G>
constexpr int kOne = G == 16 ? 4 * kPass : 2 * kPass;
constexpr int kMaxBlocks = 256;                 // stretches of a larger batch

// float -> unsigned that orders alike; every NaN above +inf, -0 as +0
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
constexpr uint32_t kMasked = 0x007fffffu;   // order_key(-inf)

// the number behind a key (of a NaN: a NaN)
__device__ __forceinline__ float key_value(uint32_t key) {
  if (key == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// of the upper half of a key (a bf16 number's: its lower bits are zeros, or
// all ones where the order is turned over)
__device__ __forceinline__ float key_value16(uint32_t key) {
  return key_value((key & 0x80000000u) && key < 0xffff0000u
                       ? key & 0xffff0000u : key | 0xffffu);
}

// Reductions over groups of G = 16 or 64 lanes, the result in every lane:
// rotations within the rows of 16, then across the rows.
template <int CTRL>
__device__ __forceinline__ uint32_t rotated(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}
template <int G, typename Op>
__device__ __forceinline__ uint32_t reduce(uint32_t v, Op op) {
  v = op(v, rotated<0x128>(v));
  v = op(v, rotated<0x124>(v));
  v = op(v, rotated<0x122>(v));
  v = op(v, rotated<0x121>(v));
  if constexpr (G == 64) {
    v = op(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
    v = op(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32)));
  }
  return v;
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  return reduce<G>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int G>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
  return reduce<G>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  return __uint_as_float(
      reduce<G>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
      }));
}

__device__ __forceinline__ float logit(const uint16_t* p) {
  return bf16_to_f32(*p);
}
__device__ __forceinline__ float logit(const float* p) { return *p; }

// G lanes, one token: lane g holds experts g, g + G, ...  The chosen experts
// go to `sel` (a.experts for a slot without one), the outputs to their
// places.  `live`: the token exists (all lanes take part in the reductions).
template <typename T, int G, int V>
__device__ __forceinline__ void select_token(const RouteArgs& a, int t,
                                             bool live, int lane,
                                             uint16_t* sel) {
  // A bf16 logit's key fills 16 bits; below it stands the expert, the lower
  // one the larger: one maximum finds both.
  constexpr bool kBoth = sizeof(T) == 2;
  const int g = lane & (G - 1);
  const T* row = static_cast<const T*>(a.logits) +
                 static_cast<size_t>(t) * a.experts;
  float l[V];
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * G + g;
    const bool in = live && e < a.experts;
    l[v] = in ? logit(row + e) : 0.0f;
    key[v] = in ? order_key(l[v]) : 0u;
    if (kBoth && in) key[v] = (key[v] & 0xffff0000u) | (0xffffu - e);
  }
  // slot j is kept by lane j % G
  constexpr int kSlots = G == 16 ? 2 : 1;
  float mine[kSlots] = {}, top = 0.0f, total = 0.0f;
  int expert[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) expert[s] = a.experts;
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) best = max(best, key[v]);
    best = group_max<G>(best);
    const bool found = best > kMasked;      // else: only masked experts left
    if (__ballot(found) == 0) break;
    uint32_t e = 0xffffffffu;
    float value;
    if constexpr (kBoth) {
      e = 0xffffu - (best & 0xffffu);
      value = key_value16(best);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (key[v] == best) key[v] = 0;
    } else {
#pragma unroll
      for (int v = V - 1; v >= 0; --v)
        if (key[v] == best) e = v * G + g;
      e = group_min<G>(e);
      value = key_value(best);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (found && static_cast<uint32_t>(v * G + g) == e) key[v] = 0;
    }
    if (j == 0) top = value;
    const float w = found ? expf(value - top) : 0.0f;
    total += w;
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
      if (found && g + s * G == j) {
        mine[s] = w;
        expert[s] = static_cast<int>(e);
      }
  }
  if (!a.renormalize) {
    total = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (live && v * G + g < a.experts) total += expf(l[v] - top);
    total = group_sum<G>(total);
  }
  if (!live) return;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const int j = g + s * G;
    if (j < a.k) {
      const bool chosen = expert[s] < a.experts;
      const size_t slot = static_cast<size_t>(t) * a.k + j;
      a.chosen[slot] = chosen ? expert[s] : -1;
      a.weights[slot] = chosen ? mine[s] / total : 0.0f;
      sel[j] = static_cast<uint16_t>(expert[s]);
    }
  }
}

// The wave's slots in order: rank among its own slots of the same expert to
// `rank`, its count of each expert to `count` (cleared before).  Lanes of a
// chunk of 64 slots find their equals by ballots, chunks follow each other.
__device__ __forceinline__ void rank_slots(int slots, int experts, int lane,
                                           const uint16_t* sel,
                                           uint16_t* rank, uint16_t* count) {
  const int bits = 32 - __builtin_clz(experts);   // `experts` itself occurs
  for (int base = 0; base < slots; base += kWave) {
    const int s = base + lane;
    const bool in = s < slots;
    const int e = in ? sel[s] : 0;
    unsigned long long same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    if (in) {
      const int before = __popcll(same & ((1ull << lane) - 1));
      const int seen = count[e];
      rank[s] = static_cast<uint16_t>(seen + before);
      // the last of the equals leaves the new count
      if ((same >> lane) == 1ull)
        count[e] = static_cast<uint16_t>(seen + before + 1);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// Exclusive sums over total[0 .. experts - 1] in place, their sum (where the
// slots without an expert begin) to total[experts].
__device__ __forceinline__ void scan_offsets(int experts, int* total,
                                             int* wave_sums) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int i = threadIdx.x;      // experts <= kThreads
  const int own = i < experts ? total[i] : 0;
  int incl = own;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int up = __shfl_up(incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == kWave - 1) wave_sums[wave] = incl;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < wave; ++w) base += wave_sums[w];
  if (i < experts) total[i] = base + incl - own;
  if (i == experts - 1) total[experts] = base + incl;
  __syncthreads();
}

// Row `base[e] + rank` is the slot's (behind the last expert's rows: one
// without an expert).
__device__ __forceinline__ void place(const RouteArgs& a, int slot, int e,
                                      int row) {
  const bool live = e < a.experts;
  a.positions[slot] = live ? row : -1;
  a.row_tokens[row] = live ? slot / a.k : -1;
}

// LDS: total, pass [experts + 1], wave_sums [kWaves]; count
// [kWaves][experts + 1], sel and rank [tokens][k] in 16 bits (a wave counts
// to 128 and one launch ranks to 8192)
unsigned select_lds(const RouteArgs& a, int tokens) {
  return (2 * (a.experts + 1) + kWaves) * 4 + kWaves * (a.experts + 1) * 2 +
         2 * tokens * a.k * 2;
}

template <typename T, int G, int V, bool ONE>
__global__ __launch_bounds__(kThreads) void route_select_kernel(RouteArgs a,
                                                                int stretch) {
  extern __shared__ __attribute__((aligned(16))) int lds[];
  constexpr int kTokens = ONE ? kOne<G> : kPass;
  const int words = a.experts + 1;
  int* total = lds;
  int* pass = total + words;
  int* wave_sums = pass + words;
  auto* count = reinterpret_cast<uint16_t*>(wave_sums + kWaves);
  uint16_t* sel = count + kWaves * words;
  uint16_t* rank = sel + kTokens * a.k;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int begin = blockIdx.x * stretch;
  const int end = min(begin + stretch, a.tokens);
  for (int e = threadIdx.x; e < words; e += kThreads) total[e] = pass[e] = 0;
  const int own = wave * kWaveTokens;          // the wave's first token
  for (int first = begin; first < end; first += kPass) {
    for (int i = threadIdx.x; i < kWaves * words; i += kThreads) count[i] = 0;
    const int mine = min(max(end - first - own, 0), kWaveTokens);
    // one launch keeps the slots of every pass
    const int at = ((ONE ? first - begin : 0) + own) * a.k;
    if constexpr (G == 16) {
      const int t = lane / 16;
      select_token<T, G, V>(a, first + own + t, t < mine, lane,
                            sel + at + t * a.k);
    } else {
      for (int t = 0; t < mine; ++t)
        select_token<T, G, V>(a, first + own + t, true, lane,
                              sel + at + t * a.k);
    }
    __syncthreads();
    rank_slots(mine * a.k, a.experts, lane, sel + at, rank + at,
               count + wave * words);
    __syncthreads();
    for (int e = threadIdx.x; e < words; e += kThreads) {
      total[e] += pass[e];                     // the passes before
      int sum = 0;
      for (int w = 0; w < kWaves; ++w) {       // and the waves before
        const int c = count[w * words + e];
        count[w * words + e] = static_cast<uint16_t>(sum);
        sum += c;
      }
      pass[e] = sum;
    }
    __syncthreads();
    for (int s = lane; s < mine * a.k; s += kWave) {
      const int e = sel[at + s];
      const int r = total[e] + count[wave * words + e] + rank[at + s];
      if constexpr (ONE)
        rank[at + s] = static_cast<uint16_t>(r);
      else                                     // waits for the second launch
        a.positions[(first + own) * a.k + s] = r;
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < words; e += kThreads) total[e] += pass[e];
  __syncthreads();
  if constexpr (ONE) {
    scan_offsets(a.experts, total, wave_sums);
    for (int e = threadIdx.x; e < words; e += kThreads)
      a.offsets[e] = total[e];
    for (int s = threadIdx.x; s < a.tokens * a.k; s += kThreads)
      place(a, s, sel[s], total[sel[s]] + rank[s]);
  } else {
    for (int e = threadIdx.x; e < words; e += kThreads)
      a.counts[blockIdx.x * words + e] = total[e];
  }
}

// Adds the counts of the workgroups before (each workgroup reads them all:
// at most 256 rows of 1025) and places the slots of its stretch.
__global__ __launch_bounds__(kThreads) void route_place_kernel(RouteArgs a,
                                                               int stretch) {
  extern __shared__ __attribute__((aligned(16))) int lds[];
  const int words = a.experts + 1;
  int* base = lds;
  int* before = base + words;
  int* wave_sums = before + words;
  for (int e = threadIdx.x; e < words; e += kThreads) base[e] = before[e] = 0;
  __syncthreads();
  // thread i: entry i % words of the workgroups i / words, + parts, ...
  const int blocks = gridDim.x;
  const int parts = max(kThreads / words, 1);
  for (int i = threadIdx.x; i < parts * words; i += kThreads) {
    const int e = i % words;
    int all = 0, mine = 0;
    // (eight loads in flight: one after the other they took 11 of 13 us)
    for (int b = i / words; b < blocks; b += 8 * parts) {
      int c[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        c[u] = a.counts[min(b + u * parts, blocks - 1) * words + e];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int at = b + u * parts;
        all += at < blocks ? c[u] : 0;
        mine += at < static_cast<int>(blockIdx.x) ? c[u] : 0;
      }
    }
    atomicAdd(&base[e], all);                  // in LDS: whole numbers
    atomicAdd(&before[e], mine);
  }
  __syncthreads();
  scan_offsets(a.experts, base, wave_sums);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e < words; e += kThreads) a.offsets[e] = base[e];
  __syncthreads();
  for (int e = threadIdx.x; e < words; e += kThreads) base[e] += before[e];
  __syncthreads();
  const int begin = blockIdx.x * stretch;
  const int end = min(begin + stretch, a.tokens);
  for (int s = begin * a.k + threadIdx.x; s < end * a.k; s += kThreads) {
    const int chosen = a.chosen[s];
    const int e = chosen < 0 ? a.experts : chosen;
    place(a, s, e, base[e] + a.positions[s]);
  }
}

// tokens of a workgroup: whole passes, at most kMaxBlocks workgroups
int stretch_of(int tokens) {
  const long long passes =
      (static_cast<long long>(tokens) + kPass - 1) / kPass;
  return static_cast<int>((passes + kMaxBlocks - 1) / kMaxBlocks * kPass);
}
int blocks_of(int tokens) {
  const int stretch = stretch_of(tokens);
  return static_cast<int>((static_cast<long long>(tokens) + stretch - 1) /
                          stretch);
}

template <typename T, int G, int V>
hipError_t launch_select(const RouteArgs& a, hipStream_t stream) {
  if (a.tokens <= kOne<G>)
    return launch_kernel(&route_select_kernel<T, G, V, true>, dim3(1),
                         dim3(kThreads), select_lds(a, kOne<G>), stream, a,
                         kOne<G>);
  const int stretch = stretch_of(a.tokens), blocks = blocks_of(a.tokens);
  hipError_t err = launch_kernel(&route_select_kernel<T, G, V, false>,
                                 dim3(blocks), dim3(kThreads),
                                 select_lds(a, kPass), stream, a, stretch);
  if (err != hipSuccess) return err;
  return launch_kernel(&route_place_kernel, dim3(blocks), dim3(kThreads),
                       (2 * (a.experts + 1) + kWaves) * 4u, stream, a,
                       stretch);
}

template <typename T>
hipError_t launch_type(const RouteArgs& a, hipStream_t stream) {
  if (a.experts <= 16) return launch_select<T, 16, 1>(a, stream);
  if (a.experts <= 32) return launch_select<T, 16, 2>(a, stream);
  if (a.experts <= 64) return launch_select<T, 16, 4>(a, stream);
  if (a.experts <= 128) return launch_select<T, 16, 8>(a, stream);
  if (a.experts <= 256) return launch_select<T, 16, 16>(a, stream);
  if (a.experts <= 512) return launch_select<T, 64, 8>(a, stream);
  return launch_select<T, 64, 16>(a, stream);
}

__global__ __launch_bounds__(64) void route_empty_kernel(int* offsets,
                                                         int words) {
  for (int e = threadIdx.x; e < words; e += 64) offsets[e] = 0;
}

// ---------------------------------------------------------------------------
// Weighted sum of a token's expert rows, fp32 in the order of the slots, one
// rounding.  Bound by memory: each row is read once.
constexpr int kCombineThreads = 256;

__global__ __launch_bounds__(kCombineThreads) void combine_kernel(
    const uint16_t* __restrict__ y, const int* __restrict__ positions,
    const float* __restrict__ weights, const uint16_t* residual,
    uint16_t* out, int k, int rows, int width, int chunks) {
  const int t = blockIdx.x;
  const int c = blockIdx.y * kCombineThreads + threadIdx.x;
  if (c >= chunks) return;
  const size_t at = static_cast<size_t>(t) * width + c * 8;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto add = [&](const uint16_t* p, float w) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __builtin_fmaf(w, __uint_as_float(u[i] << 16), v[2 * i]);
      v[2 * i + 1] = __builtin_fmaf(
          w, __uint_as_float(u[i] & 0xffff0000u), v[2 * i + 1]);
    }
  };
  for (int j = 0; j < k; ++j) {
    const int row = positions[static_cast<size_t>(t) * k + j];
    if (row < 0 || row >= rows) continue;
    add(y + static_cast<size_t>(row) * width + c * 8,
        weights[static_cast<size_t>(t) * k + j]);
  }
  if (residual != nullptr) add(residual + at, 1.0f);
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    u[i] = f32_to_bf16(v[2 * i]) |
           (static_cast<uint32_t>(f32_to_bf16(v[2 * i + 1])) << 16);
  *reinterpret_cast<uint4*>(out + at) = uint4{u[0], u[1], u[2], u[3]};
}

}  // namespace

size_t route_count_words(int tokens, int experts) {
  if (tokens <= (experts <= 256 ? kOne<16> : kOne<64>)) return 0;
  return static_cast<size_t>(blocks_of(tokens)) * (experts + 1);
}

hipError_t launch_route(const RouteArgs& a, hipStream_t stream) {
  if (a.tokens < 0 || a.experts < 1 || a.experts > kRouteMaxExperts ||
      a.k < 1 || a.k > a.experts || a.k > kRouteMaxK ||
      static_cast<long long>(a.tokens) * a.k > 0x7fffffffll)
    return hipErrorInvalidValue;
  if (a.tokens == 0)
    return launch_kernel(&route_empty_kernel, dim3(1), dim3(64), 0, stream,
                         a.offsets, a.experts + 1);
  return a.bf16 ? launch_type<uint16_t>(a, stream)
                : launch_type<float>(a, stream);
}

hipError_t launch_combine(const uint16_t* y, const int* positions,
                          const float* weights, const uint16_t* residual,
                          uint16_t* out, int tokens, int k, int rows,
                          int width, hipStream_t stream) {
  if (tokens < 0 || k < 1 || rows < 0 || width < 8 || width % 8 != 0)
    return hipErrorInvalidValue;
  if (tokens == 0) return hipSuccess;
  // (a grid has fewer than 2^32 threads along its first axis, and 2^16
  // workgroups along its second)
  constexpr int kPart = 1 << 23, kPartChunks = 65535 * kCombineThreads;
  for (int first = 0; first < tokens; first += kPart) {
    const int count = tokens - first < kPart ? tokens - first : kPart;
    const size_t slot = static_cast<size_t>(first) * k;
    for (int chunk = 0; chunk < width / 8; chunk += kPartChunks) {
      const int left = width / 8 - chunk;
      const int chunks = left < kPartChunks ? left : kPartChunks;
      const size_t col = static_cast<size_t>(chunk) * 8;
      const size_t at = static_cast<size_t>(first) * width + col;
      const dim3 grid(count,
                      (chunks + kCombineThreads - 1) / kCombineThreads);
      const hipError_t err = launch_kernel(
          &combine_kernel, grid, dim3(kCombineThreads), 0, stream, y + col,
          positions + slot, weights + slot,
          residual != nullptr ? residual + at : nullptr, out + at, k, rows,
          width, chunks);
      if (err != hipSuccess) return err;
    }
  }
  return hipSuccess;
}

}  // namespace kiosk
