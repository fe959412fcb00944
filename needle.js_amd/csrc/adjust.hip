// Penalties for repeated tokens, biases and allowed-token masks on logits, with
// the selection over the result.
//
// For row r, token v with logit l, c = times v was generated, seen = whether it
// is anywhere in the row's history (prompt or generated):
//   a = l;  seen: a = a > 0 ? a / repetition : a * repetition
//   c > 0: a = a - frequency c - presence
//   a = a + bias(v)
// in float64 without contraction, rounded once: the adjusted logits are float32
// values, as a Float32Array holds them.  bias(v) is the last entry of v in the
// row's list (Map semantics), 0 without one.  The id and log-probability are
// those of selectToken (model/runtime.ts:880-899) over the adjusted logits: the
// first maximum of the allowed ids, the log-softmax over all of them.  The
// adjusted logits leave with -inf where the mask forbids.
//
// Work: a workgroup takes segments of kSegment ids of a row.  It holds the row's
// history and biases in registers and enters those that fall into the segment in
// LDS counters and a list of the ids named; the list's ids are adjusted side by
// side (in place, by whichever lanes hold them, a wave pays the float64 sequence
// for each of its eight ids); then one pass over the segment's logits, with a
// running maximum, sum and best per thread, while the next segment's are on their
// way.  A row's workgroups meet in records, the last to arrive joins them.
#include <new>

#include "nd_internal.hpp"
#include "nd_select.hpp"
#include "nd_wave.hpp"

namespace {

using namespace nd::sel;

constexpr uint32_t kThreads = 512, kQuads = 2, kSegment = kThreads * 4 * kQuads;
constexpr uint32_t kWaves = kThreads / 64, kWords = kSegment / 32;
constexpr uint32_t kMaxRecords = 64;  // a lane of the joining wave each
constexpr uint32_t kCounterStride = 32;  // 128 bytes: an L2 line a row
constexpr uint32_t kPromptBit = 0x80000000u;

struct Record {
  float bv;         // best allowed value and its id
  uint32_t bo;
  float mx;         // JavaScript maximum of all
  uint32_t key;     // first allowed id << 1 | whether its logit is NaN
  double sum;       // sum of e^(a - mx)
  uint64_t pad;
};
static_assert(sizeof(Record) == 32, "record layout");

// The workspace: a counter of the rows that have advanced (nd_advance_row) in a line of
// its own, then every row's place, the same whatever the batch of a call, so that calls
// of any size up to the workspace's may follow one another.  Counters are zero between
// launches, records hold what the last launch left.
struct RowSpace {
  uint32_t arrived;  // workgroups of the row
  uint32_t pad[kCounterStride - 1];
  Record records[kMaxRecords];
};

template <int SCOPE>
__device__ __forceinline__ void put(uint32_t* p, uint32_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, SCOPE);
}
__device__ __forceinline__ uint32_t get(const uint32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A row's penalties.  The quotient a / repetition by the reciprocal, corrected once
// (with the reciprocal correctly rounded, a q r within an ulp of the quotient
// becomes the correctly rounded one: Markstein), where neither can leave the
// normal range; the division's own sequence takes four times the instructions.
struct Penalties {
  double rep, inv, freq, pres;
  bool plain;
};
__device__ __forceinline__ Penalties penalties(double rep, double freq, double pres) {
  return {rep, 1.0 / rep, freq, pres, fabs(rep) > 1e-30 && fabs(rep) < 1e30};
}
__device__ __forceinline__ double quotient(double a, const Penalties& p) {
  const double q = a * p.inv, c = fma(fma(-q, p.rep, a), p.inv, q);
  return p.plain && a < 1e39 ? c : a / p.rep;  // a is an f32: 1e39 is infinity's side
}

__device__ __forceinline__ float adjusted(float l, uint32_t counts, bool biased, float bias,
                                          const Penalties& p) {
#pragma clang fp contract(off)
  double a = (double)l;
  const uint32_t c = counts & ~kPromptBit;
  if (counts) a = a > 0.0 ? quotient(a, p) : a * p.rep;
  if (c) {  // an infinite penalty times no occurrence would be NaN
    a = a - p.freq * (double)c;
    a = a - p.pres;
  }
  if (biased) a = a + (double)bias;
  return (float)a;
}

// e^x for x <= 0 in float64, within 4e-11 of itself: x = k ln 2 / 64 + r,
// |r| <= 0.0055, 2^((k mod 64) / 64) from the workgroup's table with k div 64 added to
// its exponent, times the Taylor polynomial of degree 3 (remainder r^4 / 24 <
// 3.9e-11).  k is the low word of x 64 / ln 2 + 1.5 2^52.  Below -700, and of a NaN (a
// row whose maximum is NaN or infinite, whose sum is not used), e^x is e^-700: 1e-304
// in sums of 1 and more.  A sum carries 4e-11 from its terms and as much again from
// every larger maximum that it is scaled to: at most one a segment of its workgroup and
// three in the joins.  With (4 + segments) 4e-11 at most, it moves a log-probability by
// 2e-12 to 4e-12 over 8192 to 50001 normal logits; the library's exp takes five times
// the instructions.
__device__ __forceinline__ double exp_neg(double x, const double* table) {
  x = fmax(x, -700.0);
  const double shift = 6755399441055744.0, kd = fma(x, 92.33248261689366, shift);
  const int i = (int)__double_as_longlong(kd);
  const double r = fma(-(kd - shift), 0.010830424696249145, x);
  const double p = fma(fma(fma(1.0 / 6, r, 0.5), r, 1.0), r, 1.0);
  const long long t = __double_as_longlong(table[i & 63]);
  const uint32_t hi = (uint32_t)(t >> 32) + ((uint32_t)(i & ~63) << 14);
  return __longlong_as_double((long long)hi << 32 | (uint32_t)t) * p;
}

// Four logits at any 4-byte alignment (rows of an odd vocabulary).
typedef float f4 __attribute__((ext_vector_type(4)));
typedef f4 f4u __attribute__((aligned(4)));

constexpr uint32_t kHist = 4, kBias = 1;  // entries a thread holds in registers

__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  auto take = [&](int o) { v = min(v, (uint32_t)o); };
  take(__builtin_amdgcn_update_dpp(0, (int)v, nd::kQuadXor1, 0xF, 0xF, true));
  take(__builtin_amdgcn_update_dpp(0, (int)v, nd::kQuadXor2, 0xF, 0xF, true));
  take(__builtin_amdgcn_update_dpp(0, (int)v, nd::kHalfMirror, 0xF, 0xF, true));
  take(__builtin_amdgcn_update_dpp(0, (int)v, nd::kRowMirror, 0xF, 0xF, true));
  const uint32_t a = min((uint32_t)__builtin_amdgcn_readlane((int)v, 0),
                         (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
  const uint32_t b = min((uint32_t)__builtin_amdgcn_readlane((int)v, 32),
                         (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
  return min(a, b);
}

// The winner of the wave's candidates: the largest value, then the lowest id.
__device__ __forceinline__ Best wave_best(Best b) {
  float top = nd::row_max(b.order == kNone ? -INFINITY : b.v);
  top = nd::max_xor<16>(top);
  top = nd::max_xor<32>(top);
  return Best{top, wave_min(b.order != kNone && b.v == top ? b.order : kNone)};
}

// SELECT: ids and log-probabilities; STORE: the adjusted logits.  Workgroup
// (s, r) takes segments s, s + S, ... of row r; thread t the ids
// 4 (t + kThreads i) + [0, 4) of a segment.  XL: the grid is one-dimensional with a
// row's workgroups on one XCD (workgroup L runs on XCD L % 8), so that records and
// counters stay in its L2, as in the attention's chunk merge (nd_wave.hpp).
template <bool SELECT, bool STORE, bool XL>
__global__ __launch_bounds__(kThreads, 6) void adjust_kernel(
    const float* logits, uint32_t vocab, nd_logit_adjust p,
    const uint32_t* __restrict__ mask_all, float* out, uint32_t* __restrict__ ids,
    double* __restrict__ logprobs, uint32_t* __restrict__ rows_done, RowSpace* __restrict__ space,
    nd_select_advance adv, uint32_t rows, uint32_t S) {
  constexpr int kScope = XL ? __HIP_MEMORY_SCOPE_WORKGROUP : __HIP_MEMORY_SCOPE_AGENT;
  // Of the segment's ids: how often the history names them (then the adjusted
  // logit), the last bias entry + 1, a bit each if named at all, and a list of those.
  // The first two are zero but for named ids, whose readers clear them again; the
  // last two have a turn each.
  __shared__ __align__(16) uint32_t s_count[kSegment], s_bias[kSegment];
  __shared__ uint32_t s_named[2][kWords], s_listed[2];
  __shared__ uint16_t s_list[kSegment];
  __shared__ double s_table[64];
  __shared__ Record s_wave[kWaves];
  __shared__ uint32_t s_last;
  uint32_t part = blockIdx.x, r = blockIdx.y;
  if constexpr (XL) {
    const uint32_t L = blockIdx.x >> 3;
    part = L % S;
    r = 8 * (L / S) + (blockIdx.x & 7);
    if (r >= rows) return;
  }
  const uint32_t t = threadIdx.x, w = t >> 6, lane = t & 63;
  const float* row = logits + (size_t)r * vocab;
  const uint32_t words = (vocab + 31) / 32, segments = (vocab + kSegment - 1) / kSegment;
  const uint32_t* mask = mask_all ? mask_all + (size_t)r * words : nullptr;
  float next[kQuads][4];
  uint32_t next_allow[kQuads];
  auto load = [&](uint32_t base) {
#pragma unroll
    for (uint32_t i = 0; i < kQuads; ++i) {
      const uint32_t id = base + 4 * (t + i * kThreads);
      if (id + 4 <= vocab) {
        const f4u f = *reinterpret_cast<const f4u*>(row + id);
#pragma unroll
        for (int j = 0; j < 4; ++j) next[i][j] = f[j];
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) next[i][j] = id + j < vocab ? row[id + j] : -INFINITY;
      }
      next_allow[i] = id >= vocab ? 0u : mask ? mask[id >> 5] >> (id & 31) : 15u;
      if (id + 4 > vocab && id < vocab) next_allow[i] &= (1u << (vocab - id)) - 1;
    }
  };
  load(part * kSegment);
  // The row's lengths and penalties in one load, a lane each (loads under uniform
  // branches would wait for one another: 16 us against 11 at 64 x 32768), its
  // history and biases at once with it: entries past the lengths are dropped
  // when they are used.
  const void* const each[6] = {p.history_lengths, p.prompt_lengths, p.bias_counts,
                               p.repetition,      p.presence,       p.frequency};
  const uint32_t* from = nullptr;
#pragma unroll
  for (uint32_t i = 0; i < 6; ++i)
    if (lane == i) from = static_cast<const uint32_t*>(each[i]);
  const uint32_t told = from ? from[r] : 0u;
  const uint32_t* hist = p.history + (size_t)r * p.history_stride;
  const uint32_t* bias_ids = p.bias_ids + (size_t)r * p.bias_stride;
  const float* bias = p.bias + (size_t)r * p.bias_stride;
  const uint32_t most = p.history ? p.history_stride : 0, most_b = p.bias_ids ? p.bias_stride : 0;
  uint32_t he[kHist], be[kBias];
#pragma unroll
  for (uint32_t i = 0; i < kHist; ++i) {
    const uint32_t e = t + i * kThreads;
    he[i] = e < most ? hist[e] : kNone;
  }
#pragma unroll
  for (uint32_t i = 0; i < kBias; ++i) {
    const uint32_t e = t + i * kThreads;
    be[i] = e < most_b ? bias_ids[e] : kNone;
  }
  auto param = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)told, i); };
  auto penalty = [&](int i, double none) {
    return each[i] ? (double)__uint_as_float(param(i)) : none;
  };
  const uint32_t n = p.history_lengths ? min(param(0), most) : most;
  const uint32_t prompt = param(1);
  const uint32_t nb = p.bias_counts ? min(param(2), most_b) : most_b;
  const Penalties pen = penalties(penalty(3, 1.0), penalty(5, 0.0), penalty(4, 0.0));
#pragma unroll
  for (uint32_t i = 0; i < kHist; ++i)
    if (t + i * kThreads >= n) he[i] = kNone;
#pragma unroll
  for (uint32_t i = 0; i < kBias; ++i)
    if (t + i * kThreads >= nb) be[i] = kNone;

  if (n | nb) {
#pragma unroll
    for (uint32_t i = 0; i < kQuads; ++i) {
      *reinterpret_cast<uint4*>(&s_count[4 * (t + i * kThreads)]) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(&s_bias[4 * (t + i * kThreads)]) = make_uint4(0, 0, 0, 0);
    }
    if (t < kWords) s_named[0][t] = s_named[1][t] = 0;
    if (t < 2) s_listed[t] = 0;
  }
  if (SELECT && t < 64) s_table[t] = exp2((double)t / 64);
  nd::lds_barrier();

  // Calls f(id - base, index) on this thread's entries in the segment.
  auto history = [&](uint32_t base, auto f) {
#pragma unroll
    for (uint32_t i = 0; i < kHist; ++i)  // kNone lies past every segment
      if (i * kThreads < n && he[i] - base < kSegment) f(he[i] - base, t + i * kThreads);
    for (uint32_t e = t + kHist * kThreads; e < n; e += kThreads) {
      const uint32_t at = hist[e] - base;
      if (at < kSegment) f(at, e);
    }
  };
  auto biases = [&](uint32_t base, auto f) {
#pragma unroll
    for (uint32_t i = 0; i < kBias; ++i)
      if (i * kThreads < nb && be[i] - base < kSegment)
        f(be[i] - base, t + i * kThreads);
    for (uint32_t e = t + kBias * kThreads; e < nb; e += kThreads) {
      const uint32_t at = bias_ids[e] - base;
      if (at < kSegment) f(at, e);
    }
  };

  Best best{-INFINITY, kNone};
  float mx = -INFINITY;
  double sum = 0.0;
  uint32_t key = kNone;  // first allowed id << 1 | whether its logit is NaN; ids stay below 2^31
  uint32_t turn = 0;
  for (uint32_t seg = part; seg < segments; seg += S, turn ^= 1) {
    const uint32_t base = seg * kSegment;
    float v[kQuads][4];
    uint32_t allow[kQuads];
#pragma unroll
    for (uint32_t i = 0; i < kQuads; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = next[i][j];
      allow[i] = next_allow[i] & 15u;
    }
    if (n | nb) {
      uint32_t* const names = s_named[turn];
      if (t < kWords) s_named[turn ^ 1][t] = 0;  // read before the last barrier
      if (t == 0) s_listed[turn ^ 1] = 0;
      auto name = [&](uint32_t at) {
        const uint32_t bit = 1u << (at & 31);
        if (!(atomicOr(&names[at >> 5], bit) & bit)) s_list[atomicAdd(&s_listed[turn], 1u)] = at;
      };
      history(base, [&](uint32_t at, uint32_t e) {
        if (e < prompt) atomicOr(&s_count[at], kPromptBit);
        else atomicAdd(&s_count[at], 1u);
        name(at);
      });
      biases(base, [&](uint32_t at, uint32_t e) {
        atomicMax(&s_bias[at], e + 1);  // the last entry counts
        name(at);
      });
      nd::lds_barrier();
      const uint32_t listed = s_listed[turn];
      for (uint32_t i = t; i < listed; i += kThreads) {
        const uint32_t at = s_list[i], e = s_bias[at];
        if (base + at >= vocab) continue;
        const float l = row[base + at], add = e ? bias[e - 1] : 0.f;
        s_count[at] = __float_as_uint(adjusted(l, s_count[at], e != 0, add, pen));
        s_bias[at] = 0;
      }
      nd::lds_barrier();
#pragma unroll
      for (uint32_t i = 0; i < kQuads; ++i) {
        // All four at once: a branch for each would wait for the LDS eight times.
        const uint32_t at = 4 * (t + i * kThreads), named = names[at >> 5] >> (at & 31);
        uint4* const from = reinterpret_cast<uint4*>(&s_count[at]);
        const uint4 f = *from;
        *from = make_uint4(0, 0, 0, 0);
        const uint32_t f4s[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (((named >> j) & 1u) && base + at + j < vocab) v[i][j] = __uint_as_float(f4s[j]);
      }
      if (seg + S < segments) nd::lds_barrier();
    }
    if (seg + S < segments) load(base + S * kSegment);
    if constexpr (STORE) {
#pragma unroll
      for (uint32_t i = 0; i < kQuads; ++i) {
        const uint32_t id0 = base + 4 * (t + i * kThreads);
        float* to = out + (size_t)r * vocab + id0;
        f4u o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (allow[i] >> j) & 1u ? v[i][j] : -INFINITY;
        if (id0 + 4 <= vocab) *reinterpret_cast<f4u*>(to) = o;
        else
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j)
            if (id0 + j < vocab) to[j] = o[j];
      }
    }
    if constexpr (SELECT) {
      // Past the vocabulary v is -inf: no maximum, e^-inf = 0 in the sum.
      float top = v[0][0], win = -INFINITY;
#pragma unroll
      for (uint32_t i = 0; i < kQuads; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          top = __builtin_elementwise_maximum(top, v[i][j]);
          win = fmaxf(win, (allow[i] >> j) & 1u ? v[i][j] : -INFINITY);  // a NaN never wins
        }
      // The lowest id of a new best value; one of -inf is the first allowed id, if any.
      if (win > best.v) {
        best.v = win;
#pragma unroll
        for (int q = 4 * (int)kQuads - 1; q >= 0; --q)
          if (((allow[q / 4] >> (q % 4)) & 1u) && v[q / 4][q % 4] == win)
            best.order = base + 4 * (t + q / 4 * kThreads) + q % 4;
      }
      if (key == kNone) {
#pragma unroll
        for (int q = 4 * (int)kQuads - 1; q >= 0; --q)
          if ((allow[q / 4] >> (q % 4)) & 1u)
            key = (base + 4 * (t + q / 4 * kThreads) + q % 4) << 1 |
                  (uint32_t)(v[q / 4][q % 4] != v[q / 4][q % 4]);
      }
      top = __builtin_elementwise_maximum(top, mx);
      const double md = (double)top;
      sum = mx == top ? sum : mx == -INFINITY ? 0.0 : sum * exp_neg((double)mx - md, s_table);
      mx = top;
      if (top != -INFINITY) {
#pragma unroll
        for (uint32_t i = 0; i < kQuads; ++i)
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) sum += exp_neg((double)v[i][j] - md, s_table);
      }
    }
  }
  if constexpr (!SELECT) return;
  // Records of the wave's lanes to one, in every lane.
  auto join = [&] {
    const float own = mx;
    best = wave_best(best);
    key = wave_min(key);
    mx = nd::wave_max_js(mx);
    sum = nd::wave_sum(own == -INFINITY ? 0.0 : sum * exp_neg((double)own - (double)mx, s_table));
  };
  join();
  if (lane == 0) s_wave[w] = Record{best.v, best.order, mx, key, sum, 0};
  nd::lds_barrier();
  if (w == 0) {
    const Record o = s_wave[lane & (kWaves - 1)];
    const bool in = lane < kWaves;
    best = in ? Best{o.bv, o.bo} : Best{-INFINITY, kNone};
    mx = in ? o.mx : -INFINITY;
    key = in ? o.key : kNone;
    sum = in ? o.sum : 0.0;
    join();
  }
  // The row's choice, by one thread.
  auto finish = [&] {
    uint32_t id = kNone;
    double lp = __builtin_nan("");
    if (key != kNone) {
      // A NaN first candidate stays; without a value above -inf the first is it.  A
      // maximum of +inf has a sum of NaN.
      id = (key & 1) || best.order == kNone ? key >> 1 : best.order;
      if (!(key & 1) && mx != INFINITY)
        lp = (double)(best.order == kNone ? -INFINITY : best.v) - (double)mx - log(sum);
    }
    ids[r] = id;
    logprobs[r] = lp;
    if (adv.tokens) nd_advance_row(adv, r, rows, id, lp, rows_done);
  };
  if (S == 1) {
    if (t == 0) finish();
    return;
  }
  RowSpace* const own = space + r;
  if (t == 0) {
    uint32_t* rec = reinterpret_cast<uint32_t*>(own->records + part);
    put<kScope>(rec, __float_as_uint(best.v));
    put<kScope>(rec + 1, best.order);
    put<kScope>(rec + 2, __float_as_uint(mx));
    put<kScope>(rec + 3, key);
    const uint64_t bits = (uint64_t)__double_as_longlong(sum);
    put<kScope>(rec + 4, (uint32_t)bits);
    put<kScope>(rec + 5, (uint32_t)(bits >> 32));
    __builtin_amdgcn_s_waitcnt(0);  // the record has completed
    const bool last = __hip_atomic_fetch_add(&own->arrived, 1u, __ATOMIC_RELAXED, kScope) == S - 1;
    if (last) put<kScope>(&own->arrived, 0u);
    s_last = last;
  }
  __syncthreads();
  if (!s_last || w != 0) return;

  const uint32_t* rec = reinterpret_cast<const uint32_t*>(own->records + (lane < S ? lane : 0));
  best = Best{__uint_as_float(get(rec)), get(rec + 1)};
  mx = __uint_as_float(get(rec + 2));
  key = get(rec + 3);
  const uint64_t lo = get(rec + 4), hi = get(rec + 5);
  sum = __longlong_as_double((long long)(hi << 32 | lo));
  if (lane >= S) {
    best = Best{-INFINITY, kNone};
    mx = -INFINITY;
    key = kNone;
    sum = 0.0;
  }
  join();
  if (lane == 0) finish();
}

}  // namespace

struct nd_selector {
  uint32_t batch = 0;
  void* work = nullptr;  // nd_adjust_bytes(batch)
};

size_t nd_adjust_bytes(uint32_t batch) {
  return kCounterStride * 4 + (size_t)batch * sizeof(RowSpace);
}

hipError_t nd_launch_adjust(const float* logits, uint32_t batch, uint32_t vocab,
                            const nd_logit_adjust& p, const uint32_t* mask, float* out,
                            uint32_t* ids, double* logprobs, void* work, hipStream_t s,
                            const nd_select_advance* adv) {
  const uint32_t segments = (vocab + kSegment - 1) / kSegment;
  uint32_t* const rows_done = static_cast<uint32_t*>(work);
  // As few segments a workgroup as would let the GPU hold them all at once (three
  // workgroups to a CU, by their LDS) if a row's divided evenly, and as few workgroups
  // a row as that leaves, rounded up: up to twice as many as it holds.  With the logits
  // in the last-level cache, 100 rows of 8 segments take 14.1 us in 4 workgroups a row
  // (400 in all), 14.3 in 5, 15.5 in 8; 301 rows of 13 take 47.0 in 3 (903), 47.4 in 2,
  // 52.4 in 13.  From memory the latter take 53.7 in 3.
  const uint64_t held = 768, each = ((uint64_t)batch * segments + held - 1) / held;
  uint32_t S = (uint32_t)((segments + each - 1) / each);
  if (S > kMaxRecords) S = kMaxRecords;
  const bool xl = nd_xcd_local() && S > 1;
  auto kernel = !ids ? adjust_kernel<false, true, false>
                : xl ? (out ? adjust_kernel<true, true, true> : adjust_kernel<true, false, true>)
                     : (out ? adjust_kernel<true, true, false> : adjust_kernel<true, false, false>);
  hipLaunchKernelGGL(kernel, ids && xl ? dim3((batch + 7) / 8 * 8 * S) : dim3(S, batch),
                     dim3(kThreads), 0, s, logits, vocab, p, mask, out, ids, logprobs,
                     rows_done, reinterpret_cast<RowSpace*>(rows_done + kCounterStride),
                     adv ? *adv : nd_select_advance{}, batch, S);
  return hipGetLastError();
}

void nd_selector_release(nd_selector* w) {
  hipFree(w->work);
  delete w;
}

extern "C" {

nd_status nd_selector_create(nd_ctx* ctx, uint32_t batch, nd_selector** out) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  if (!out) return nd_fail(ctx, ND_ERR_INVALID, "out is NULL");
  *out = nullptr;
  if (batch == 0 || batch > 65535)
    return nd_fail(ctx, ND_ERR_INVALID, "nd_selector_create: 1..65535 rows, got %u", batch);
  ND_ON_DEVICE(ctx);
  nd_selector* w = new (std::nothrow) nd_selector();
  if (!w) return nd_fail(ctx, ND_ERR_NOMEM, "no host memory");
  w->batch = batch;
  hipError_t e = hipMalloc(&w->work, nd_adjust_bytes(batch));
  if (e == hipSuccess) e = hipMemsetAsync(w->work, 0, nd_adjust_bytes(batch), ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    nd_selector_release(w);
    return nd_hip_fail(ctx, e, "selection workspace");
  }
  if (!nd_hold(ctx->selectors, w)) {
    nd_selector_release(w);
    return nd_fail(ctx, ND_ERR_NOMEM, "no host memory");
  }
  *out = w;
  return ND_OK;
}

nd_status nd_selector_free(nd_ctx* ctx, nd_selector* w) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  if (!w) return ND_OK;
  if (!ctx->selectors.erase(w))
    return nd_fail(ctx, ND_ERR_INVALID, "workspace does not belong to context");
  ND_ON_DEVICE(ctx);
  ND_HIP(ctx, hipDeviceSynchronize());  // calls may have used any stream
  nd_selector_release(w);
  return ND_OK;
}

static nd_status check_adjust(nd_ctx* ctx, const nd_selector* w, uint32_t batch, uint32_t vocab,
                              const nd_logit_adjust* p) {
  if (!w || !ctx->selectors.count(const_cast<nd_selector*>(w)))
    return nd_fail(ctx, ND_ERR_INVALID, "workspace does not belong to context");
  if (batch > w->batch)
    return nd_fail(ctx, ND_ERR_INVALID, "%u rows, room for %u", batch, w->batch);
  if (vocab == 0 || vocab >= (1u << 31))
    return nd_fail(ctx, ND_ERR_INVALID, "vocabulary of %u ids", vocab);
  if (!p) return ND_OK;
  if ((p->bias_ids == nullptr) != (p->bias == nullptr))
    return nd_fail(ctx, ND_ERR_INVALID, "bias ids and values go together");
  if ((p->history && p->history_stride >= (1u << 31)) ||
      (p->bias_ids && p->bias_stride >= (1u << 31)))
    return nd_fail(ctx, ND_ERR_INVALID, "history and bias rows hold less than 2^31 entries");
  return ND_OK;
}

nd_status nd_select_adjusted_d(nd_ctx* ctx, nd_selector* w, const float* logits, uint32_t batch,
                               uint32_t vocab, const nd_logit_adjust* adjust, const uint32_t* mask,
                               float* out, uint32_t* ids, double* logprobs, void* stream) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  nd_status st = check_adjust(ctx, w, batch, vocab, adjust);
  if (st != ND_OK) return st;
  if (batch == 0) return ND_OK;
  if (!logits || (!ids != !logprobs) || (!ids && !out))
    return nd_fail(ctx, ND_ERR_INVALID,
                   "logits, and ids with log-probabilities or adjusted logits, must not be NULL");
  const nd_logit_adjust none{};
  ND_ON_DEVICE(ctx);
  ND_HIP(ctx, nd_launch_adjust(logits, batch, vocab, adjust ? *adjust : none, mask, out, ids,
                               logprobs, w->work, nd_pick_stream(ctx, stream), nullptr));
  return ND_OK;
}

nd_status nd_select_adjusted(nd_ctx* ctx, nd_selector* w, const float* logits, uint32_t batch,
                             uint32_t vocab, const nd_logit_adjust* adjust, const uint32_t* mask,
                             float* out, uint32_t* ids, double* logprobs) {
  if (!ctx) return nd_fail(nullptr, ND_ERR_BACKEND, "context is NULL");
  nd_status st = check_adjust(ctx, w, batch, vocab, adjust);
  if (st != ND_OK) return st;
  if (batch == 0) return ND_OK;
  if (!logits || (!ids != !logprobs) || (!ids && !out))
    return nd_fail(ctx, ND_ERR_INVALID,
                   "logits, and ids with log-probabilities or adjusted logits, must not be NULL");
  nd_logit_adjust h = adjust ? *adjust : nd_logit_adjust{};
  const size_t b = batch, lb = b * vocab * 4, mb = b * (((size_t)vocab + 31) / 32) * 4;
  // Every array of the call in one block: sources first, then results.
  struct Part {
    const void** at;
    size_t bytes;
  };
  const void *src = logits, *msrc = mask;
  Part parts[] = {{&src, lb},
                  {&msrc, mb},
                  {(const void**)&h.history, b * h.history_stride * 4},
                  {(const void**)&h.history_lengths, b * 4},
                  {(const void**)&h.prompt_lengths, b * 4},
                  {(const void**)&h.repetition, b * 4},
                  {(const void**)&h.presence, b * 4},
                  {(const void**)&h.frequency, b * 4},
                  {(const void**)&h.bias_ids, b * h.bias_stride * 4},
                  {(const void**)&h.bias, b * h.bias_stride * 4},
                  {(const void**)&h.bias_counts, b * 4}};
  auto a256 = [](size_t v) { return (v + 255) & ~size_t(255); };
  size_t total = a256(b * 8) + a256(b * 4);
  for (const Part& p : parts) total += *p.at ? a256(p.bytes) : 0;
  char* dev = nullptr;
  ND_ON_DEVICE(ctx);
  ND_HIP(ctx, hipMalloc(&dev, total));
  double* dlp = reinterpret_cast<double*>(dev);
  uint32_t* did = reinterpret_cast<uint32_t*>(dev + a256(b * 8));
  char* next = dev + a256(b * 8) + a256(b * 4);
  hipError_t e = hipSuccess;
  for (const Part& p : parts) {
    if (!*p.at) continue;
    if (e == hipSuccess && p.bytes)
      e = hipMemcpyAsync(next, *p.at, p.bytes, hipMemcpyHostToDevice, ctx->stream);
    *p.at = next;
    next += a256(p.bytes);
  }
  float* dl = static_cast<float*>(const_cast<void*>(src));
  if (e == hipSuccess)
    e = nd_launch_adjust(dl, batch, vocab, h, static_cast<const uint32_t*>(msrc), out ? dl : nullptr,
                         ids ? did : nullptr, dlp, w->work, ctx->stream, nullptr);
  if (e == hipSuccess && out) e = hipMemcpyAsync(out, dl, lb, hipMemcpyDeviceToHost, ctx->stream);
  if (e == hipSuccess && ids) e = hipMemcpyAsync(ids, did, b * 4, hipMemcpyDeviceToHost, ctx->stream);
  if (e == hipSuccess && ids)
    e = hipMemcpyAsync(logprobs, dlp, b * 8, hipMemcpyDeviceToHost, ctx->stream);
  const hipError_t es = hipStreamSynchronize(ctx->stream);
  hipFree(dev);
  ND_HIP(ctx, e);
  ND_HIP(ctx, es);
  return ND_OK;
}

}  // extern "C"
