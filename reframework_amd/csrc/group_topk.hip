// Selection of the experts of each token from its router logits by groups, with
// softmax or sigmoid scores and a bias that counts for the choice alone:
//   s = softmax(l) or 1 / (1 + exp(-l))
//   c = s + bias
//   group score: the largest c of the group, or the sum of its largest two
//   the KG groups of largest score stay; of their experts the K of largest c
//   w = s of the chosen, over their sum (+ 1e-20) if renormalize, times scale
// Ties go to the lower group and the lower expert; a NaN choice ranks last.
//
// The chosen ids are those of 64-bit arithmetic. Without a bias (and with groups
// by their best expert) the choice is made on the logits, in whose order the
// scores are. Otherwise c is computed in 32 bits first, and where two values that
// the result depends on lie within the error of that, the token's choice is made
// again in 64 bits: seldom (a distance of some 1e-6 among values that lie 1e-2
// apart) but for equal logits with equal biases, so it need not be fast. What 64
// bits do not tell apart is a tie (sigmoid scores of logits over 37 are all 1).
//
// The error of 32 bits, which kScoreError, kRounding and their like cover (u = 2^-24):
//   e = exp(v), v = l - max <= 0: the difference, log2(e) and the product are off by
//     2.3 u |v| in all, the unit by 2 u, so e by (2.3 |v| + 2) u: at most 2.9 u of the largest
//     e, as |v| exp(v) <= 0.37
//   the sum of the e: 2 u and 2.3 u times the mean of |v| by e, which is at most 3.4 for 256
//     experts, so 9.9 u; and u for each of its additions, 7 in a lane and 6 over the lanes
//     (rows of 16 lanes: 15 and 4); its reciprocal u
//   the difference of two scores: (9.9 + 13 + 1) u from the sum, common to both; 2.9 u and
//     u from their products each: 31.7 u = 1.9e-6 of the largest score (rows: 37.7 u =
//     2.25e-6); of two sums of two scores twice that
//   sigmoid scores: 2 u from the reciprocal, u from 1 + e, less than that from e: below
//     5 u each
//   adding the bias: u |c|; the sum of two choices: u of it; the test's own difference: u
// A distance is tested against the sum of both sides' errors, so each side's is half.
//
// One wave per token. A lane holds up to NV consecutive experts of one group (64
// lanes over the groups, rounded up to a power of two), so lane order is expert
// order and a group's lanes are neighbours. Each lane sorts its experts by c; a
// selection is then a maximum over the lanes' heads (DPP), a ballot whose lowest
// lane is the lowest expert, and a shift of that lane's list. Bound by that chain of
// instructions: 4.2 us for 8 tokens of 160 experts, 4 for 999 of 64, of which a launch is
// 2.5; the bytes of 16384 tokens of 256 experts take 3.8, the kernel of many tokens
// below 13 (1.4 TB/s).
#include <climits>

#include "common.h"

namespace moe355 {
namespace {

constexpr int kThreads = 256;

// Ordered integers of a choice: larger value, larger key; +0 and -0 alike, NaN
// below -infinity, and kDead (no expert) below NaN.
template <typename F>
struct Key;

template <>
struct Key<float> {
  typedef int type;
  static constexpr int kDead = INT_MIN, kFirst = INT_MIN + 32;  // keys from kFirst on are of numbers
  __device__ __forceinline__ static int of(float v) {
    const int b = __float_as_int(v + 0.f);
    return v != v ? INT_MIN + 1 : b ^ ((b >> 31) & 0x7fffffff);
  }
  __device__ __forceinline__ static float value(int k) {
    return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
  }
};

template <>
struct Key<double> {
  typedef long long type;
  static constexpr long long kDead = LLONG_MIN, kFirst = LLONG_MIN + 2;
  __device__ __forceinline__ static long long of(double v) {
    const long long b = __double_as_longlong(v + 0.0);
    return v != v ? LLONG_MIN + 1 : b ^ ((b >> 63) & 0x7fffffffffffffffll);
  }
  __device__ __forceinline__ static double value(long long k) {
    return __longlong_as_double(k ^ ((k >> 63) & 0x7fffffffffffffffll));
  }
};

// v of the lane that the DPP control names; kDead, which a maximum ignores, in lanes
// without a source (as its identity lets the compiler fold the move into v_max_i32).
template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ int dpp_key(int v) {
  return __builtin_amdgcn_update_dpp(INT_MIN, v, kCtrl, kRowMask, 0xf, false);
}

template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ long long dpp_key(long long v) {
  // lanes without a source get INT_MIN : 0, which is kDead
  const unsigned lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRowMask, 0xf, false);
  const unsigned hi = dpp_key<kCtrl, kRowMask>(static_cast<int>(v >> 32));
  return static_cast<long long>((static_cast<unsigned long long>(hi) << 32) | lo);
}

__device__ __forceinline__ int lane_key(int v, int lane) {
  return __builtin_amdgcn_readlane(v, lane);
}

__device__ __forceinline__ long long lane_key(long long v, int lane) {
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
  const unsigned hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
  return static_cast<long long>((static_cast<unsigned long long>(hi) << 32) | lo);
}

template <typename I>
__device__ __forceinline__ I wave_max_key(I v) {
  v = max(v, dpp_key<0x111>(v));       // row_shr 1, 2, 4, 8, then the rows' last lanes
  v = max(v, dpp_key<0x112>(v));
  v = max(v, dpp_key<0x114>(v));
  v = max(v, dpp_key<0x118>(v));
  v = max(v, dpp_key<0x142, 0xa>(v));
  v = max(v, dpp_key<0x143, 0xc>(v));
  return lane_key(v, kWave - 1);
}

// exp(v) for the choice: 32 bits on the transcendental unit (about 2^-23 of the result
// per unit of |v|, which the test for near values covers), or exactly enough.
__device__ __forceinline__ float exp_of(float v) {
  return __builtin_amdgcn_exp2f(v * 1.4426950408889634f);
}
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
// e * top + bias in two roundings: as one (where the compiler saw fit, which was not the
// same for all places of a lane's list) equal choices differed in their last bit.
template <typename F>
__device__ __forceinline__ F choice_of(F e, F top, F bias) {
#pragma clang fp contract(off)
  const F score = e * top;
  return score + bias;
}
__device__ __forceinline__ float inverse_of(float v) { return __builtin_amdgcn_rcpf(v); }
__device__ __forceinline__ double inverse_of(double v) { return 1.0 / v; }

// Sum over the wave, the same in every lane.
__device__ __forceinline__ float wave_sum_of(float v) {
  const auto add = [](float x, int moved) { return x + __int_as_float(moved); };
  const auto bits = [](float x) { return __float_as_int(x); };
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x111, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x112, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x114, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x118, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x142, 0xa, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x143, 0xc, 0xf, false));
  return __int_as_float(__builtin_amdgcn_readlane(bits(v), kWave - 1));
}

__device__ __forceinline__ double wave_sum_of(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

struct Place {
  int e0, n;     // this lane's experts: e0 .. e0 + n - 1
  int group;     // of this lane (may be past the last: n is 0 then)
  int width;     // lanes of a group
};

// Largest two of b1 >= b2 over runs of `width` lanes (a power of two up to 64), in all
// of them.
template <typename I>
__device__ __forceinline__ void top2_of_group(I& b1, I& b2, int width) {
  const auto merge = [&](I x1, I x2) {
    const I lo = min(b1, x1);
    b1 = max(b1, x1);
    b2 = max(max(b2, x2), lo);
  };
  if (width >= 2) merge(dpp_key<0xb1>(b1), dpp_key<0xb1>(b2));      // quad_perm 1 0 3 2
  if (width >= 4) merge(dpp_key<0x4e>(b1), dpp_key<0x4e>(b2));      // quad_perm 2 3 0 1
  if (width >= 8) merge(dpp_key<0x141>(b1), dpp_key<0x141>(b2));    // row_half_mirror
  if (width >= 16) merge(dpp_key<0x140>(b1), dpp_key<0x140>(b2));   // row_mirror
  for (int o = 16; o < width; o <<= 1) merge(__shfl_xor(b1, o, kWave), __shfl_xor(b2, o, kWave));
}

// Whether the groups that are kept are left open: whether a kept one, less its error, does
// not lie above each of the others, plus theirs. A group's error grows with the
// choices that were added for it, not with what is left of them: two that
// cancel leave a small score and the error of large ones. Infinite scores are
// exact. max_of: the maximum over the token's lanes.
template <typename KF, typename F, typename M>
__device__ __forceinline__ bool group_open(typename KF::type score, F error, bool kept, bool group,
                                           M max_of) {
  typedef typename KF::type I;
  const F v = KF::value(score);
  error = fabs(v) < INFINITY ? error : F(0);
  const bool real = score >= KF::kFirst;  // no NaN
  const I low = real ? KF::of(v - error) : score, high = real ? KF::of(v + error) : score;
  const I worst = ~max_of(kept ? ~low : KF::kDead), best = max_of(group && !kept ? high : KF::kDead);
  return best >= KF::kFirst && !(KF::value(worst) > KF::value(best));
}

// The error of a score relative to the token's largest, of a choice relative to its own
// magnitude (a group's: to those of the choices in it).
constexpr float kScoreError = 1e-6f, kRounding = 2.5e-7f;

// The choice of one token into chosen[0..K) (LDS). F float returns whether 32 bits
// leave it open (`exact`: the choice is made on the logits themselves, which leave
// nothing open); then nothing else is valid.
template <typename F, int NV>
__device__ __forceinline__ bool select(const GroupTopkArgs& a, const Place& p, const float (&l)[NV],
                                       const float (&bias)[NV], bool exact, float m, int lane,
                                       int* chosen) {
  typedef Key<F> KF;
  typedef typename KF::type I;
  F top = 1;  // a score is at most this
  I key[NV];
  int idx[NV];
  {
    F c[NV], sum = 0;
    if (exact) {
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = l[i];
    } else if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        c[i] = inverse_of(F(1) + exp_of(-static_cast<F>(l[i]))) + static_cast<F>(bias[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        c[i] = exp_of(static_cast<F>(l[i]) - static_cast<F>(m));
        sum += i < p.n ? c[i] : F(0);
      }
      top = F(1) / wave_sum_of(sum);
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = choice_of<F>(c[i], top, static_cast<F>(bias[i]));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      key[i] = i < p.n ? KF::of(c[i]) : KF::kDead;
      idx[i] = i;
    }
  }
  // Insertion sort, largest first, the lower expert first among equals; then the
  // experts' places in one register, 4 bits each.
#pragma unroll
  for (int i = 1; i < NV; ++i)
#pragma unroll
    for (int j = i; j > 0; --j) {
      const bool swap = key[j] > key[j - 1];
      const I hi = swap ? key[j] : key[j - 1], lo = swap ? key[j - 1] : key[j];
      const int ih = swap ? idx[j] : idx[j - 1], il = swap ? idx[j - 1] : idx[j];
      key[j - 1] = hi;
      key[j] = lo;
      idx[j - 1] = ih;
      idx[j] = il;
    }
  unsigned list = 0;
#pragma unroll
  for (int i = NV - 1; i >= 0; --i) list = (list << 4) | static_cast<unsigned>(idx[i]);

  // Whether hi >= lo lie too near each other for 32 bits (of a lo twice as far from 0
  // as hi the rounding is below the distance).
  auto near = [&](I hi, I lo) {
    const F x = KF::value(hi), y = KF::value(lo);
    return lo >= KF::kFirst &&
           !(x - y > F(2 * kScoreError) * top + F(2 * kRounding) * fabs(x));  // infinite ones too
  };
  constexpr bool kTest = sizeof(F) == sizeof(float);
  bool open = false;
  if (a.KG < a.G) {
    I b1 = key[0], b2 = NV > 1 ? key[NV > 1 ? 1 : 0] : KF::kDead;
    top2_of_group(b1, b2, p.width);
    // A group's score as a key; with a NaN, and of a single expert, its best.
    const bool two = a.top2 && b1 > KF::kDead + 1 && b2 > KF::kDead + 1;
    I score = two ? KF::of(KF::value(b1) + KF::value(b2)) : b1;
    if (p.group >= a.G) score = KF::kDead;
    int rank = 0;
    for (int g = 0; g < a.G; ++g) {
      const I other = lane_key(score, g * p.width);
      rank += other > score || (other == score && g < p.group) ? 1 : 0;
    }
    const bool kept = p.group < a.G && rank < a.KG;
    if (kTest && !exact) {
      const F size = fabs(KF::value(b1)) + (two ? fabs(KF::value(b2)) : F(0));
      const F error = F(two ? 2 * kScoreError : kScoreError) * top + F(kRounding) * size;
      open = group_open<KF>(score, error, kept, p.group < a.G, [](I v) { return wave_max_key(v); });
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = kept ? key[i] : KF::kDead;
  }

  I mine = KF::kDead, best = KF::kDead;  // lane k: the k-th value; the one after the last
  for (int k = 0; k <= a.K; ++k) {
    best = wave_max_key(key[0]);
    if (k == a.K) break;
    if (kTest) mine = lane == k ? best : mine;
    if (lane == static_cast<int>(__builtin_ctzll(__ballot(key[0] == best)))) {
      chosen[k] = p.e0 + static_cast<int>(list & 15u);
      list >>= 4;
#pragma unroll
      for (int i = 0; i + 1 < NV; ++i) key[i] = key[i + 1];
      key[NV - 1] = KF::kDead;
    }
  }
  if (kTest && !exact) {
    const I down = __shfl_down(mine, 1, kWave);
    const I next = lane == a.K - 1 ? best : down;
    open = open || __ballot(lane < a.K && near(mine, next)) != 0;
  }
  return open;
}

// This wave's place among the experts: `lanes` lanes in all, `width` per group.
template <int NV>
__device__ __forceinline__ Place place_of(const GroupTopkArgs& a, int lane, int width) {
  Place p;
  p.width = width;
  p.group = lane / width;
  const int first = (lane % width) * NV, S = a.E / a.G;
  p.n = p.group < a.G ? min(max(S - first, 0), NV) : 0;
  p.e0 = p.group * S + first;
  return p;
}

// This lane's logits and biases, 16 bytes a load where groups are whole ones (`vec`): with
// 4 bytes a load every instruction of a wave would touch a line per lane.
template <int NV>
__device__ __forceinline__ void load_experts(const float* src, const Place& p, bool vec, float (&v)[NV]) {
  if (NV % 4 == 0 && vec) {
#pragma unroll
    for (int i = 0; i < NV; i += 4) {
      const f32x4 x = i < p.n ? *reinterpret_cast<const f32x4*>(src + p.e0 + i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4 && i + j < NV; ++j) v[i + j] = x[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = i < p.n ? src[p.e0 + i] : 0.f;
  }
}

template <int NV>
__device__ __forceinline__ void load_token(const GroupTopkArgs& a, const Place& p, const float* row,
                                           float (&l)[NV], float (&bias)[NV]) {
  load_experts<NV>(row, p, a.vec, l);
  if (a.bias) {
    load_experts<NV>(a.bias, p, a.vec, bias);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) bias[i] = 0.f;
  }
}

__device__ __forceinline__ bool by_logit(const GroupTopkArgs& a) {
  return !a.bias && (!a.top2 || a.KG == a.G);
}

// The k-th weight and id of token t.
__device__ __forceinline__ void store_choice(const GroupTopkArgs& a, int t, int k, float w, int e) {
  const size_t at = static_cast<size_t>(t) * a.out_ld + k;
  a.topk_w[at] = w;
  if (a.ids_int64)
    static_cast<int64_t*>(a.topk_ids)[at] = e;
  else
    static_cast<int32_t*>(a.topk_ids)[at] = e;
}

template <int NV>
__global__ __launch_bounds__(kThreads) void group_topk_kernel(const GroupTopkArgs a, int width) {
  __shared__ int chosen[kThreads / kWave][MOE355_MAX_GROUPED_TOPK];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int t = blockIdx.x * (kThreads / kWave) + wave;
  if (t >= a.T) return;
  const Place p = place_of<NV>(a, lane, width);
  const float* row = a.logits + static_cast<size_t>(t) * a.E;
  float l[NV], bias[NV];
  load_token<NV>(a, p, row, l, bias);
  int mk = Key<float>::of(-INFINITY);
#pragma unroll
  for (int i = 0; i < NV; ++i) mk = i < p.n ? max(mk, Key<float>::of(l[i])) : mk;
  const float m = Key<float>::value(wave_max_key(mk));

  if (select<float, NV>(a, p, l, bias, by_logit(a), m, lane, chosen[wave]))
    select<double, NV>(a, p, l, bias, by_logit(a), m, lane, chosen[wave]);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

  // Lane k finishes the k-th weight from its logit.
  float w;
  const int e = lane < a.K ? chosen[wave][lane] : 0;
  const float x = row[e];
  if (a.sigmoid) {
    w = 1.0f / (1.0f + expf(-x));
  } else {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += i < p.n ? exp_of(l[i] - m) : 0.f;
    w = expf(x - m) / wave_sum_of(s);
  }
  w = lane < a.K ? w : 0.f;
  if (a.renormalize) w /= wave_sum_of(w) + 1e-20f;
  w *= a.scale;
  if (lane < a.K) store_choice(a, t, lane, w, e);
}

// ---------------------------------------------------------------- many tokens
// The kernel above is bound by its instructions (621 of a wave per token at 256
// experts of 8 groups, top-8; this one's 261). For many tokens a row of 16 lanes takes a token, four
// to a wave, so that the maxima over lanes are four DPP rotations for four tokens;
// and a key carries its place i among its lane's experts in its last 4 bits (as 15 -
// i), so that a comparison of the sort is one maximum and one minimum. Keys are then
// cut to 2^-19 of the value: choices nearer than that are left to `select`, as
// are those within the error of 32 bits. Logits whose last 4 bits are 0 (16-bit
// values) lose nothing.
constexpr int kRow = 16;
constexpr int kRowTopk = 8;  // largest K
constexpr float kRowScoreError = 1.2e-6f;             // its lanes' sums are longer
constexpr float kRowRounding = kRounding + 0x1p-19f;  // with the cut of the keys

__device__ __forceinline__ int row_max_key(int v) {
  v = max(v, dpp_key<0x121>(v));  // row_ror 1, 2, 4, 8
  v = max(v, dpp_key<0x122>(v));
  v = max(v, dpp_key<0x124>(v));
  return max(v, dpp_key<0x128>(v));
}

__device__ __forceinline__ float row_sum(float v) {
  const auto moved = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl.value, 0xf, 0xf, false));
  };
  v += moved(v, std::integral_constant<int, 0x121>());
  v += moved(v, std::integral_constant<int, 0x122>());
  v += moved(v, std::integral_constant<int, 0x124>());
  return v + moved(v, std::integral_constant<int, 0x128>());
}

// key of the lane `kLanes` further in the row.
template <int kLanes>
__device__ __forceinline__ int row_ahead(int v) {
  return __builtin_amdgcn_update_dpp(v, v, 0x120 + (kRow - kLanes), 0xf, 0xf, false);
}

template <int kFrom, int kTo, typename F>
__device__ __forceinline__ void unroll(F f) {
  if constexpr (kFrom < kTo) {
    f(std::integral_constant<int, kFrom>());
    unroll<kFrom + 1, kTo>(f);
  }
}

// NV experts per lane of a row (4 NW), NW per lane of the wave that a token left open
// is chosen by.
template <int NW>
__global__ __launch_bounds__(kThreads) void group_topk_rows_kernel(const GroupTopkArgs a, int width) {
  constexpr int NV = 4 * NW;
  constexpr int kList = NV < kRowTopk + 1 ? NV : kRowTopk + 1;  // of a lane that can be chosen
  typedef Key<float> KF;
  __shared__ int chosen[kThreads / kWave][MOE355_MAX_GROUPED_TOPK];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int sub = lane & (kRow - 1);
  const int t0 = (blockIdx.x * (kThreads / kWave) + wave) * (kWave / kRow);
  if (t0 >= a.T) return;
  const int t = min(t0 + lane / kRow, a.T - 1);  // rows past the last repeat it
  const int wr = width / 4;                      // lanes of a group
  const Place p = place_of<NV>(a, sub, wr);
  const float* row = a.logits + static_cast<size_t>(t) * a.E;
  float l[NV], bias[NV];
  load_token<NV>(a, p, row, l, bias);

  const bool exact = by_logit(a);
  int mk = KF::of(-INFINITY), bits = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    mk = i < p.n ? max(mk, KF::of(l[i])) : mk;
    bits |= __float_as_int(l[i]);
  }
  const float m = KF::value(row_max_key(mk));
  float top = 1.f, sum = 0.f;
  int key[NV];
  {
    float c[NV];
    if (exact && a.sigmoid) {
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = l[i];
    } else if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = inverse_of(1.f + exp_of(-l[i])) + bias[i];
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        c[i] = exp_of(l[i] - m);
        sum += i < p.n ? c[i] : 0.f;
      }
      sum = row_sum(sum);
      top = 1.f / sum;
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = exact ? l[i] : choice_of(c[i], top, bias[i]);
    }
    if (exact) top = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      key[i] = i < p.n ? max(KF::of(c[i]), INT_MIN + 16) & ~15 | (15 - i) : KF::kDead;
  }
  // A key without its place, cut towards zero (the bits of a negative value are
  // inverted in its key, and those of -infinity have to stay), its value, and whether two
  // lie too near each other: 2^-19 of each from the cut, and what `select` allows.
  const auto placeless = [](int k) { return (k & ~15) | ((k >> 31) & 15); };
  const auto cut = [&](int k) { return KF::value(placeless(k)); };
  const bool lossless = exact && row_max_key(bits & 15) == 0;
  const auto near = [&](int hi, int lo) {
    const float x = cut(hi), y = cut(lo);
    return lo >= KF::kFirst && !(x - y > 2 * kRowScoreError * top + 3 * kRowRounding * fabsf(x));
  };

  // Largest first (odd-even merge sort of the NV keys).
  unroll<0, 4>([&](auto lp) {
    constexpr int P = 1 << decltype(lp)::value;
    if constexpr (P < NV) {
      unroll<0, decltype(lp)::value + 1>([&](auto lk) {
        constexpr int K2 = P >> decltype(lk)::value;
#pragma unroll
        for (int j = K2 % P; j + K2 < NV; j += 2 * K2)
#pragma unroll
          for (int i = 0; i < K2; ++i)
            if (i + j + K2 < NV && (i + j) / (2 * P) == (i + j + K2) / (2 * P)) {
              const int hi = max(key[i + j], key[i + j + K2]);
              key[i + j + K2] = min(key[i + j], key[i + j + K2]);
              key[i + j] = hi;
            }
      });
    }
  });

  bool open = false;
  if (a.KG < a.G) {
    int b1 = key[0], b2 = key[1];
    top2_of_group(b1, b2, wr);
    const bool two = a.top2 && b2 >= KF::kFirst;
    int score = two ? KF::of(cut(b1) + cut(b2)) : placeless(b1);
    if (p.group >= a.G) score = KF::kDead;
    int rank = 0;  // groups above this one
    unroll<1, kRow>([&](auto d) {
      constexpr int D = decltype(d)::value;
      if (D % wr) return;
      const int other = row_ahead<D>(score);
      const bool first = sub + D >= kRow;  // `other` is of a lower group
      rank += other > score || (other == score && first) ? 1 : 0;
    });
    const bool kept = p.group < a.G && rank < a.KG;
    if (!lossless) {
      const float size = fabsf(cut(b1)) + (two ? fabsf(cut(b2)) : 0.f);
      const float error = (two ? 2 : 1) * kRowScoreError * top + kRowRounding * size;
      open = group_open<KF>(score, error, kept, p.group < a.G, [](int v) { return row_max_key(v); });
    }
#pragma unroll
    for (int i = 0; i < kList; ++i) key[i] = kept ? key[i] : KF::kDead;
  }

  // Of equal values the first lane of the row is chosen, and in it the first place.
  int* const list = chosen[wave] + (lane & ~(kRow - 1)) / kRow * kRowTopk;
  int mine = KF::kDead, next = KF::kDead;  // lane k: the k-th value, and the one after it
  unroll<0, kRowTopk + 1>([&](auto kc) {
    constexpr int k = decltype(kc)::value;
    if (k > a.K) return;
    const int head = key[0] & ~15, best = row_max_key(head);
    next = sub == k - 1 ? best : next;
    if constexpr (k < kRowTopk) {
      if (k == a.K) return;
      mine = sub == k ? best : mine;
      const unsigned long long at = __ballot(head == best);
      const unsigned half = lane < 32 ? static_cast<unsigned>(at) : static_cast<unsigned>(at >> 32);
      if (sub == __builtin_ctz(half >> (lane & 16))) {
        list[k] = p.e0 + 15 - (key[0] & 15);
        // What is left of the lane's list can be chosen kRowTopk - k times more.
        constexpr int kLeft = NV < kRowTopk + 1 - k ? NV : kRowTopk + 1 - k;
#pragma unroll
        for (int i = 0; i + 1 < kLeft; ++i) key[i] = key[i + 1];
        key[kLeft - 1] = KF::kDead;
      }
    }
  });
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  int e = sub < a.K ? list[sub] : 0;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  float x = row[e];
  if (!lossless) {
    // What is chosen from what is not lies apart even as cut; the order of what is
    // chosen, where the cut values are near, by the whole ones.
    float c = x;
    if (!exact) {
      const float b = a.bias ? a.bias[e] : 0.f;
      c = a.sigmoid ? inverse_of(1.f + exp_of(-x)) + b : choice_of(exp_of(x - m), top, b);
    }
    const float after = __int_as_float(row_ahead<1>(__float_as_int(c)));
    const int e_after = row_ahead<1>(e);
    const bool ordered = exact ? c > after || (c == after && e < e_after)
                               : c - after > 2 * kRowScoreError * top + 2 * kRounding * fabsf(c);
    open = open || (sub < a.K && near(mine, next) && (sub == a.K - 1 || !ordered));
  }

  // Tokens left open, one after the other by the whole wave: on the logits where those
  // decide, else in 64 bits at once (32 bits first took 2 us longer, as in a launch of
  // thousands of tokens one is open in 64 bits too).
  const unsigned long long left = __ballot(open);
  for (int r = 0; r < kWave / kRow; ++r) {
    if (!((left >> (kRow * r)) & 0xffffull) || t0 + r >= a.T) continue;
    const Place pw = place_of<NW>(a, lane, width);
    float lw[NW], bw[NW];
    load_token<NW>(a, pw, a.logits + static_cast<size_t>(t0 + r) * a.E, lw, bw);
    const float mw = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m), kRow * r));
    if (exact)
      select<float, NW>(a, pw, lw, bw, true, mw, lane, chosen[wave]);
    else
      select<double, NW>(a, pw, lw, bw, false, mw, lane, chosen[wave]);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (lane / kRow == r && sub < a.K) {
      e = chosen[wave][sub];
      x = row[e];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }

  float w = a.sigmoid ? 1.0f / (1.0f + expf(-x)) : expf(x - m) / sum;
  w = sub < a.K ? w : 0.f;
  if (a.renormalize) w /= row_sum(w) + 1e-20f;
  w *= a.scale;
  if (sub < a.K && t0 + lane / kRow < a.T) store_choice(a, t, sub, w, e);
}

// Tokens from which four to a wave are faster (256 experts of 8 groups with a bias, one /
// four to a wave, us a call in a graph: 1024 tokens 4.7 / 9.3, 4096 9.1 / 9.6, 6144 12.0 /
// 10.8, 16384 19 / 13.8, 32768 32 / 20.8; below, the longer chain of a wave's
// instructions shows).
constexpr int kRowTokens = 6144;

}  // namespace

hipError_t launch_group_topk(const GroupTopkArgs& args, hipStream_t s) {
  if (args.T == 0) return hipSuccess;
  GroupTopkArgs a = args;
  const auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  a.vec = a.E / a.G % 4 == 0 && aligned(a.logits) && aligned(a.bias);
  // Lanes of a group: 64 over the groups, rounded up to a power of two (G <= 64).
  int slots = 1;
  while (slots < a.G) slots *= 2;
  const int width = kWave / slots, per = (a.E / a.G + width - 1) / width;
  if (a.T >= kRowTokens && slots <= kRow && per <= 4 && a.K <= kRowTopk) {
    const int tokens = kThreads / kRow;
    const dim3 rows((a.T - 1) / tokens + 1), threads(kThreads);
    if (per <= 1)
      group_topk_rows_kernel<1><<<rows, threads, 0, s>>>(a, width);
    else if (per <= 2)
      group_topk_rows_kernel<2><<<rows, threads, 0, s>>>(a, width);
    else
      group_topk_rows_kernel<4><<<rows, threads, 0, s>>>(a, width);
    return hipGetLastError();
  }
  const int tokens = kThreads / kWave;
  const dim3 grid((a.T - 1) / tokens + 1), block(kThreads);
  if (per <= 1)
    group_topk_kernel<1><<<grid, block, 0, s>>>(a, width);
  else if (per <= 2)
    group_topk_kernel<2><<<grid, block, 0, s>>>(a, width);
  else if (per <= 4)
    group_topk_kernel<4><<<grid, block, 0, s>>>(a, width);
  else
    group_topk_kernel<8><<<grid, block, 0, s>>>(a, width);
  return hipGetLastError();
}

}  // namespace moe355
