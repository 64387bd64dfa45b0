// Selection of the experts of each token from its router logits by groups, with
// softmax or sigmoid scores and a bias that counts for the choice alone:
//   s = softmax(l) or 1 / (1 + exp(-l))
//   c = s + bias
//   group score: the largest c of the group, or the sum of its largest two
//   the KG groups of largest score stay; of their experts the K of largest c
//   w = s of the chosen, over their sum (+ 1e-20) if renormalize, times scale
// Ties go to the lower group and the lower expert; a NaN choice ranks last.
//
// The chosen ids are those of exact arithmetic. Without a bias (and with groups
// by their best expert) the choice is made on the logits, in whose order the
// scores are. Otherwise c is computed in 32 bits first, and where two values that
// the result depends on lie within the error of that, the token's choice is made
// again in 64 bits: seldom (a distance of some 1e-6 among values that lie 1e-2
// apart) but for equal logits with equal biases, so it need not be fast.
//
// One wave per token. A lane holds up to NV consecutive experts of one group (64
// lanes over the groups, rounded up to a power of two), so lane order is expert
// order and a group's lanes are neighbours. Each lane sorts its experts by c; a
// selection is then a maximum over the lanes' heads (DPP), a ballot whose lowest
// lane is the lowest expert, and a shift of that lane's list.
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
  static constexpr int kDead = INT_MIN;
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
  static constexpr long long kDead = LLONG_MIN;
  __device__ __forceinline__ static long long of(double v) {
    const long long b = __double_as_longlong(v + 0.0);
    return v != v ? LLONG_MIN + 1 : b ^ ((b >> 63) & 0x7fffffffffffffffll);
  }
  __device__ __forceinline__ static double value(long long k) {
    return __longlong_as_double(k ^ ((k >> 63) & 0x7fffffffffffffffll));
  }
};

template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ int dpp_key(int v) {
  return __builtin_amdgcn_update_dpp(v, v, kCtrl, kRowMask, 0xf, false);
}

template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ long long dpp_key(long long v) {
  const unsigned lo = dpp_key<kCtrl, kRowMask>(static_cast<int>(v));
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

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

template <typename F>
__device__ __forceinline__ F wave_sum_of(F v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

struct Place {
  int e0, n;     // this lane's experts: e0 .. e0 + n - 1
  int group;     // of this lane (may be past the last: n is 0 then)
  int width;     // lanes of a group
};

// The choice of one token, lane k < K of the wave getting the k-th expert. F float
// returns whether 32 bits leave it open (`exact`: the choice is made on the logits
// themselves, which leave nothing open); then nothing else is valid.
template <typename F, int NV>
__device__ __forceinline__ bool select(const GroupTopkArgs& a, const Place& p, const float (&l)[NV],
                                       const float (&bias)[NV], bool exact, float m, int lane,
                                       int* chosen) {
  typedef Key<F> KF;
  typedef typename KF::type I;
  // Error of c in 32 bits, relative to the largest score plus |c|: some 2^-22
  // from the score (the exponential, the sum, a division), 2^-24 from the sum
  // with the bias. Twice that separates two values; 1e-6 leaves a margin.
  F top = 1;
  I key[NV];
  unsigned idx = 0;  // the lane's experts, 4 bits each, in the order of key[]
  {
    F c[NV], sum = 0;
    if (exact) {
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = l[i];
    } else if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        c[i] = F(1) / (F(1) + exp_of(-static_cast<F>(l[i]))) + static_cast<F>(bias[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        c[i] = exp_of(static_cast<F>(l[i]) - static_cast<F>(m));
        sum += i < p.n ? c[i] : F(0);
      }
      top = F(1) / wave_sum_of(sum);
#pragma unroll
      for (int i = 0; i < NV; ++i) c[i] = c[i] * top + static_cast<F>(bias[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      key[i] = i < p.n ? KF::of(c[i]) : KF::kDead;
      idx |= static_cast<unsigned>(i) << (4 * i);
    }
  }
  // Insertion sort, largest first, the lower expert first among equals.
#pragma unroll
  for (int i = 1; i < NV; ++i)
#pragma unroll
    for (int j = i; j > 0; --j) {
      const bool swap = key[j] > key[j - 1];
      const I hi = swap ? key[j] : key[j - 1], lo = swap ? key[j - 1] : key[j];
      key[j - 1] = hi;
      key[j] = lo;
      const unsigned pair = (idx >> (4 * (j - 1))) & 0xffu;
      const unsigned turned = ((pair >> 4) | (pair << 4)) & 0xffu;
      idx ^= swap ? (pair ^ turned) << (4 * (j - 1)) : 0u;
    }

  bool open = false;
  auto near = [&](I hi, I lo) {  // hi >= lo
    if (sizeof(F) != sizeof(float) || exact || lo <= KF::kDead + 1) return false;
    const F x = KF::value(hi), y = KF::value(lo);
    return !(x - y > F(1e-6) * (top + fabs(x)));  // infinite ones too
  };
  if (a.KG < a.G) {
    I b1 = key[0], b2 = NV > 1 ? key[NV > 1 ? 1 : 0] : KF::kDead;
    for (int o = 1; o < p.width; o <<= 1) {
      const I x1 = __shfl_xor(b1, o, kWave), x2 = __shfl_xor(b2, o, kWave);
      const I lo = b1 > x1 ? x1 : b1;
      b2 = max(max(b2, x2), lo);
      b1 = max(b1, x1);
    }
    // A group's score as a key; a sum with a NaN, and of a single expert, as its best.
    I score = b1;
    if (a.top2 && b1 > KF::kDead + 1 && b2 > KF::kDead + 1)
      score = KF::of(KF::value(b1) + KF::value(b2));
    if (p.group >= a.G) score = KF::kDead;
    int rank = 0;
    I worst = 0, best_out = KF::kDead;  // of the kept, and of the others
    for (int g = 0; g < a.G; ++g) {
      const I other = lane_key(score, g * p.width);
      rank += other > score || (other == score && g < p.group) ? 1 : 0;
    }
    const bool kept = p.group < a.G && rank < a.KG;
    if (sizeof(F) == sizeof(float) && !exact) {
      worst = ~wave_max_key(kept ? ~score : KF::kDead);
      best_out = wave_max_key(!kept && p.group < a.G ? score : KF::kDead);
      // sums of two are of twice the error
      if (near(worst, best_out) ||
          (a.top2 && best_out > KF::kDead + 1 &&
           !(KF::value(worst) - KF::value(best_out) > F(4e-6) * (top + fabs(KF::value(worst))))))
        open = true;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = kept ? key[i] : KF::kDead;
  }

  I before = 0;
  int mine = 0;
  for (int k = 0; k <= a.K; ++k) {
    const I best = wave_max_key(key[0]);
    if (k > 0) open = open || near(before, best);
    before = best;
    if (k == a.K) break;
    const int win = __builtin_ctzll(__ballot(key[0] == best));
    const int e = __builtin_amdgcn_readlane(p.e0 + static_cast<int>(idx & 15u), win);
    mine = lane == k ? e : mine;
    const bool here = lane == win;
#pragma unroll
    for (int i = 0; i + 1 < NV; ++i) key[i] = here ? key[i + 1] : key[i];
    key[NV - 1] = here ? KF::kDead : key[NV - 1];
    idx = here ? idx >> 4 : idx;
  }
  *chosen = mine;
  return open;
}

template <int NV>
__global__ __launch_bounds__(kThreads) void group_topk_kernel(const GroupTopkArgs a, int width) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int t = blockIdx.x * (kThreads / kWave) + wave;
  if (t >= a.T) return;
  const int S = a.E / a.G;
  Place p;
  p.width = width;
  p.group = lane / width;
  const int first = (lane % width) * NV;
  p.n = p.group < a.G ? min(max(S - first, 0), NV) : 0;
  p.e0 = p.group * S + first;

  const float* row = a.logits + static_cast<size_t>(t) * a.E;
  float l[NV], bias[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    l[i] = i < p.n ? row[p.e0 + i] : 0.f;
    bias[i] = a.bias && i < p.n ? a.bias[p.e0 + i] : 0.f;
  }
  int mk = Key<float>::of(-INFINITY);
#pragma unroll
  for (int i = 0; i < NV; ++i) mk = i < p.n ? max(mk, Key<float>::of(l[i])) : mk;
  const float m = Key<float>::value(wave_max_key(mk));

  const bool exact = !a.bias && (!a.top2 || a.KG == a.G);
  int e = 0;
  if (select<float, NV>(a, p, l, bias, exact, m, lane, &e))
    select<double, NV>(a, p, l, bias, exact, m, lane, &e);

  // Lane k finishes the k-th weight from its logit.
  float w = 0.f;
  const float x = row[e];
  if (a.sigmoid) {
    w = 1.0f / (1.0f + expf(-x));
  } else {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += i < p.n ? expf(l[i] - m) : 0.f;
    w = expf(x - m) / wave_sum(s);
  }
  w = lane < a.K ? w : 0.f;
  if (a.renormalize) w /= wave_sum(w) + 1e-20f;
  w *= a.scale;
  if (lane < a.K) {
    const size_t at = static_cast<size_t>(t) * a.out_ld + lane;
    a.topk_w[at] = w;
    if (a.ids_int64)
      static_cast<int64_t*>(a.topk_ids)[at] = e;
    else
      static_cast<int32_t*>(a.topk_ids)[at] = e;
  }
}

}  // namespace

hipError_t launch_group_topk(const GroupTopkArgs& a, hipStream_t s) {
  if (a.T == 0) return hipSuccess;
  // Lanes of a group: 64 over the groups, rounded up to a power of two (G <= 64).
  int slots = 1;
  while (slots < a.G) slots *= 2;
  const int width = kWave / slots, per = (a.E / a.G + width - 1) / width;
  const int tokens = kThreads / kWave;
  const dim3 grid((a.T + tokens - 1) / tokens), block(kThreads);
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
