// What the kernels of the distillation (distill.cu, distill_stream.cuh) have in common: the list of a row, the loss, and the factors of the
// gradient.
#pragma once
#include "row_types.cuh"
#include "launch.h"
#include <cfloat>
#include <cmath>

namespace ds41 {
namespace {

enum DistillMode { kDistillLoss, kDistillGrad, kDistillBoth };
constexpr int kDisGroup = 4;                  // vectors of a thread that are copied, waited for and worked on together
constexpr int kDisGroups = 5;                 // (the last for the one vector more of a slice that does not begin on a vector)
constexpr int kDisVectors = kDisGroup * (kDisGroups - 1);
constexpr int kDisTop = DS41_B200_DISTILL_MAX_TOP;
constexpr int kDisOwn = kDisTop / 32;         // entries of a lane
constexpr double kDisMost = 1.01;             // what a list's probabilities may add up to: 1, and the rounding of stored values

struct DistillParams {
  ds41_b200_distill_args a;
  int in_place;                               // grad is logits
  int slice, team;                            // ids of a CTA (a multiple of 32), CTAs of a row
  int groups;                                 // of a row that is streamed
  float log2e_t;                              // log2(e) / T
  double inverse_t;                           // 1 / T
};

__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait(int left) {
  switch (left) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
  }
}
template <int kBarrier, int kCount> __device__ __forceinline__ void barrier_of() {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"n"(kBarrier), "n"(kCount) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {   // 2 ulp; 0 for -inf and below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The power of (x - m) c, with c = log2(e) / T, as that of x c - r with r = m c rounded: one fused multiply-add, its argument as exact, if
// the rounding of r is made good for once a row.  That rounding is up to 2^-24 |r|, so the shortcut is for |r| below 2^24, where its power lies
// between 0.7 and 1.42; at 2^31 it would be infinite or 0.  Beyond (logits past 1.2e7 T: masked places, a type's lowest values) the power
// is that of (x - m) c.  (The rounding is asked for by name: what takes r must not get the product that it was rounded from.)
constexpr float kDisNear = 16777216.f;
__device__ __forceinline__ bool near_exponent(float r) { return fabsf(r) < kDisNear; }
__device__ __forceinline__ float rounded_product(float m, float c) { return __fmul_rn(m, c); }
__device__ __forceinline__ float excess(float m, float c, float r) { return near_exponent(r) ? fmaf(m, c, -r) : 0.f; }
// What a sum of such powers relative to m is multiplied by where the maximum rises to `top`: it stands relative to r where that is near, and
// to the product itself where it is not, whichever side either is on.  (The maximum before the first has r = -inf.)
__device__ __forceinline__ float rise(float m, float r, float top, float top_r, float c) {
  const float down = near_exponent(top_r) ? (near_exponent(r) ? __fsub_rn(r, top_r) : fmaf(m, c, -top_r))
                                          : (near_exponent(r) ? -fmaf(top, c, -r) : (m - top) * c);
  return exp2_approx(down);
}

// Out of line, once each: what runs a few times a row shall not push the loops out of the instruction cache.
__device__ __noinline__ double exp_of(double x) { return exp(x); }
__device__ __noinline__ double log_of(double x) { return log(x); }
__device__ __noinline__ double over(double x, double y) { return x / y; }

// What is known of a row besides its ids outside the list, the same in every CTA of the team.
struct DistillRow {
  float scale;
  int reject;                                 // of the list
  float4 stats;                               // of the forward pass, in the gradient's
  float zmax, share;                          // largest logit of the entries that count; sum of exp((z - zmax) / T), an entry per id
  double kept, entropy, rest;                 // with w the unnormalised weights: sum of w, of w (ln w - (z - zmax) / T); 1 - the list's sum
  double inverse, inverse_rest;               // 1 / (sum of w), 1 / (that + rest)
};

// Where a row's list lies in shared memory.
struct DistillList { double *weights; int *ids; float *zs; };

template <int kMode> __device__ __forceinline__ bool skipped(const DistillRow &r) { return kMode != kDistillLoss && r.scale == 0.f; }
template <int kMode> __device__ __forceinline__ float row_scale_of(const DistillParams &p, int row) {
  return kMode != kDistillLoss && p.a.row_scale && row < p.a.rows ? load_input(p.a.row_scale + row) : 1.f;
}

// A row's slice as one of its CTA's threads sees it, which takes vectors t, t + kCompute, ... of it ("at" 0, kCompute, ...).  Place 0 is
// where the vector of the slice's first id begins.
template <class T, int kCompute>
struct DistillSlice {
  static constexpr int kVec = RowType<T>::kVec;
  const T *x;
  const uint4 *from;                          // the thread's first vector
  int lead, vecs;                             // vectors of the slice
  int mine, wholes;                           // its vectors are the slice's below `mine`, and hold no other slice's ids below `wholes`
  bool cut;                                   // ... but for the first one
  __device__ __forceinline__ DistillSlice(const DistillParams &p, int row, int begin, int len, int t) {
    x = static_cast<const T *>(p.a.logits) + size_t(row) * size_t(p.a.logits_stride) + begin;
    lead = int((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % kVec);
    vecs = (lead + len + kVec - 1) / kVec;
    from = reinterpret_cast<const uint4 *>(x - lead) + t;
    mine = vecs - t; wholes = (lead + len) / kVec - t;
    cut = lead && t == 0;
  }
  __device__ __forceinline__ bool whole(int at) const { return at < wholes && !(cut && at == 0); }
  __device__ __forceinline__ bool any_partial() const { return cut || wholes < mine; }
};

// A vector that is not whole comes and goes by its ids, `from` .. `to`.
template <class T>
__device__ __noinline__ void copy_ids(T *to_first, const T *from_first, int from, int to) {
#pragma unroll 1
  for (int i = from; i < to; ++i) to_first[i] = from_first[i];
}

// A row's list, by one warp: the entries that count, one per id, and what they amount to.
template <class T, int kMode>
__device__ __forceinline__ void gather_list(const DistillParams &p, int row, DistillRow &r, const DistillList &list_of, int lane) {
  using R = RowType<T>;
  const ds41_b200_distill_args &a = p.a;
  const int top_room = (a.top + 3) & ~3;
  double *const w_list = list_of.weights;
  int *const id_list = list_of.ids;
  float *const z_list = list_of.zs;
  const T *whole = static_cast<const T *>(a.logits) + size_t(row) * size_t(a.logits_stride);
  const uint32_t *mask = a.mask ? a.mask + size_t(row) * size_t(a.mask_stride) : nullptr;
  const int own = (a.top + 31) / 32;
  // the ids and values, then the logits they name: as many on their way at a time as there are
#pragma unroll 4
  for (int k = 0; k < own; ++k) {
    const int e = lane + 32 * k;
    if (e >= a.top) break;
    id_list[e] = load_input(a.teacher_ids + size_t(row) * size_t(a.ids_stride) + e);
    const size_t at = size_t(row) * size_t(a.values_stride) + e;
    w_list[e] = a.teacher_dtype == DS41_B200_F64 ? load_input(static_cast<const double *>(a.teacher_values) + at)
                                                 : double(load_input(static_cast<const float *>(a.teacher_values) + at));
  }
#pragma unroll 4
  for (int k = 0; k < own; ++k) {
    const int e = lane + 32 * k, id = e < a.top ? id_list[e] : -1;
    if (id < 0 || id >= a.vocab) continue;
    const bool is = !mask || ((load_input(mask + (id >> 5)) >> (id & 31)) & 1u);
    z_list[e] = is ? R::load(whole[id]) : -INFINITY;
  }
  unsigned named = 0u, counts = 0u;           // a bit per entry of the lane
  bool bad = false;
  double most = -DBL_MAX;
  float zmax = -FLT_MAX;
#pragma unroll 1
  for (int k = 0; k < own; ++k) {
    const int e = lane + 32 * k, id = e < a.top ? id_list[e] : -1;
    if (id >= 0 && id < a.vocab) {
      const float z = z_list[e];
      named |= 1u << k;
      bad |= !(w_list[e] < INFINITY) || !(z < INFINITY);
      if (!(z == -INFINITY)) { counts |= 1u << k; most = fmax(most, w_list[e]); zmax = fmaxf(zmax, z); }
    }
    if (e < top_room && !((counts >> k) & 1u)) id_list[e] = -2 - e;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    most = fmax(most, __shfl_xor_sync(0xffffffffu, most, o));
    zmax = fmaxf(zmax, __shfl_xor_sync(0xffffffffu, zmax, o));
  }
  __syncwarp();
  unsigned first = counts;                  // entries with no other of the same id in front of them
#pragma unroll 1
  for (int k = 0; k < own; ++k) {
    if (!((counts >> k) & 1u)) continue;
    const int e = lane + 32 * k, id = id_list[e];
#pragma unroll 2
    for (int j = 0; 4 * j < e; ++j) {
      const int4 q = reinterpret_cast<const int4 *>(id_list)[j];
      const int before = e - 4 * j;
      if (q.x == id || (before > 1 && q.y == id) || (before > 2 && q.z == id) || (before > 3 && q.w == id)) { first &= ~(1u << k); break; }
    }
  }
  const bool again = __any_sync(0xffffffffu, first != counts);
  double list = 0.0, kept = 0.0, entropy = 0.0;
  float share = 0.f;
#pragma unroll 1
  for (int k = 0; k < own; ++k) {
    const int e = lane + 32 * k;
    if (!((named >> k) & 1u)) continue;
    const double log_w = a.tail ? w_list[e] : (w_list[e] - most) * p.inverse_t, w = exp_of(log_w);
    list += w;
    const bool is = (counts >> k) & 1u;
    w_list[e] = is ? w : 0.0;
    if (!is) continue;
    kept += w;
    if (!again) {
      const double gap = (double(z_list[e]) - double(zmax)) * p.inverse_t;
      if (w > 0.0) entropy += w * (log_w - gap);
      share += exp2_approx((z_list[e] - zmax) * p.log2e_t);
    }
  }
  if (again) {                              // an id's first entry takes the weights of the later ones
    __syncwarp();
    double merged[kDisOwn];
#pragma unroll 1
  for (int k = 0; k < own; ++k) {
      const int e = lane + 32 * k;
      merged[k] = e < a.top ? w_list[e] : 0.0;
      if (!((first >> k) & 1u)) continue;
#pragma unroll 1
      for (int j = e + 1; j < a.top; ++j)
        if (id_list[j] == id_list[e]) merged[k] += w_list[j];
      const double gap = (double(z_list[e]) - double(zmax)) * p.inverse_t;
      if (merged[k] > 0.0) entropy += merged[k] * (log_of(merged[k]) - gap);
      share += exp2_approx((z_list[e] - zmax) * p.log2e_t);
    }
    __syncwarp();
#pragma unroll 1
  for (int k = 0; k < own; ++k) {
      const int e = lane + 32 * k;
      if (e >= a.top) continue;
      w_list[e] = merged[k];
      if (((counts & ~first) >> k) & 1u) id_list[e] = -2 - e;
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    list += __shfl_xor_sync(0xffffffffu, list, o);
    kept += __shfl_xor_sync(0xffffffffu, kept, o);
    entropy += __shfl_xor_sync(0xffffffffu, entropy, o);
    share += __shfl_xor_sync(0xffffffffu, share, o);
  }
  bad = __any_sync(0xffffffffu, bad);
  if (lane < 2) (lane ? r.inverse_rest : r.inverse) = over(1.0, kept + (lane && a.tail ? fmax(0.0, 1.0 - list) : 0.0));
  if (lane == 0) {
    r.reject = bad ? DS41_B200_ROW_NONFINITE : a.tail && list > kDisMost ? DS41_B200_ROW_NOT_NORMALIZED : !(kept > 0.0) ? DS41_B200_ROW_EMPTY : 0;
    r.zmax = zmax; r.share = share; r.kept = kept; r.entropy = entropy;
    r.rest = a.tail ? fmax(0.0, 1.0 - list) : 0.0;
    if (kMode == kDistillGrad) r.stats = reinterpret_cast<const float4 *>(a.stats)[row];
  }
  __syncwarp();
}

// Loss, stats and status of a row that is done, by one thread; result: (maximum, sum) of its ids outside the list.
template <int kMode>
__device__ __forceinline__ void finish_row(const DistillParams &p, int row, const DistillRow &r, float2 result) {
  const ds41_b200_distill_args &a = p.a;
  const double t = a.temperature;
  if (skipped<kMode>(r)) {
    a.loss[row] = 0.f; a.status[row] = 0;
    if (a.stats) reinterpret_cast<float4 *>(a.stats)[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    return;
  }
  const float rest_max = result.x, rest_sum = result.y, nan = __int_as_float(0x7fffffff);
  const int reject = r.reject ? r.reject : rest_sum < INFINITY ? 0 : DS41_B200_ROW_NONFINITE;
  float loss = reject == DS41_B200_ROW_EMPTY ? 0.f : nan;
  float4 stats = make_float4(nan, nan, nan, nan);
  if (!reject) {
    const bool any = rest_sum != 0.f;
    const double zmax = r.zmax, largest = any ? fmax(double(rest_max), zmax) : zmax;
    const double down = any ? (double(rest_max) - largest) * p.inverse_t : 0.0, list_down = (zmax - largest) * p.inverse_t;
    const double log_rest = log_of(double(rest_sum));
    const double log_sum = log_of((any ? double(rest_sum) * exp_of(down) : 0.0) + double(r.share) * exp_of(list_down));
    const double inverse = any ? r.inverse_rest : r.inverse, kept = r.kept * inverse, tail = any ? r.rest * inverse : 0.0;
    double sum = r.entropy * inverse + kept * (log_of(inverse) + log_sum - list_down);
    if (tail > 0.0) sum += tail * (log_of(tail) - (down + log_rest - log_sum));
    loss = float(t * t * sum);
    stats = make_float4(float(largest), float(log_sum), any ? rest_max : -INFINITY, any ? float(log_rest) : -INFINITY);
  }
  a.loss[row] = loss;
  a.status[row] = reject;
  if (a.stats) reinterpret_cast<float4 *>(a.stats)[row] = stats;
}

// The gradient of a row's listed ids in begin .. begin + len, by one warp, behind that of all others.  all: the row's maximum and 1 / its sum
// (NaN: the row has been filled).
template <class T>
__device__ __forceinline__ void set_listed(const DistillParams &p, int row, const DistillRow &r, const DistillList &list, float2 result,
                                           float2 all, int begin, int len, int lane) {
  if (!(all.y == all.y)) return;
  const ds41_b200_distill_args &a = p.a;
  const double inverse = result.y != 0.f ? r.inverse_rest : r.inverse, factor = double(r.scale) * a.temperature;
  T *const grad = static_cast<T *>(a.grad) + size_t(row) * size_t(a.grad_stride) + begin;
#pragma unroll 1
  for (int e = lane; e < a.top; e += 32) {
    const unsigned local = unsigned(list.ids[e]) - unsigned(begin);
    if (local >= unsigned(len)) continue;
    const float q = exp2_approx((list.zs[e] - all.x) * p.log2e_t) * all.y;
    grad[local] = RowType<T>::store(float(factor * (double(q) - list.weights[e] * inverse)));
  }
  __syncwarp();                               // (the list's memory is the next but one row's)
}

// How the gradient of the ids outside the list is made of their logits: the power of fma(z, scaled, minus) * factor + shift, times size (FP32)
// or with its sign from `sign` (16-bit types).
struct DistillFactors {
  int reject;
  float rest_max, rest_sum;                   // of the ids outside the list: maximum, sum relative to it (0: there are none)
  float largest, inverse_sum;                 // of all ids: maximum, 1 / the sum
  bool close;                                 // scaled = log2(e) / T, minus = offset, factor = 1, shift = 0
  float offset, scaled, minus, factor, shift, size;
  uint32_t sign;
};
template <int kMode, int kBytes>
__device__ __forceinline__ DistillFactors gradient_factors(const DistillParams &p, const DistillRow &r, float rest_max, float rest_sum) {
  const float log2e_t = p.log2e_t;
  DistillFactors f;
  f.reject = r.reject;
  float q_rest;                               // share of the ids outside the list
  bool any;
  if (kMode == kDistillGrad) {
    f.largest = r.stats.x; f.inverse_sum = exp2_approx(-r.stats.y * 1.44269504f);
    any = r.stats.w > -INFINITY;
    rest_max = r.stats.z;
    rest_sum = any ? exp2_approx(r.stats.w * 1.44269504f) : 0.f;
    q_rest = any ? rest_sum * exp2_approx((rest_max - f.largest) * log2e_t) * f.inverse_sum : 0.f;
    if (!f.reject && !(r.stats.x == r.stats.x)) f.reject = DS41_B200_ROW_NONFINITE;
  } else {
    any = rest_sum != 0.f;
    f.largest = any ? fmaxf(rest_max, r.zmax) : r.zmax;
    const float part = any ? rest_sum * exp2_approx((rest_max - f.largest) * log2e_t) : 0.f;
    f.inverse_sum = 1.f / (part + r.share * exp2_approx((r.zmax - f.largest) * log2e_t));
    q_rest = part * f.inverse_sum;
    if (!f.reject && !(rest_sum < INFINITY)) f.reject = DS41_B200_ROW_NONFINITE;
  }
  // (no ids outside the list: a maximum of theirs that is none would make the power's correction below infinite, and 0 times it NaN)
  if (!any) rest_max = 0.f;
  f.rest_max = rest_max; f.rest_sum = rest_sum;
  const float tail = any ? float(r.rest * r.inverse_rest) : 0.f, coef = any ? r.scale * float(p.a.temperature) * (q_rest - tail) / rest_sum : 0.f;
  // 16-bit types: the factor's size goes into the exponent, its sign into the words (exponents below 512 are off by 2^-16, a power
  // by as much, which is little beside the rounding to 16 bits)
  const float rest_c = rounded_product(rest_max, log2e_t), over_c = excess(rest_max, log2e_t, rest_c);
  f.close = kBytes == 4 ? near_exponent(rest_c) : fabsf(rest_c) < 256.f;
  const float shift = kBytes == 4 ? 0.f : log2f(fabsf(coef));
  f.size = kBytes == 4 ? coef * exp2_approx(f.close ? -over_c : 0.f) : 1.f;
  f.offset = kBytes == 4 ? -rest_c : __fsub_rn(__fsub_rn(shift, rest_c), over_c);
  f.sign = kBytes != 4 && coef < 0.f ? 0x80008000u : 0u;
  f.scaled = f.close ? log2e_t : 1.f; f.factor = f.close ? 1.f : log2e_t;
  f.minus = f.close ? f.offset : -rest_max; f.shift = f.close ? 0.f : shift;
  return f;
}

}  // namespace
}  // namespace ds41
