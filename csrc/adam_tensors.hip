// One Adam / AdamW step over a list of tensors of any shape and of mixed types, with moments in 32 or in 8 bits.
//
//   g' = g * scale * clip (+ wd * p, coupled),  m = b1 m + (1 - b1) g',  v = b2 v + ((1 - b2) g') g'
//   p  = p (1 - lr wd, decoupled) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Two launches whatever the number of tensors (up to 112 each): the global gradient norm, whose last workgroup also
// derives the step's factors (without clipping: that workgroup alone), and the update.  t is the tensor's own count of
// steps: one that is left out of some (no gradient) is corrected for those it took.  The factors of all tensors are
// computed side by side from their counts, and the update's first workgroup of a tensor advances its count.  The
// table of tensors travels by value in the kernel arguments, so a captured graph holds its own copy.
//
// Moments in 8 bits.  A block of 256 consecutive elements of one tensor shares a power of two 2^e, the one at or below
// its largest magnitude; an element keeps y = |x| / 2^e in [0, 2] as 4 bits of exponent and 3 (m, with a sign) or 4 (v)
// of mantissa: 14 binades and, below them, the even steps of the lowest.  The parameter update takes the unrounded
// moments; only what is kept for the next step is rounded, up or down by chance so that its mean is the value:
// floor(y / step + u), u a 16-bit hash of (seed, step, element).  Rounding to nearest would freeze the second moment:
// a step changes it by at most the part 1 - b2 of its distance, far below half a step of 4 mantissa bits (2^-6 .. 2^-5).
// (v itself is kept, not its square root, since the mean has to hold for v: a root that is right in the mean makes its
// square too large by its variance, step after step.)  A v above zero never falls to zero, which would leave
// m / eps as the update; a block's tiny v are held at its lowest code instead, and such elements move less.
// A block with a NaN or an infinity reads as NaN afterwards.
//
// Bound by memory: 28 bytes an fp32 parameter (p, m, v read and written, g read), 16 in 8 bits: 403 million weights in
// 1.32 ms, 4.9 TB/s (a copy: 4.7 - 4.8).  The norm is a pass of its own, 51 us for 64 million bf16 gradients.  Moments in 8 bits are
// computed in 64 bits up to their rounding (an element in some 10^6 falls on another code where they are off by an ulp of
// fp32, and a code is 3 to 6 % of the value), all else in fp32; nothing is contracted, so that the formulas give the same
// bits wherever they are evaluated.
#include <initializer_list>

#include "adam_tensors.h"
#include "common.h"

namespace {

#pragma clang fp contract(off)

constexpr int TPB = 256;
constexpr int WAVES = TPB / 64;
constexpr int NORM_TPB = 512;
constexpr int NORM_GROUPS = 256;          // workgroups of the norm at most: each ends with an add on one counter (30 ns)
constexpr long NORM_ELEMENTS = 8192;      // and has at least so many elements
enum { CTL_GS = 0, CTL_GS_LOW, CTL_DECAY, CTL_SKIP };  // gradient's factor: GS + GS_LOW; SKIP: this step changes nothing
enum { ADAM_F_SIZE = 0, ADAM_F_BC2, ADAM_F_T };  // a tensor's step size, 1 / sqrt(1 - b2^t), t

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__bf16 x) { return (float)x; }
__device__ __forceinline__ float up(_Float16 x) { return (float)x; }

template <typename T>
struct Four;
template <>
struct Four<float> {
  typedef f32x4 vec;
};
template <>
struct Four<__bf16> {
  typedef bf16x4 vec;
};
template <>
struct Four<_Float16> {
  typedef _Float16 vec __attribute__((ext_vector_type(4)));
};

// elements i .. i + 3 of a tensor of n (past its end: zeros); vec: 4-element accesses are aligned
template <typename T>
__device__ __forceinline__ void load4(const T* p, long i, long n, bool vec, float (&x)[4]) {
  if (vec && i + 4 <= n) {
    const typename Four<T>::vec v = *reinterpret_cast<const typename Four<T>::vec*>(p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = up((T)v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i + k < n ? up(p[i + k]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, long i, long n, bool vec, const float (&x)[4]) {
  if (vec && i + 4 <= n) {
    typename Four<T>::vec v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (T)x[k];
    *reinterpret_cast<typename Four<T>::vec*>(p + i) = v;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = (T)x[k];
  }
}
template <typename T>
__device__ __forceinline__ bool aligned4(const T* p) {
  return ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0;
}

// the tensor that workgroup `g` takes: the last that starts at or before it, so never an empty one
__device__ __forceinline__ int tensor_of(const AdamTable& t, unsigned g) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= g) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ---- 8-bit moments -----------------------------------------------------------------------------------------------------
constexpr int EXP_MIN = -100, EXP_MAX = 126, EXP_NAN = -128;

// the block's exponent from its largest magnitude's upper half (the same in all lanes)
__device__ __forceinline__ int block_exp(unsigned top) {
  if (top >= (1151u << 20)) return EXP_NAN;  // NaN, infinity, or past fp32's
  return min(max((int)(top >> 20) - 1023, EXP_MIN), EXP_MAX);
}

template <int DIG>
__device__ __forceinline__ unsigned encode(double x, int e, unsigned chance) {
  const unsigned high = (unsigned)(__builtin_bit_cast(uint64_t, x) >> 32);
  const unsigned field = (unsigned)max((int)(high >> 20 & 2047u) - (1010 + e), 0);  // x's exponent over the lowest binade's
  const double scale = __builtin_bit_cast(double, (uint64_t)((unsigned)(DIG + 16 + 13 + 1023 - e) - field << 20) << 32);
  const unsigned q = ((unsigned)(fabs(x) * scale) + chance) >> 16;
  const unsigned code = min((field << DIG) + q, 15u << DIG);
  return DIG == 4 ? max(code, min(high, 1u)) : code | (high >> 24 & 128u);  // v: not to zero; m: with its sign
}
// A code read as the top bits of a float is y 2^-113, the lowest steps being the float's own subnormals.  times: for
// values 1, or what they are to be multiplied by.
__device__ __forceinline__ double unit(int e, double times) {
  return e == EXP_NAN ? (double)NAN : __builtin_bit_cast(double, (uint64_t)(113 + e + 1023) << 52) * times;
}
template <int DIG>
__device__ __forceinline__ double decode(unsigned code, double unit) {
  unsigned bits = code << (23 - DIG);
  if (DIG == 3) bits = (bits & 0x07ffffffu) | (code & 128u) << 24;
  return (double)__builtin_bit_cast(float, bits) * unit;
}

// 32 random bits of element i: a hash of (seed, step, i); key: that of the elements that share i's upper half
__device__ __forceinline__ uint32_t key_of(uint64_t seed, uint32_t step, uint32_t high) {
  return (uint32_t)seed ^ (step * 0x9E3779B1u) ^ ((uint32_t)(seed >> 32) * 0x85EBCA77u) ^ (high * 0x27D4EB2Fu);
}
__device__ __forceinline__ uint32_t chance_of(uint32_t key, uint32_t i) {
  uint32_t x = key ^ i;
  x ^= x >> 16;
  x *= 0x7FEB352Du;
  x ^= x >> 15;
  x *= 0x846CA68Bu;
  return x ^ (x >> 16);
}

// upper half of the largest of four magnitudes per lane over the wave; a NaN's is above infinity's
__device__ __forceinline__ unsigned wave_top(const double (&x)[4]) {
  unsigned u = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) u = max(u, (unsigned)(__builtin_bit_cast(uint64_t, x[k]) >> 32) & 0x7fffffffu);
  // over the rows of 16 lanes by exchanges within them, then over the four as scalars
  u = max(u, (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xf, 0xf, false));   // lane ^ 1
  u = max(u, (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xf, 0xf, false));   // lane ^ 2
  u = max(u, (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, 0x141, 0xf, 0xf, false));  // 7 - lane of 8
  u = max(u, (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, 0x140, 0xf, 0xf, false));  // 15 - lane of 16
  auto lane = [&](int i) { return (unsigned)__builtin_amdgcn_readlane((int)u, i); };
  return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}

// ---- norm and this step's factors --------------------------------------------------------------------------------------
// Sum of squares, in 64 bits, of elements i0 .. i1 of a tensor: 16-byte loads where the start allows them, four of a
// thread's in flight.
template <typename G>
__device__ __forceinline__ double squares(const G* g, long i0, long i1) {
  constexpr int V = 16 / (int)sizeof(G), U = 4;
  typedef G vec __attribute__((ext_vector_type(V)));
  double sum = 0.0;
  long i = i0 + threadIdx.x;
  if (((uintptr_t)(g + i0) & 15) == 0) {
    const vec* v = reinterpret_cast<const vec*>(g + i0);
    const long n = (i1 - i0) / V;
    long k = threadIdx.x;
    for (; k + (U - 1) * NORM_TPB < n; k += U * NORM_TPB) {
      vec x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = v[k + u * NORM_TPB];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) sum = fma((double)up((G)x[u][e]), (double)up((G)x[u][e]), sum);
    }
    for (; k < n; k += NORM_TPB) {
      const vec x = v[k];
#pragma unroll
      for (int e = 0; e < V; ++e) sum = fma((double)up((G)x[e]), (double)up((G)x[e]), sum);
    }
    i += n * V;
  }
  for (; i < i1; i += NORM_TPB) sum = fma((double)up(g[i]), (double)up(g[i]), sum);
  return sum;
}

__device__ __forceinline__ double whole_power(double x, unsigned n) {
  double p = 1.0;
  for (; n; n >>= 1, x *= x)
    if (n & 1) p *= x;
  return p;
}

// by a whole workgroup: the tensors' factors by all waves but the first, whose first thread takes what they share
__device__ __forceinline__ void finish(const AdamState& s, double sq) {
  const float lr = s.lr[0];
  for (int k = (int)threadIdx.x - 64; k >= 0 && k < s.count; k += NORM_TPB - 64) {
    const float t = s.steps[k] + 1.f;
    const float size = (float)((double)lr / (1.0 - whole_power(s.dbeta1, (unsigned)t)));
    const float bc2 = (float)(1.0 / sqrt(1.0 - whole_power(s.dbeta2, (unsigned)t)));
    reinterpret_cast<f32x4*>(s.factors)[k] = f32x4{size, bc2, t, 0.f};
  }
  if (threadIdx.x != 0) return;
  const double norm = sqrt(sq) * s.scale;
  const bool bad = !isfinite((float)norm), skip = s.skip && bad;
  if (s.max_norm > 0.0 || s.skip) {
    s.norm[0] = (float)norm;
    if (bad) s.nonfinite[0] += 1.f;
  }
  s.ctl[CTL_SKIP] = skip ? 1.f : 0.f;
  if (!skip) s.step[0] += 1.f;
  double gs = s.scale;
  if (s.max_norm > 0.0) {
    const double c = s.max_norm / (norm + 1e-6);
    gs *= c < 1.0 ? c : (c != c ? c : 1.0);  // a NaN norm stays visible (as torch's clipping), unless skipped
  }
  s.ctl[CTL_GS] = (float)gs;
  s.ctl[CTL_GS_LOW] = (float)(gs - (double)(float)gs);
  s.ctl[CTL_DECAY] = s.decoupled ? (float)(1.0 - (double)lr * (double)s.wd) : 1.f;
}

__global__ __launch_bounds__(NORM_TPB) void adam_factors_kernel(AdamState s) { finish(s, 0.0); }

// part0: this launch's first partial; last: the list ends with this launch, whose last workgroup takes the sum
__global__ __launch_bounds__(NORM_TPB) void adam_norm_kernel(AdamTable t, AdamState s, int part0, int nparts, int last) {
  __shared__ double scratch[NORM_TPB / 64];
  __shared__ unsigned arrived;
  // a stretch of the list, so that the tensor is looked up once and then followed
  double sum = 0.0;
  unsigned w = (unsigned)((unsigned long long)t.groups * blockIdx.x / gridDim.x);
  const unsigned end = (unsigned)((unsigned long long)t.groups * (blockIdx.x + 1) / gridDim.x);
  for (int k = tensor_of(t, w); w < end; ++k) {
    const unsigned next = min(end, k + 1 < t.count ? t.first[k + 1] : t.groups);
    const long i0 = (long)(w - t.first[k]) * t.group, i1 = min(t.n[k], (long)(next - t.first[k]) * t.group);
    const int gt = t.type[k] >> 2;
    if (gt == ADAM_F32) sum += squares((const float*)t.g[k], i0, i1);
    else if (gt == ADAM_BF16) sum += squares((const __bf16*)t.g[k], i0, i1);
    else sum += squares((const _Float16*)t.g[k], i0, i1);
    w = next;
  }
  sum = wave_sum_d(sum);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double p = 0.0;
    for (int w = 0; w < NORM_TPB / 64; ++w) p += scratch[w];
    __hip_atomic_store(s.parts + part0 + blockIdx.x, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    arrived = 0;
    if (last) arrived = __hip_atomic_fetch_add(s.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) + 1;
  }
  __syncthreads();
  if (arrived != gridDim.x) return;  // (never 0 == gridDim.x)
  // the last to arrive: every partial of this launch is there, earlier launches' are too; summed in a fixed order
  sum = 0.0;
  for (int k = threadIdx.x; k < nparts; k += NORM_TPB)
    sum += __hip_atomic_load(s.parts + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  sum = wave_sum_d(sum);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = sum;
  __syncthreads();
  double sq = 0.0;
  for (int w = 0; w < NORM_TPB / 64; ++w) sq += scratch[w];
  finish(s, sq);
  if (threadIdx.x == 0) __hip_atomic_store(s.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---- update ------------------------------------------------------------------------------------------------------------
template <typename P, typename G, bool WIDE, int PER>
__device__ __forceinline__ void update(P* p, G* g, long n, int tensor, unsigned block0, unsigned wg, const AdamState& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float gs = s.ctl[CTL_GS], decay = s.ctl[CTL_DECAY];
  const float* f = s.factors + 4 * (long)tensor;
  const float size = f[ADAM_F_SIZE], inv_bc2 = f[ADAM_F_BC2], taken = f[ADAM_F_T];
  const bool skip = s.ctl[CTL_SKIP] != 0.f;  // asked for with all loads on their way, which would wait for it otherwise
  const double gs64 = (double)gs + (double)s.ctl[CTL_GS_LOW];
  const uint32_t t = (uint32_t)taken;
  const bool pv = aligned4(p), gv = aligned4(g);
  const long b0 = ((long)wg * WAVES + wave) * PER;  // the wave's first block of the tensor
  float pp[PER][4], gg[PER][4], mm[PER][4], vv[PER][4];
  unsigned mc[PER], vc[PER];
  int em[PER], ev[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const long i = (b0 + u) * ADAM_BLOCK + lane * 4;
    if ((b0 + u) * ADAM_BLOCK >= n) continue;
    // whole blocks by all lanes at once: with the other way's loads into the same registers in between, each waits for the last
    const bool whole = (b0 + u + 1) * ADAM_BLOCK <= n;
    if (__builtin_amdgcn_readfirstlane(whole && pv && gv)) {
      load4(p, i, i + 4, true, pp[u]);
      load4(g, i, i + 4, true, gg[u]);
    } else {
      load4(p, i, n, pv, pp[u]);
      load4(g, i, n, gv, gg[u]);
    }
    const long sb = (long)block0 + b0 + u, si = sb * ADAM_BLOCK + lane * 4;  // the state is padded to whole blocks
    if constexpr (WIDE) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(s.m32 + si), b = *reinterpret_cast<const f32x4*>(s.v32 + si);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mm[u][k] = a[k];
        vv[u][k] = b[k];
      }
    } else {
      mc[u] = *reinterpret_cast<const unsigned*>(s.m8 + si);
      vc[u] = *reinterpret_cast<const unsigned*>(s.v8 + si);
      em[u] = s.em[sb];
      ev[u] = s.ev[sb];
    }
  }
  if (skip) {
    if (!s.zero_grad) return;
#pragma unroll 1
    for (int u = 0; u < PER; ++u) store4(g, (b0 + u) * ADAM_BLOCK + lane * 4, n, gv, {0.f, 0.f, 0.f, 0.f});
    return;
  }
  if (wg == 0 && threadIdx.x == 0) s.steps[tensor] = taken;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const long i = (b0 + u) * ADAM_BLOCK + lane * 4;
    if ((b0 + u) * ADAM_BLOCK >= n) continue;
    const long sb = (long)block0 + b0 + u, si = sb * ADAM_BLOCK + lane * 4;
    double m64[4], v64[4];
    if constexpr (!WIDE) {
      const double um = unit(__builtin_amdgcn_readfirstlane(em[u]), s.dbeta1), uv = unit(__builtin_amdgcn_readfirstlane(ev[u]), s.dbeta2);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        double x = (double)gg[u][k] * gs64;  // past the end: 0, or NaN with the whole block
        if (!s.decoupled) x = x + (double)pp[u][k] * s.dwd;
        m64[k] = decode<3>((mc[u] >> (8 * k)) & 255u, um) + x * (1.0 - s.dbeta1);
        v64[k] = decode<4>((vc[u] >> (8 * k)) & 255u, uv) + x * (1.0 - s.dbeta2) * x;
        mm[u][k] = (float)m64[k];
        vv[u][k] = (float)v64[k];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (WIDE) {
        float x = gg[u][k] * gs;
        if (!s.decoupled) x = x + pp[u][k] * s.wd;
        if (i + k >= n) x = 0.f;
        mm[u][k] = mm[u][k] * s.beta1 + x * s.one_beta1;
        vv[u][k] = vv[u][k] * s.beta2 + x * s.one_beta2 * x;
      }
      // root and reciprocal of the hardware, each within an ulp: the update's part of the parameter's own rounding
      const float root = __builtin_amdgcn_sqrtf(vv[u][k]) * inv_bc2;
      pp[u][k] = pp[u][k] * decay - mm[u][k] * __builtin_amdgcn_rcpf(root + s.eps) * size;
    }
    store4(p, i, n, pv, pp[u]);
    if (s.zero_grad) {
      const float z[4] = {0.f, 0.f, 0.f, 0.f};
      store4(g, i, n, gv, z);
    }
    if constexpr (WIDE) {
      *reinterpret_cast<f32x4*>(s.m32 + si) = f32x4{mm[u][0], mm[u][1], mm[u][2], mm[u][3]};
      *reinterpret_cast<f32x4*>(s.v32 + si) = f32x4{vv[u][0], vv[u][1], vv[u][2], vv[u][3]};
    } else {
      const int e1 = block_exp(wave_top(m64)), e2 = block_exp(wave_top(v64));
      const uint32_t key = key_of(s.seed, t, (uint32_t)(sb >> 24));  // 2^24 blocks have 2^32 elements
      unsigned a = 0, b = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const unsigned r = chance_of(key, (uint32_t)si + k);
        a |= encode<3>(m64[k], e1, r & 0xFFFFu) << (8 * k);
        b |= encode<4>(v64[k], e2, r >> 16) << (8 * k);
      }
      if (e1 == EXP_NAN) a = 0;
      if (e2 == EXP_NAN) b = 0;
      *reinterpret_cast<unsigned*>(s.m8 + si) = a;
      *reinterpret_cast<unsigned*>(s.v8 + si) = b;
      if (lane == 0) {
        s.em[sb] = (signed char)e1;
        s.ev[sb] = (signed char)e2;
      }
    }
  }
}

template <bool WIDE, int PER>
__global__ __launch_bounds__(TPB) void adam_update_kernel(AdamTable t, AdamState s) {
  const int k = tensor_of(t, blockIdx.x);
  const unsigned wg = blockIdx.x - t.first[k];
  const long n = t.n[k];
  const int i = t.place + k;
  switch (t.type[k]) {
    case ADAM_F32 | ADAM_F32 << 2: update<float, float, WIDE, PER>((float*)t.p[k], (float*)t.g[k], n, i, t.block[k], wg, s); break;
    case ADAM_F32 | ADAM_BF16 << 2: update<float, __bf16, WIDE, PER>((float*)t.p[k], (__bf16*)t.g[k], n, i, t.block[k], wg, s); break;
    case ADAM_F32 | ADAM_F16 << 2: update<float, _Float16, WIDE, PER>((float*)t.p[k], (_Float16*)t.g[k], n, i, t.block[k], wg, s); break;
    case ADAM_BF16 | ADAM_BF16 << 2: update<__bf16, __bf16, WIDE, PER>((__bf16*)t.p[k], (__bf16*)t.g[k], n, i, t.block[k], wg, s); break;
    case ADAM_F16 | ADAM_F16 << 2: update<_Float16, _Float16, WIDE, PER>((_Float16*)t.p[k], (_Float16*)t.g[k], n, i, t.block[k], wg, s); break;
  }
}

// ---- moments as values, and back ---------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(TPB) void adam_read_kernel(const unsigned char* m8, const unsigned char* v8,
                                                        const signed char* em, const signed char* ev, T* m, T* v, long blocks) {
  const int lane = threadIdx.x & 63;
  for (long b = (long)blockIdx.x * WAVES + (threadIdx.x >> 6); b < blocks; b += (long)gridDim.x * WAVES) {
    const long i = b * ADAM_BLOCK + lane * 4;
    const unsigned a = *reinterpret_cast<const unsigned*>(m8 + i), c = *reinterpret_cast<const unsigned*>(v8 + i);
    const double u1 = unit(em[b], 1.0), u2 = unit(ev[b], 1.0);
    float x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned ca = (a >> (8 * k)) & 255u;
      x[k] = (float)decode<3>(ca, u1);
      y[k] = (float)decode<4>((c >> (8 * k)) & 255u, u2);
    }
    store4(m, i, i + 4, true, x);
    store4(v, i, i + 4, true, y);
  }
}

// A loaded state: to the nearest code (chance 1/2).  A block whose largest value is a power of two takes it as y = 2,
// the grid's top, so that values that were read from codes always fall on codes again.
__device__ __forceinline__ int load_exp(const double (&x)[4]) {
  const unsigned top = wave_top(x);
  const int e = block_exp(top);
  bool more = false;  // an element past the power of two itself
#pragma unroll
  for (int k = 0; k < 4; ++k) more |= (__builtin_bit_cast(uint64_t, x[k]) & ~(1ull << 63)) > (uint64_t)(top >> 20) << 52;
  return e > EXP_MIN && !__any(more) ? e - 1 : e;
}
__global__ __launch_bounds__(TPB) void adam_write_kernel(unsigned char* m8, unsigned char* v8, signed char* em,
                                                         signed char* ev, const float* m, const float* v, long blocks) {
  const int lane = threadIdx.x & 63;
  for (long b = (long)blockIdx.x * WAVES + (threadIdx.x >> 6); b < blocks; b += (long)gridDim.x * WAVES) {
    const long i = b * ADAM_BLOCK + lane * 4;
    float x[4], y[4];
    load4(m, i, i + 4, true, x);
    load4(v, i, i + 4, true, y);
    const double xd[4] = {x[0], x[1], x[2], x[3]}, yd[4] = {y[0], y[1], y[2], y[3]};
    const int e1 = load_exp(xd), e2 = load_exp(yd);
    unsigned a = 0, c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (e1 != EXP_NAN) a |= encode<3>(xd[k], e1, 0x8000u) << (8 * k);
      if (e2 != EXP_NAN) c |= encode<4>(fmax(yd[k], 0.0), e2, 0x8000u) << (8 * k);
    }
    *reinterpret_cast<unsigned*>(m8 + i) = a;
    *reinterpret_cast<unsigned*>(v8 + i) = c;
    if (lane == 0) {
      em[b] = (signed char)e1;
      ev[b] = (signed char)e2;
    }
  }
}

inline int grid_blocks(long blocks) {
  const long g = (blocks + WAVES - 1) / WAVES;
  return (int)(g < 1 ? 1 : g > 16384 ? 16384 : g);
}

}  // namespace

// Elements of a workgroup of the update: 16 blocks (its loads in flight hide the memory's latency), or 4 where that
// leaves compute units idle (the encoder's 0.8 million weights).  Partials that one launch of the norm leaves.
extern "C" int mta_adam_group(long elements) { return elements < (4L << 20) ? 4 * ADAM_BLOCK : 16 * ADAM_BLOCK; }
extern "C" int mta_adam_norm_parts() { return NORM_GROUPS; }

// tables: `count` of them.  The norm over all of them first (with clipping or skipping), then the update of each.  0, or: 2 a
// table has more workgroups than a launch, 4 a launch failed
extern "C" int mta_adam_tensors(const AdamTable* tables, int count, const AdamState* s, int wide, hipStream_t st) {
  for (int k = 0; k < count; ++k)
    if (tables[k].groups < 1 || tables[k].groups > ADAM_GROUPS) return 2;
  auto start = [&](const void* f, unsigned grid, int threads, std::initializer_list<const void*> args) {
    void* p[8];
    int n = 0;
    for (const void* a : args) p[n++] = const_cast<void*>(a);
    return hipLaunchKernel(f, dim3(grid), dim3(threads), p, 0, st) == hipSuccess;
  };
  if (s->max_norm > 0.0 || s->skip) {
    int part0 = 0;
    for (int k = 0; k < count; ++k) {
      const long want = ((long)tables[k].groups * tables[k].group + NORM_ELEMENTS - 1) / NORM_ELEMENTS;
      const int parts = (int)(want < NORM_GROUPS ? want : NORM_GROUPS), all = part0 + parts, last = k + 1 == count;
      if (!start((const void*)adam_norm_kernel, parts, NORM_TPB, {&tables[k], s, &part0, &all, &last})) return 4;
      part0 = all;
    }
  } else if (!start((const void*)adam_factors_kernel, 1, NORM_TPB, {s})) {
    return 4;
  }
  for (int k = 0; k < count; ++k) {
    const bool few = tables[k].group == 4 * ADAM_BLOCK;
    auto kernel = wide ? (few ? adam_update_kernel<true, 1> : adam_update_kernel<true, 4>)
                       : (few ? adam_update_kernel<false, 1> : adam_update_kernel<false, 4>);
    if (!start((const void*)kernel, tables[k].groups, TPB, {&tables[k], s})) return 4;
  }
  return 0;
}

extern "C" void mta_adam_read(const AdamState* s, void* m, void* v, int bf16, long blocks, hipStream_t st) {
  if (bf16)
    adam_read_kernel<__bf16><<<grid_blocks(blocks), TPB, 0, st>>>(s->m8, s->v8, s->em, s->ev, (__bf16*)m, (__bf16*)v, blocks);
  else
    adam_read_kernel<float><<<grid_blocks(blocks), TPB, 0, st>>>(s->m8, s->v8, s->em, s->ev, (float*)m, (float*)v, blocks);
}

extern "C" void mta_adam_write(const AdamState* s, const float* m, const float* v, long blocks, hipStream_t st) {
  adam_write_kernel<<<grid_blocks(blocks), TPB, 0, st>>>(s->m8, s->v8, s->em, s->ev, m, v, blocks);
}
