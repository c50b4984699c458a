// Attention for sequences of any length (windows past the 64 tokens of attention.hip, padded batches, causal order,
// query heads that share key heads, single queries), forward and backward, in bf16, fp16 and fp32.
//
//   S = scale Q K^T over the keys a query sees,  L = log sum_j exp S_j,  P = exp(S - L),  O = P V
//   dV = P^T dO,  dP = dO V^T,  delta = rowsum(dO * O),  dS = P * (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q
//
// P is never stored: the forward keeps a running maximum and sum for each row, the backward recomputes P from L.
// Query i stands at position i + Tk - Tq; it sees the keys j < len (its sequence's), with `causal` those with
// j <= its position.  A row that sees no key has O = 0, L = -inf and no gradient.
//
// The rows of one problem (sequence, key head) are the G = H / Hkv query heads of its group times the Tq tokens, token
// major: row r is token r / G of query head r % G.  So the group's heads share every K / V tile that is staged, and the
// gradients of a shared key head are sums over rows inside one workgroup, without atomics.
//
// Every product runs on v_mfma_f32_32x32x16 (fp32: eight v_mfma_f32_32x32x2, the same fragments).  The scores are
// computed transposed where the row statistics are needed (forward, dQ: S^T = K Q^T, a lane owns ONE row and 16 of 32
// keys), so a row maximum is 15 in-lane operations and one exchange of the wave's halves, and the accumulator of one
// product is, element for element, the B operand of the next one: its 8 values of a 16-key step are the keys
// {4 h + 0..3, 8 + 4 h + 0..3} (h: the lane's half), and the A operand (V^T, K^T, dO^T, Q^T) is read from LDS with the
// same order of its contraction index -- P and dS never leave the registers.
#include <type_traits>
#include <utility>

#include "common.h"
#include "mha.h"

namespace {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <typename T>
struct El;
template <>
struct El<__bf16> {
  typedef bf16x8 frag;
  typedef bf16x4 quad;
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct El<_Float16> {
  typedef f16x8 frag;
  typedef f16x4 quad;
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct El<float> {
  typedef f32x8 frag;
  typedef f32x4 quad;
  // element j of the two halves is contraction index 8 h + j on both sides: any pairing of equal indices will do
  static __device__ __forceinline__ f32x16 mma(const frag& a, const frag& b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

constexpr int THREADS = 256, WAVES = 4;
constexpr int AHEAD = 3;  // steps that an operand is read from LDS before its product (2 .. 6 measured: 3 and 4 best)
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ---- LDS image of a tile: rows of DP elements in 16-byte chunks, chunk c of row r at r * CH + (c ^ swz(r)) ------------
// Both ways of reading are free of bank conflicts: a b128 row read takes the same chunk of 16 consecutive rows, which
// the swizzle spreads over all 16 chunk columns of a 256-byte bank line; a transposed read takes 4 aligned chunks of
// 4 consecutive rows, which it spreads over the 4 groups of 4 columns.
template <int CH>
__device__ __forceinline__ int swz(int r) {
  if constexpr (CH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (CH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return (r >> 2) & 3;
}

// LDS places are byte addresses of 32 bits; a tile starts on 1024 bytes
template <typename V>
__device__ __forceinline__ V lds_get(unsigned at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) V*>(at);
}
template <typename V>
__device__ __forceinline__ void lds_put(unsigned at, const V& v) {
  *reinterpret_cast<__attribute__((address_space(3))) V*>(at) = v;
}

__device__ __forceinline__ unsigned lds_base(const char* shared) { return (unsigned)(uintptr_t)shared; }

template <typename T, int DP>
struct Tile {
  static constexpr int EPC = 16 / (int)sizeof(T);  // elements of a chunk
  static constexpr int CH = DP / EPC;
  static constexpr int ROW_BYTES = DP * (int)sizeof(T);
  typedef typename El<T>::frag frag;

  // Operand fragment whose row is lane & 31 and whose 16 contraction indices are columns 16 kk ..: 8 of half h.  The chunk
  // is (2 kk + h) ^ swz: as the swizzle does not reach past a row, the lane's address is a constant of its own, xor 32 kk.
  static __device__ __forceinline__ unsigned row_lane(int lane) {
    const int r = lane & 31, c = (sizeof(T) == 2 ? 1 : 2) * (lane >> 5);
    return (r * CH + (c ^ swz<CH>(r))) * 16;
  }
  static __device__ __forceinline__ frag rows(unsigned t, int kk) {  // t: row_lane + the place of the 32 rows
    if constexpr (sizeof(T) == 2) {
      return lds_get<frag>(t ^ (32 * kk));
    } else {
      const f32x4 a = lds_get<f32x4>(t ^ (64 * kk)), b = lds_get<f32x4>(t ^ (64 * kk) ^ 16);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // Operand fragment whose row is COLUMN 32 db + (lane & 31) and whose contraction indices are 16 rows of the tile, in
  // the order {4 h + 0..3, 8 + 4 h + 0..3}: two transposing 64-bit reads (16 lanes read 4 rows x 16 columns, each lane
  // gets a column's 4 rows); fp32 has no such read, its 32 lanes read 32 consecutive floats of a row instead.  Rows 8 on
  // from another have the swizzle's bit 1 (32 bytes) flipped.
  static __device__ __forceinline__ unsigned col_lane(int lane) {
    if constexpr (sizeof(T) == 2) {
      const int r = 4 * (lane >> 5) + ((lane >> 2) & 3), c = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
      return (r * CH + (c ^ swz<CH>(r))) * 16 + (lane & 1) * 8;
    } else {
      return 0;
    }
  }
  static __device__ __forceinline__ frag cols(unsigned t, int db, int lane) {  // t: col_lane + the place of the 16 rows
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds4;
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const unsigned at = t ^ (64 * db);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4*>(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4*>((at ^ 32) + 8 * ROW_BYTES));
      const s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(frag, v);
    } else {
      frag f;
      const int d = 32 * db + (lane & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 4 * (lane >> 5) + (j & 3) + 8 * (j >> 2);  // of 16 rows; the swizzle has a period of 16
        f[j] = lds_get<float>(t + (r * CH + ((d >> 2) ^ swz<CH>(r))) * 16 + (d & 3) * 4);
      }
      return f;
    }
  }
};

// A tile of ROWS rows on its way from memory to LDS through registers: thread -> 16-byte chunk tid % CH of rows
// tid / CH + RPI i.  Rows past the `valid` ones (at least one) repeat the last: what is computed from them is masked, and
// holds no number that the last row did not bring in.  Columns past D meet zeros in the other operand, or are columns of a
// result that are not stored.  In keys and values they are zeros (an infinite element, which takes a key's weight to 0, would
// make a NaN with a zero): their threads load nothing and keep the zeros that their registers start with.  In q and dout,
// where an infinity is a NaN in any case, they repeat the first columns (a condition there costs the dK / dV kernel 6 %).
// Every load goes into the register where it stays until store(): nothing waits for it before.
template <typename T, int DP, int ROWS, int NT = THREADS>
struct Stage {  // NT threads: the workgroup, or a wave
  static constexpr int CH = Tile<T, DP>::CH, EPC = Tile<T, DP>::EPC, RPI = NT / CH, N = ROWS / RPI;
  static_assert(ROWS % RPI == 0 && NT % CH == 0, "whole passes");
  u32x4 r[N] = {};
  static __device__ __forceinline__ int row() { return threadIdx.x % NT / CH; }
  static __device__ __forceinline__ int elem() { return threadIdx.x % CH * EPC; }
  // p: the thread's chunk of the tile's first row; rs: elements from row to row
  __device__ __forceinline__ void load(const T* p, long rs, int valid, int D) {
    if (elem() >= D) return;
    if (valid >= ROWS) {
      const T* q = p + row() * rs;
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const u32x4*>(q + i * (RPI * rs));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const u32x4*>(p + min(row() + i * RPI, valid - 1) * rs);
    }
  }
  // at(row of the tile): the row's address; rows before `first` repeat it
  template <typename F>
  __device__ __forceinline__ void gather(F&& at, int e, int first, int valid) {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = *reinterpret_cast<const u32x4*>(at(max(first, min(row() + i * RPI, valid - 1))) + e);
  }
  __device__ __forceinline__ void store(unsigned t) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int rw = row() + i * RPI, c = threadIdx.x % CH;
      lds_put(t + (rw * CH + (c ^ swz<CH>(rw))) * 16, r[i]);
    }
  }
};

// N steps of `use(i, operand)` whose operands `read(i)` (LDS) are AHEAD steps ahead of their use, in exactly this order:
// left alone the compiler puts each read right before its product and waits out the LDS latency, some 120 cycles for
// each 32 cycles of product.  What else a step does (vector operations on other values) runs while its product does.
template <int I>
using Int = std::integral_constant<int, I>;
template <typename F, typename R, typename U, int... I>
__device__ __forceinline__ void stream_steps(R&& read, U&& use, std::integer_sequence<int, I...>) {
  constexpr int N = sizeof...(I);
  F ring[AHEAD];
  auto first = [&](auto i) __attribute__((always_inline)) {
    if constexpr (decltype(i)::value < AHEAD) ring[decltype(i)::value] = read(i);
  };
  auto step = [&](auto i) __attribute__((always_inline)) {
    constexpr int K = decltype(i)::value;
    __builtin_amdgcn_sched_barrier(0);
    use(i, ring[K % AHEAD]);
    if constexpr (K + AHEAD < N) ring[K % AHEAD] = read(Int<K + AHEAD>{});
  };
  __builtin_amdgcn_sched_barrier(0);
  (first(Int<I>{}), ...);
  (step(Int<I>{}), ...);
  __builtin_amdgcn_sched_barrier(0);
}
template <int N, typename F, typename R, typename U>
__device__ __forceinline__ void stream(R&& read, U&& use) {
  stream_steps<F>(read, use, std::make_integer_sequence<int, N>{});
}

// row of a problem -> its token (the row's query head is row - token * G)
__device__ __forceinline__ int token_of(const MhaArgs& A, int row) {
  return (int)(((unsigned long long)(unsigned)row * A.gmul) >> A.gshift);
}

// a lane's row straight from memory as operand fragments (null: zeros)
template <typename T, int DP>
__device__ __forceinline__ void load_frags(typename El<T>::frag (&f)[DP / 16], const T* p, int D, int h) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const int d = 16 * kk + 8 * h;
    typename El<T>::frag z = {};
    f[kk] = z;
    if (p != nullptr && d < D) f[kk] = *reinterpret_cast<const typename El<T>::frag*>(p + d);
  }
}

// both halves' values of the same lane & 31 (v_permlane32_swap exchanges the first register's upper half with the
// second's lower half)
__device__ __forceinline__ void halves(float x, float& lo, float& hi) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned a = r[0], b = r[1];
  lo = __builtin_bit_cast(float, a);
  hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float half_max(float x) {
  float lo, hi;
  halves(x, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float half_sum(float x) {
  float lo, hi;
  halves(x, lo, hi);
  return lo + hi;
}

// values 8 s .. 8 s + 7 of an accumulator as the next product's operand.  Rounded to 16 bits here (half a step, 2^-8 /
// 2^-11 of each value); sums of the same values are taken from the unrounded ones.
template <typename T>
__device__ __forceinline__ typename El<T>::frag as_frag(const f32x16& a, int s) {
  typename El<T>::frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)a[8 * s + j];
  return f;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  typename El<T>::quad v = {(T)a, (T)b, (T)c, (T)d};
  *reinterpret_cast<typename El<T>::quad*>(p) = v;
}

// accumulator row of register r: 8 (r / 4) + r % 4 + 4 h
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + (r & 3) + 4 * h; }

// workgroup -> (problem, tile): the tiles of one problem share its K / V, so they go to one of the 8 XCDs (workgroups
// are dealt to them in turn) and find them in its L2
__device__ __forceinline__ bool place(int problems, int tiles, int& problem, int& tile) {
  const int id = blockIdx.x;
  if (problems >= 8) {
    problem = (id / 8 / tiles) * 8 + (id & 7);
    tile = (id / 8) % tiles;
  } else {
    problem = id % problems;
    tile = id / problems;
  }
  return problem < problems;
}
inline long grid_of(long problems, long tiles) { return (problems >= 8 ? (problems + 7) / 8 * 8 : problems) * tiles; }

template <typename T>
__device__ __forceinline__ const T* at(const void* p, const long (&s)[3], long b, long t, long h) {
  return static_cast<const T*>(p) + b * s[0] + t * s[1] + h * s[2];
}
template <typename T>
__device__ __forceinline__ T* at(void* p, const long (&s)[3], long b, long t, long h) {
  return static_cast<T*>(p) + b * s[0] + t * s[1] + h * s[2];
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// A wave's 32 rows against 32-key blocks: S^T, running maximum and sum, O^T.  `acc`, `top` and `l` (this half's sum of
// exponentials) are of row lane & 31.
//
// The exponentials are 2^(S c - top), top the largest S c of the first block that the row sees anything of, so that its
// weight is 1 without rounding, and a whole number more when it follows: a row's sums are rescaled by powers of two,
// exactly, also where they are operands of 16 bits already.  It may lag the largest S c by up to 8: exponentials stay below
// 2^8, and the accumulators are rescaled (DP / 2 multiplications) only when some row passes that (2 x 4096 tokens causal, 32 heads of 128 on 8 key heads, bf16: 332 -> 322 us against a rescale in every tile).
template <typename T, int DP>
struct Rows {
  typedef typename El<T>::frag frag;
  typedef Tile<T, DP> TL;
  frag q[DP / 16];
  f32x16 acc[DP / 32];
  float top, l;  // top: -inf while nothing is seen
  int see;       // keys that the row sees
  int dim;       // (fp32) products with what is past it, eight instructions each, are left out
  float c;

  __device__ __forceinline__ void start(float scale, int D) {
    c = scale * LOG2E;
    dim = D;
    top = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = f32x16{};
  }
  // hides what the row does not see of keys key0 .. (a block), and lets the tops follow; true if some moved, this by alpha
  __device__ __forceinline__ bool follow(f32x16& s, int key0, bool masked, int h, float& alpha) {
    if (masked) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = acc_row(r, h) < see - key0 ? s[r] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = half_max(mx) * c;
    if (!__any(mx > top + 8.f)) return false;
    const float by = mx > top + 8.f ? ceilf(mx - top) : 0.f;  // infinite where nothing was seen yet: the sums are 0
    alpha = __builtin_amdgcn_exp2f(-by);
    top = by < INFINITY ? top + by : mx;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
    return true;
  }
  __device__ __forceinline__ float weight(float s, float base) const { return __builtin_amdgcn_exp2f(fmaf(s, c, -base)); }
  __device__ __forceinline__ float base() const { return top == -INFINITY ? 0.f : top; }  // nothing seen: all weights 0

  // one block of 32 keys, rows r0 .. of the tiles
  __device__ __forceinline__ void block(unsigned kt, unsigned vt, int r0, int key0, bool masked, int lane) {
    const int h = lane >> 5;
    const unsigned kl = kt + r0 * TL::ROW_BYTES + TL::row_lane(lane), vl = vt + r0 * TL::ROW_BYTES + TL::col_lane(lane);
    f32x16 s;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      if (sizeof(T) == 2 || 16 * kk < dim) s = El<T>::mma(TL::rows(kl, kk), q[kk], kk == 0 ? f32x16{} : s);
    float alpha;
    follow(s, key0, masked, h, alpha);
    const float b = base();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = weight(s[r], b);
      l += s[r];
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const frag p = as_frag<T>(s, st);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) acc[d] = El<T>::mma(TL::cols(vl + 16 * st * TL::ROW_BYTES, d, lane), p, acc[d]);
    }
  }

  // Two blocks (64 keys) in four phases: S of block 0; S of block 1 and the weights of block 0; the sums of block 0 and
  // the weights of block 1; the sums of block 1.
  __device__ __forceinline__ void blocks2(unsigned kt, unsigned vt, int key0, int all, int lane) {
    constexpr int M = DP / 16;  // operands of a phase
    const int h = lane >> 5;
    const unsigned kl = kt + TL::row_lane(lane), vl = vt + TL::col_lane(lane);
    f32x16 s[2];
    frag p[2][2];
    float alpha, b;
    auto weights = [&](int nb, int i) __attribute__((always_inline)) {  // part i of M of a block's
#pragma unroll
      for (int r = i * 16 / M; r < (i + 1) * 16 / M; ++r) {
        const float w = weight(s[nb][r], b);
        l += w;
        p[nb][r >> 3][r & 7] = (T)w;
      }
    };
    stream<M, frag>([&](auto i) __attribute__((always_inline)) { return TL::rows(kl, decltype(i)::value); },
                    [&](auto i, const frag& x) __attribute__((always_inline)) {
                      constexpr int kk = decltype(i)::value;
                      s[0] = El<T>::mma(x, q[kk], kk == 0 ? f32x16{} : s[0]);
                    });
    follow(s[0], key0, key0 + 32 > all, h, alpha);
    b = base();
    stream<M, frag>([&](auto i) __attribute__((always_inline)) { return TL::rows(kl + 32 * TL::ROW_BYTES, decltype(i)::value); },
                    [&](auto i, const frag& x) __attribute__((always_inline)) {
                      constexpr int kk = decltype(i)::value;
                      s[1] = El<T>::mma(x, q[kk], kk == 0 ? f32x16{} : s[1]);
                      weights(0, kk);
                    });
    if (follow(s[1], key0 + 32, key0 + 64 > all, h, alpha)) {
      b = base();
#pragma unroll
      for (int i = 0; i < 16; ++i) p[0][i >> 3][i & 7] = (T)((float)p[0][i >> 3][i & 7] * alpha);  // block 0's too, exactly
    }
    stream<2 * M, frag>(
        [&](auto i) __attribute__((always_inline)) {
          constexpr int nb = decltype(i)::value / M, k = decltype(i)::value % M;
          return TL::cols(vl + (32 * nb + 16 * (k / (DP / 32))) * TL::ROW_BYTES, k % (DP / 32), lane);
        },
        [&](auto i, const frag& x) __attribute__((always_inline)) {
          constexpr int nb = decltype(i)::value / M, k = decltype(i)::value % M, st = k / (DP / 32), d = k % (DP / 32);
          acc[d] = El<T>::mma(x, p[nb][st], acc[d]);
          if constexpr (nb == 0) weights(1, k);
        });
  }
};

// rows of a problem that end in memory: joined output and log-sum-exp, or the sums of a key range
template <typename T, int DP>
__device__ __forceinline__ void put_row(const MhaArgs& A, int problem, int split, int row, const f32x16 (&acc)[DP / 32], float top, float l,
                                        int h) {
  const int R = A.G * A.Tq;
  if (row >= R) return;
  const int b = problem / A.Hkv, tq = token_of(A, row), hq = problem % A.Hkv * A.G + row - tq * A.G;
  if (A.splits > 1) {
    float* p = A.part + (((long)split * A.B * A.Hkv + problem) * R + row) * (A.D + 2);
    if (h == 0) {
      p[A.D] = top;
      p[A.D + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * d + acc_row(r, h) < A.D) p[32 * d + acc_row(r, h)] = acc[d][r];
    return;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a NaN sum stays one
  T* o = at<T>(A.o, A.os, b, tq, hq);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 32 * d + 8 * i + 4 * h;
      if (col < A.D)
        store4<T>(o + col, acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv, acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv);
    }
  if (h == 0 && A.lse) A.lse[((long)b * A.H + hq) * A.Tq + tq] = l == 0.f ? -INFINITY : (top + __log2f(l)) * LN2;
}

// Waves on a SIMD (workgroups on a compute unit) that the forward kernels' registers are cut for: 128 floats a row do not
// fit into 256 registers (one query against 16 caches of 4096 keys, 8 heads: 672 us spilled).
template <typename T>
constexpr int forward_waves(int dp) {
  return dp * sizeof(T) >= 512 ? 1 : 2;
}

// Many rows: 128 of a problem to a workgroup, 32 to a wave; all waves walk the same key tiles.  2 x 4096 tokens causal, 32
// heads of 128 on 8, bf16: 310 us, 0.89 PFLOP/s (a large library product: 1.17), bound by the vector work between the
// products; 100 x 252, 4 heads of 32: 14.4 us, bound by the exponentials.  (64 rows a wave, each LDS
// operand meeting two, needs 512 registers and so leaves one wave on a SIMD: 472 against 350 us on the prompt above.)
template <typename T, int DP, int BN>
__global__ __launch_bounds__(THREADS, forward_waves<T>(DP)) void mha_fwd_kernel(MhaArgs A) {
  typedef Tile<T, DP> TL;
  constexpr int TILE = BN * TL::ROW_BYTES, BM = 32 * WAVES;
  extern __shared__ char shared[];  // [2][K tile | V tile]
  const unsigned lds = lds_base(shared);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int R = A.G * A.Tq, ntile = (R + BM - 1) / BM;
  int problem, tile;
  if (!place(A.B * A.Hkv, ntile, problem, tile)) return;
  if (A.causal) tile = ntile - 1 - tile;  // the longest rows first
  const int b = problem / A.Hkv, hk = problem % A.Hkv, off = A.Tk - A.Tq;
  const int n = A.lens ? min(max(A.lens[b], 0), A.Tk) : A.Tk;
  auto seen_by = [&](int row) { return A.causal ? max(0, min(n, token_of(A, row) + off + 1)) : n; };
  // key tiles of the workgroup; keys that some, and that all of the wave's rows see
  const int kend = seen_by(min((tile + 1) * BM, R) - 1);
  const int jt1 = (kend + BN - 1) / BN;
  const int row0 = tile * BM + 32 * wave, row = row0 + (lane & 31);
  const int wend = row0 < R ? seen_by(min(row0 + 32, R) - 1) : 0, wall = row0 < R ? seen_by(row0) : 0;

  Rows<T, DP> w;
  w.start(A.scale, A.D);
  w.see = row < R ? seen_by(row) : 0;
  const int t = token_of(A, min(row, R - 1));
  load_frags<T, DP>(w.q, row < R ? at<T>(A.q, A.qs, b, t, hk * A.G + row - t * A.G) : nullptr, A.D, h);
  typedef Stage<T, DP, BN> ST;
  ST sk, sv;
  const T* kp = at<T>(A.k, A.ks, b, 0, hk) + ST::elem();
  const T* vp = at<T>(A.v, A.vs, b, 0, hk) + ST::elem();
  auto fetch = [&](int jt) {
    sk.load(kp + (long)jt * BN * A.ks[1], A.ks[1], n - jt * BN, A.D);
    sv.load(vp + (long)jt * BN * A.vs[1], A.vs[1], n - jt * BN, A.D);
  };
  if (jt1 > 0) {
    fetch(0);
    sk.store(lds);
    sv.store(lds + TILE);
  }
  mta_wait_vmem();  // the rows' operands too: a wait for them inside the loop would wait for the next tile as well
  __syncthreads();
  for (int jt = 0; jt < jt1; ++jt) {
    const unsigned kt = lds + (jt & 1) * 2 * TILE, nt = lds + ((jt + 1) & 1) * 2 * TILE;
    if (jt + 1 < jt1) fetch(jt + 1);
    if (jt * BN < wend) {
      if constexpr (BN == 64 && sizeof(T) == 2) {
        w.blocks2(kt, kt + TILE, jt * BN, wall, lane);
      } else {
#pragma unroll
        for (int nb = 0; nb < BN / 32; ++nb) w.block(kt, kt + TILE, 32 * nb, jt * BN + 32 * nb, jt * BN + 32 * nb + 32 > wall, lane);
      }
    }
    if (jt + 1 < jt1) {
      sk.store(nt);
      sv.store(nt + TILE);
    }
    __syncthreads();
  }
  put_row<T, DP>(A, problem, 0, row, w.acc, w.top, half_sum(w.l), h);
}

// between a wave's LDS writes and its lanes' reads of each other's, and back: the LDS serves a wave in order, so only the
// compiler has to keep it
__device__ __forceinline__ void wave_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// Few rows: 32 of a problem to a workgroup; every wave takes all of them and every fourth 32-key block of the workgroup's
// range, through LDS of its own, so that nothing waits for the other waves; their sums are joined at the end.  One query
// against 16 caches of up to 32768 keys, 32 heads of 128 on 8, bf16: 298 us for 1573 MB, 5.3 TB/s, bound by memory,
// and 7 us for the join of its ranges.
template <typename T, int DP>
__global__ __launch_bounds__(THREADS, forward_waves<T>(DP)) void mha_few_kernel(MhaArgs A) {
  typedef Tile<T, DP> TL;
  constexpr int TILE = 32 * TL::ROW_BYTES;
  extern __shared__ char shared[];  // [wave][K block | V block]
  const unsigned lds = lds_base(shared);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int R = A.G * A.Tq, ntile = (R + 31) / 32;
  int problem, tile;
  if (!place(A.B * A.Hkv, ntile * A.splits, problem, tile)) return;
  const int split = tile % A.splits;
  tile /= A.splits;
  if (A.causal) tile = ntile - 1 - tile;  // the longest rows first
  const int b = problem / A.Hkv, hk = problem % A.Hkv, off = A.Tk - A.Tq;
  const int n = A.lens ? min(max(A.lens[b], 0), A.Tk) : A.Tk;
  auto seen_by = [&](int row) { return A.causal ? max(0, min(n, token_of(A, row) + off + 1)) : n; };
  const int row = 32 * tile + (lane & 31);
  const int kend = seen_by(min(32 * tile + 32, R) - 1), kall = seen_by(32 * tile);
  const int j1 = min((kend + 31) / 32, (split + 1) * A.split_tiles);  // 32-key blocks
  Rows<T, DP> w;
  w.start(A.scale, A.D);
  {
    const int t = token_of(A, min(row, R - 1));
    w.see = row < R ? seen_by(row) : 0;
    load_frags<T, DP>(w.q, row < R ? at<T>(A.q, A.qs, b, t, hk * A.G + row - t * A.G) : nullptr, A.D, h);
  }
  typedef Stage<T, DP, 32, 64> ST;
  ST sk, sv;
  const T* kp = at<T>(A.k, A.ks, b, 0, hk) + ST::elem();
  const T* vp = at<T>(A.v, A.vs, b, 0, hk) + ST::elem();
  auto fetch = [&](int j) {
    sk.load(kp + (long)j * 32 * A.ks[1], A.ks[1], n - j * 32, A.D);
    sv.load(vp + (long)j * 32 * A.vs[1], A.vs[1], n - j * 32, A.D);
  };
  const unsigned kt = lds + wave * 2 * TILE;
  int j = split * A.split_tiles + wave;
  if (j < j1) fetch(j);
  for (; j < j1; j += WAVES) {
    sk.store(kt);
    sv.store(kt + TILE);
    wave_order();
    if (j + WAVES < j1) fetch(j + WAVES);
    w.block(kt, kt + TILE, 0, j * 32, j * 32 + 32 > kall, lane);
    wave_order();
  }
  float l = half_sum(w.l);
  __syncthreads();
  // join the four waves' sums: maxima and sums first, then the rows, one 32-column block at a time
  float* ml = reinterpret_cast<float*>(shared);  // [WAVES][2][32]
  float* rows = ml + WAVES * 64;              // [WAVES][32 columns][33]
  if (h == 0) {
    ml[wave * 64 + lane] = w.top;
    ml[wave * 64 + 32 + lane] = l;
  }
  __syncthreads();
  float m = -INFINITY;
#pragma unroll
  for (int v = 0; v < WAVES; ++v) m = fmaxf(m, ml[v * 64 + (lane & 31)]);
  const float base = m == -INFINITY ? 0.f : m;
  l = 0.f;
#pragma unroll
  for (int v = 0; v < WAVES; ++v)
    l += ml[v * 64 + 32 + (lane & 31)] * __builtin_amdgcn_exp2f(ml[v * 64 + (lane & 31)] - base);
  const float mine = __builtin_amdgcn_exp2f(w.top - base);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
    for (int r = 0; r < 16; ++r) rows[(wave * 32 + acc_row(r, h)) * 33 + (lane & 31)] = w.acc[d][r] * mine;
    __syncthreads();
    if (wave == 0)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float a = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) a += rows[(v * 32 + acc_row(r, h)) * 33 + (lane & 31)];
        w.acc[d][r] = a;
      }
    __syncthreads();
  }
  if (wave == 0) put_row<T, DP>(A, problem, split, row, w.acc, m, l, h);
}

// joins the key ranges of the rows: one wave a row, 64 ranges at a time
template <typename T>
__global__ __launch_bounds__(THREADS) void mha_join_kernel(MhaArgs A) {
  const int lane = threadIdx.x & 63;
  const long R = (long)A.G * A.Tq, rows = R * A.B * A.Hkv;
  const long i = (long)blockIdx.x * WAVES + (threadIdx.x >> 6);
  if (i >= rows) return;
  const long step = rows * (A.D + 2);
  const float* p = A.part + i * (A.D + 2);
  float top = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
  const bool c0 = lane < A.D, c1 = lane + 64 < A.D;
  for (int s0 = 0; s0 < A.splits; s0 += 64) {
    const int n = min(64, A.splits - s0);
    const float* ps = p + s0 * step;
    const float t = lane < n ? ps[lane * step + A.D] : -INFINITY, part = lane < n ? ps[lane * step + A.D + 1] : 0.f;
    float to = t;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor(to, o, 64));
    to = fmaxf(top, to);
    const float base = to == -INFINITY ? 0.f : to, old = __builtin_amdgcn_exp2f(top - base);
    const float w = __builtin_amdgcn_exp2f(t - base);
    l = l * old + wave_sum(w * part);
    a0 *= old;
    a1 *= old;
    top = to;
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
      const float ws = mta_readlane(w, s);
      if (c0) a0 = fmaf(ws, ps[s * step + lane], a0);
      if (c1) a1 = fmaf(ws, ps[s * step + lane + 64], a1);
    }
  }
  const long problem = i / R;
  const int row = (int)(i % R), b = (int)(problem / A.Hkv), tq = token_of(A, row), hq = (int)(problem % A.Hkv) * A.G + row - tq * A.G;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* o = at<T>(A.o, A.os, b, tq, hq);
  if (c0) o[lane] = (T)(a0 * inv);
  if (c1) o[lane + 64] = (T)(a1 * inv);
  if (lane == 0 && A.lse) A.lse[((long)b * A.H + hq) * A.Tq + tq] = l == 0.f ? -INFINITY : (top + __log2f(l)) * LN2;
}

// Waves on a SIMD (workgroups on a compute unit) that the backward kernels' registers are cut for.  Two instead of one at
// dim 64: 6 x 1500 tokens, 8 heads, fp16, both directions 177 -> 142 us; at dim 128 a wave's sums alone are 128 registers,
// and cut to 256 it spills.
template <typename T>
constexpr int backward_waves(int dp) {
  return dp > 64 ? 1 : 2;
}

// float16 holds P and dS = P (dP - delta) poorly where P or dO is small (below 2^-14 in steps of 2^-24), and dS not at
// all past 65504.  There P is kept times 2^12 for dV (by a shift of its exponent), and dS times a power of two that takes
// max |dO|, of the row (dQ) or of the rows so far that see the key (dK), to 2 .. 4; the sums are divided by them.  Weights stay normal down
// to 2^-26 and 2^-15; dS overflows only past |dP| of 16000 max |dO|, where V's rows add up to as much.
template <typename T>
constexpr bool SCALED = sizeof(T) == 2 && !std::is_same_v<T, __bf16>;
constexpr float SHIFT = 12.f;
__device__ __forceinline__ float ds_scale(float top) {  // top: max |dO|, finite or not
  const int e = __builtin_bit_cast(int, top) >> 23;
  return e == 0 || e == 255 ? 1.f : __builtin_bit_cast(float, (254 - e + 1) << 23);
}

// ---- backward, dQ: one tile of BN keys against a wave's 32 rows ----------------------------------------------------------
// lc, delta: L log2(e) and rowsum(dO * O) of the lane's row; times: its dS is kept times this (SCALED); left: keys of the
// tile that it sees (MASKED)
template <typename T, int DP, int BN, bool MASKED>
__device__ __forceinline__ void dq_tile(unsigned kt, unsigned vt, const typename El<T>::frag (&qf)[DP / 16],
                                        const typename El<T>::frag (&dof)[DP / 16], f32x16 (&acc)[DP / 32], float c, float lc, float delta,
                                        float times, int left, int dim, int lane) {
  typedef Tile<T, DP> TL;
  typedef typename El<T>::frag frag;
  const int h = lane >> 5;
  const unsigned kr = kt + TL::row_lane(lane), vr = vt + TL::row_lane(lane), kc = kt + TL::col_lane(lane);
  if constexpr (BN == 64 && sizeof(T) == 2) {
    // as dkv_tile: the weights of one block of 32 keys between the products of the other
    constexpr int N = DP / 8, M = DP / 16;  // products of S and dP, and of the sum, of one block
    f32x16 s[2], dp[2];
    frag df[2][2];
    auto weight = [&](int nb, int r) __attribute__((always_inline)) {
      float d = __builtin_amdgcn_exp2f(fmaf(s[nb][r], c, -lc)) * (SCALED<T> ? fmaf(dp[nb][r], times, -delta * times) : dp[nb][r] - delta);
      if constexpr (MASKED) d = 32 * nb + acc_row(r, h) < left ? d : 0.f;
      df[nb][r >> 3][r & 7] = (T)d;
    };
    stream<2 * N + 2 * M, frag>(
        [&](auto i) __attribute__((always_inline)) {
          constexpr int I = decltype(i)::value, k = I < 2 * N ? I % N : (I - 2 * N) % M, nb = I < 2 * N ? I / N : (I - 2 * N) / M;
          if constexpr (I < 2 * N) return TL::rows((k & 1 ? vr : kr) + 32 * nb * TL::ROW_BYTES, k >> 1);
          else return TL::cols(kc + (32 * nb + 16 * (k / (DP / 32))) * TL::ROW_BYTES, k % (DP / 32), lane);
        },
        [&](auto i, const frag& x) __attribute__((always_inline)) {
          constexpr int I = decltype(i)::value, k = I < 2 * N ? I % N : (I - 2 * N) % M, nb = I < 2 * N ? I / N : (I - 2 * N) / M;
          if constexpr (I < 2 * N) {
            if constexpr ((k & 1) == 0) s[nb] = El<T>::mma(x, qf[k >> 1], k == 0 ? f32x16{} : s[nb]);
            else dp[nb] = El<T>::mma(x, dof[k >> 1], k == 1 ? f32x16{} : dp[nb]);
            if constexpr (nb == 1) {
#pragma unroll
              for (int q = 0; q < 16 / N; ++q) weight(0, k * (16 / N) + q);
            }
          } else {
            constexpr int st = k / (DP / 32), d = k % (DP / 32);
            acc[d] = El<T>::mma(x, df[nb][st], acc[d]);
            if constexpr (nb == 0) {
#pragma unroll
              for (int q = 0; q < 16 / M; ++q) weight(1, k * (16 / M) + q);
            }
          }
        });
    return;
  }
#pragma unroll
  for (int nb = 0; nb < BN / 32; ++nb) {
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      if (16 * kk < dim) {  // what is past it is left out
        s = El<T>::mma(TL::rows(kr + 32 * nb * TL::ROW_BYTES, kk), qf[kk], s);
        dp = El<T>::mma(TL::rows(vr + 32 * nb * TL::ROW_BYTES, kk), dof[kk], dp);
      }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lc)) * (SCALED<T> ? fmaf(dp[r], times, -delta * times) : dp[r] - delta);
      if constexpr (MASKED) s[r] = 32 * nb + acc_row(r, h) < left ? s[r] : 0.f;
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const frag ds = as_frag<T>(s, st);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) acc[d] = El<T>::mma(TL::cols(kc + (32 * nb + 16 * st) * TL::ROW_BYTES, d, lane), ds, acc[d]);
    }
  }
}

// sum over a tile's keys of P * dP (this half's): delta of a row all of whose keys are in LDS
template <typename T, int DP, int BN>
__device__ __forceinline__ float dq_delta(unsigned kt, unsigned vt, const typename El<T>::frag (&qf)[DP / 16],
                                          const typename El<T>::frag (&dof)[DP / 16], float c, float lc, int left, int lane) {
  typedef Tile<T, DP> TL;
  const unsigned kr = kt + TL::row_lane(lane), vr = vt + TL::row_lane(lane);
  float sum = 0.f;
#pragma unroll 1
  for (int nb = 0; nb < BN / 32; ++nb) {
    f32x16 s, dp;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      s = El<T>::mma(TL::rows(kr + 32 * nb * TL::ROW_BYTES, kk), qf[kk], kk == 0 ? f32x16{} : s);
      dp = El<T>::mma(TL::rows(vr + 32 * nb * TL::ROW_BYTES, kk), dof[kk], kk == 0 ? f32x16{} : dp);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      sum += 32 * nb + acc_row(r, lane >> 5) < left ? __builtin_amdgcn_exp2f(fmaf(s[r], c, -lc)) * dp[r] : 0.f;
  }
  return sum;
}

// ---- backward, dQ (and delta) ------------------------------------------------------------------------------------------
// a wave's 32 rows: operands, statistics, sums; row lane & 31 is this lane's
template <typename T, int DP>
struct GradRows {
  typename El<T>::frag q[DP / 16], dout[DP / 16];
  f32x16 acc[DP / 32];
  float c, lc, delta, times;
  int see;
  long stat;
  bool real;

  // first: the workgroup that leaves the rows' statistics for the dK / dV kernel
  __device__ __forceinline__ void start(const MhaArgs& A, int b, int hk, int row, int n, bool first, int lane) {
    const int h = lane >> 5, R = A.G * A.Tq;
    real = row < R;
    const int tq = real ? row / A.G : 0, hq = hk * A.G + (real ? row % A.G : 0);
    see = real ? (A.causal ? min(n, tq + A.Tk - A.Tq + 1) : n) : 0;
    stat = ((long)b * A.H + hq) * A.Tq + tq;
    load_frags<T, DP>(q, real ? at<T>(A.q, A.qs, b, tq, hq) : nullptr, A.D, h);
    load_frags<T, DP>(dout, real ? at<T>(A.dout, A.dos, b, tq, hq) : nullptr, A.D, h);
    times = 1.f;
    if constexpr (SCALED<T>) {
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)dout[kk][j]));
      top = half_max(top);
      times = ds_scale(top);
      if (real && h == 0 && first) A.delta[(long)A.B * A.H * A.Tq + stat] = top;
    }
    delta = 0.f;
    typename El<T>::frag of[DP / 16];
    load_frags<T, DP>(of, real ? at<T>(A.o, A.os, b, tq, hq) : nullptr, A.D, h);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)of[kk][j], (float)dout[kk][j], delta);
    delta = half_sum(delta);
    c = A.scale * LOG2E;
    lc = real ? A.lse[stat] * LOG2E : INFINITY;
    if (lc == -INFINITY) lc = INFINITY;  // a row that sees nothing: every exponential is 0
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = f32x16{};
  }
  template <int BN>
  __device__ __forceinline__ void tile(unsigned kt, unsigned vt, int key0, int all, int D, int lane) {
    if (key0 + BN > all) dq_tile<T, DP, BN, true>(kt, vt, q, dout, acc, c, lc, delta, times, see - key0, D, lane);
    else dq_tile<T, DP, BN, false>(kt, vt, q, dout, acc, c, lc, delta, times, 0, D, lane);
  }
};

// Many rows: 128 of a problem to a workgroup, 32 to a wave, walking the key tiles (4096 tokens causal, 32 heads of 128 on
// 8, bf16: 354 us, 0.58 PFLOP/s with one wave a SIMD; 6 x 1500, 8 of 64, fp16: 50 us); dq_splits > 1: a range of
// them, summed by a further launch
template <typename T, int DP, int BN>
__global__ __launch_bounds__(THREADS, backward_waves<T>(DP)) void mha_dq_kernel(MhaArgs A) {
  typedef Tile<T, DP> TL;
  constexpr int TILE = BN * TL::ROW_BYTES, BM = 32 * WAVES;
  extern __shared__ char shared[];  // [2][K tile | V tile]
  const unsigned lds = lds_base(shared);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int R = A.G * A.Tq, ntile = (R + BM - 1) / BM;
  int problem, tile;
  if (!place(A.B * A.Hkv, ntile * A.dq_splits, problem, tile)) return;
  const int split = tile % A.dq_splits;
  tile /= A.dq_splits;
  if (A.causal) tile = ntile - 1 - tile;  // the longest rows first
  const int b = problem / A.Hkv, hk = problem % A.Hkv, off = A.Tk - A.Tq;
  const int n = A.lens ? min(max(A.lens[b], 0), A.Tk) : A.Tk;
  const int t_lo = tile * BM / A.G, t_hi = (min((tile + 1) * BM, R) - 1) / A.G;
  const int kend = A.causal ? max(0, min(n, t_hi + off + 1)) : n;
  const int kall = A.causal ? max(0, min(n, t_lo + off + 1)) : n;
  const int jt0 = split * A.dq_split_tiles, jt1 = min((kend + BN - 1) / BN, jt0 + A.dq_split_tiles);
  GradRows<T, DP> w;
  w.start(A, b, hk, tile * BM + 32 * wave + (lane & 31), n, split == 0, lane);
  typedef Stage<T, DP, BN> ST;
  ST sk, sv;
  const T* kp = at<T>(A.k, A.ks, b, 0, hk) + ST::elem();
  const T* vp = at<T>(A.v, A.vs, b, 0, hk) + ST::elem();
  auto fetch = [&](int jt) {
    sk.load(kp + (long)jt * BN * A.ks[1], A.ks[1], n - jt * BN, A.D);
    sv.load(vp + (long)jt * BN * A.vs[1], A.vs[1], n - jt * BN, A.D);
  };
  // Rows of few keys: out rounded to 16 bits, and made of weights rounded to 16, is not exact enough for a delta that
  // nearly equals dP (their gradients were off by 2.1 instead of 1.4 roundings).  Their two tiles fit into the two buffers,
  // so delta is summed from P and dP in fp32 first.
  const bool few = sizeof(T) == 2 && split == 0 && kend <= 2 * BN;
  if (jt0 < jt1) {
    fetch(jt0);
    sk.store(lds);
    sv.store(lds + TILE);
    if (few && jt1 > 1) {  // (split 0 starts at tile 0)
      fetch(1);
      sk.store(lds + 2 * TILE);
      sv.store(lds + 3 * TILE);
    }
  }
  mta_wait_vmem();  // the row's operands too: a wait for them inside the loop would wait for the next tile as well
  __syncthreads();
  if (few) {
    w.delta = 0.f;
    for (int jt = 0; jt < jt1; ++jt)
      w.delta += dq_delta<T, DP, BN>(lds + jt * 2 * TILE, lds + jt * 2 * TILE + TILE, w.q, w.dout, w.c, w.lc, w.see - jt * BN, lane);
    w.delta = half_sum(w.delta);
  }
  if (w.real && h == 0 && split == 0) A.delta[w.stat] = w.delta;
  for (int jt = jt0; jt < jt1; ++jt) {
    const unsigned kt = lds + ((jt - jt0) & 1) * 2 * TILE, vt = kt + TILE;
    const bool more = !few && jt + 1 < jt1;
    if (more) fetch(jt + 1);
    w.template tile<BN>(kt, vt, jt * BN, kall, A.D, lane);
    if (more) {
      const unsigned nt = lds + ((jt + 1 - jt0) & 1) * 2 * TILE;
      sk.store(nt);
      sv.store(nt + TILE);
    }
    __syncthreads();
  }
  if (!w.real) return;
  const float back = 1.f / w.times;
  const int row = tile * BM + 32 * wave + (lane & 31), tq = row / A.G;
  T* o = at<T>(A.dq, A.dqs, b, tq, hk * A.G + row - tq * A.G);
  float* part = A.part + (((long)split * A.B * A.Hkv + problem) * R + row) * A.D;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 32 * d + 8 * i + 4 * h;
      if (col >= A.D) continue;
      const f32x4 x = {w.acc[d][4 * i] * back, w.acc[d][4 * i + 1] * back, w.acc[d][4 * i + 2] * back, w.acc[d][4 * i + 3] * back};
      if (A.dq_splits > 1) *reinterpret_cast<f32x4*>(part + col) = x;
      else store4<T>(o + col, x[0] * A.scale, x[1] * A.scale, x[2] * A.scale, x[3] * A.scale);
    }
}

// The sums of four waves over one 32 x 32 block: every wave gets rows 8 wave + 4 h .. + 3 of its lane's column.
// rows: [WAVES][32][33] floats of LDS.
__device__ __forceinline__ f32x4 join_waves(float* rows, const f32x16& acc, int wave, int lane) {
  const int h = lane >> 5;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 16; ++r) rows[(wave * 32 + acc_row(r, h)) * 33 + (lane & 31)] = acc[r];
  __syncthreads();
  f32x4 a = {};
#pragma unroll
  for (int v = 0; v < WAVES; ++v)
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] += rows[(v * 32 + 8 * wave + 4 * h + j) * 33 + (lane & 31)];
  return a;
}
constexpr int JOIN_BYTES = WAVES * 32 * 33 * 4;

// Few rows: 32 of a problem to a workgroup; as in the forward, its waves share the keys and add their sums.
template <typename T, int DP>
__global__ __launch_bounds__(THREADS, backward_waves<T>(DP)) void mha_dq_few_kernel(MhaArgs A) {
  typedef Tile<T, DP> TL;
  constexpr int TILE = 32 * TL::ROW_BYTES;
  extern __shared__ char shared[];  // [wave][K block | V block], delta [wave][32]
  const unsigned lds = lds_base(shared);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int R = A.G * A.Tq, ntile = (R + 31) / 32;
  int problem, tile;
  if (!place(A.B * A.Hkv, ntile, problem, tile)) return;
  if (A.causal) tile = ntile - 1 - tile;
  const int b = problem / A.Hkv, hk = problem % A.Hkv, off = A.Tk - A.Tq;
  const int n = A.lens ? min(max(A.lens[b], 0), A.Tk) : A.Tk;
  auto seen_by = [&](int row) { return A.causal ? max(0, min(n, token_of(A, row) + off + 1)) : n; };
  const int kend = seen_by(min(32 * tile + 32, R) - 1), kall = seen_by(32 * tile);
  const int j1 = (kend + 31) / 32;
  const int row = 32 * tile + (lane & 31);
  GradRows<T, DP> w;
  w.start(A, b, hk, row, n, wave == 0, lane);
  typedef Stage<T, DP, 32, 64> ST;
  ST sk, sv;
  const T* kp = at<T>(A.k, A.ks, b, 0, hk) + ST::elem();
  const T* vp = at<T>(A.v, A.vs, b, 0, hk) + ST::elem();
  auto fetch = [&](int j) {
    sk.load(kp + (long)j * 32 * A.ks[1], A.ks[1], n - j * 32, A.D);
    sv.load(vp + (long)j * 32 * A.vs[1], A.vs[1], n - j * 32, A.D);
  };
  const unsigned kt = lds + wave * 2 * TILE;
  int j = wave;
  if (j < j1) fetch(j);
  if (kend <= 32 * WAVES) {  // delta from P and dP, as above: a wave has one block
    float part = 0.f;
    if (j < j1) {
      sk.store(kt);
      sv.store(kt + TILE);
      wave_order();
      part = dq_delta<T, DP, 32>(kt, kt + TILE, w.q, w.dout, w.c, w.lc, w.see - j * 32, lane);
    }
    part = half_sum(part);
    float* parts = reinterpret_cast<float*>(shared + WAVES * 2 * TILE);
    if (h == 0) parts[wave * 32 + lane] = part;
    __syncthreads();
    w.delta = 0.f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) w.delta += parts[v * 32 + (lane & 31)];
  }
  if (w.real && h == 0 && wave == 0) A.delta[w.stat] = w.delta;
  for (; j < j1; j += WAVES) {
    sk.store(kt);
    sv.store(kt + TILE);
    wave_order();
    if (j + WAVES < j1) fetch(j + WAVES);
    w.template tile<32>(kt, kt + TILE, j * 32, kall, A.D, lane);
    wave_order();
  }
  const float times = A.scale / w.times;
  const int tq = min(row, R - 1) / A.G;
  T* o = at<T>(A.dq, A.dqs, b, tq, hk * A.G + min(row, R - 1) - tq * A.G);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) {
    const f32x4 a = join_waves(reinterpret_cast<float*>(shared), w.acc[d], wave, lane);
    const int col = 32 * d + 8 * wave + 4 * h;
    if (w.real && col < A.D) store4<T>(o + col, a[0] * times, a[1] * times, a[2] * times, a[3] * times);
  }
}

template <typename T, int DP, int BR>
constexpr int dkv_buffer() {
  return (2 * BR * DP * (int)sizeof(T) + (SCALED<T> ? 4 * BR + 1 : 3 * BR) * 4 + 1023) / 1024 * 1024;
}

// ---- backward, dK and dV: one tile of BR rows against a wave's 32 keys --------------------------------------------------
// qt, dot: LDS tiles; f: the rows' L log2(e), delta and the keys each sees, BR of each
template <typename T, int DP, int BR, bool MASKED>
__device__ __forceinline__ void dkv_tile(unsigned qt, unsigned dot, unsigned f, const typename El<T>::frag (&kf)[DP / 16],
                                         const typename El<T>::frag (&vf)[DP / 16], f32x16 (&dk)[DP / 32], f32x16 (&dv)[DP / 32], float c,
                                         float times, int key, int dim, int lane) {
  typedef typename El<T>::frag frag;
  typedef Tile<T, DP> TL;
  const int h = lane >> 5;
  const unsigned qr = qt + TL::row_lane(lane), dor = dot + TL::row_lane(lane), qc = qt + TL::col_lane(lane), doc = dot + TL::col_lane(lane);
  f += 16 * h;
  if constexpr (BR == 64 && sizeof(T) == 2) {
    // Two blocks of 32 rows in four phases of N products: S and dP of block 0; of block 1, and the weights of block 0;
    // the sums of block 0, and the weights of block 1; the sums of block 1.
    constexpr int N = DP / 8, PER = 16 / N > 0 ? 16 / N : 1;  // products of a phase; weights computed in one step
    f32x16 s[2], dp[2];
    frag pf[2][2], df[2][2];
    f32x4 lc[4], de[4];
    auto stats = [&](int nb, int i) __attribute__((always_inline)) {
      lc[i] = lds_get<f32x4>(f + 4 * (32 * nb + 8 * i));
      de[i] = lds_get<f32x4>(f + 4 * (BR + 32 * nb + 8 * i));
    };
    auto weight = [&](int nb, int r) __attribute__((always_inline)) {
      float p = __builtin_amdgcn_exp2f(fmaf(s[nb][r], c, -lc[r >> 2][r & 3])), d = p * (dp[nb][r] - de[r >> 2][r & 3]);
      if constexpr (SCALED<T>) d *= times;
      if constexpr (MASKED) {
        const bool sees = key < lds_get<int>(f + 4 * (2 * BR + 32 * nb + acc_row(r, 0)));
        p = sees ? p : 0.f;
        d = sees ? d : 0.f;
      }
      pf[nb][r >> 3][r & 7] = (T)p;
      df[nb][r >> 3][r & 7] = (T)d;
    };
    stream<4 * N, frag>(
        [&](auto i) __attribute__((always_inline)) {
          constexpr int ph = decltype(i)::value / N, k = decltype(i)::value % N, nb = ph & 1;
          if constexpr (ph < 2) return TL::rows((k & 1 ? dor : qr) + 32 * nb * TL::ROW_BYTES, k >> 1);
          else return TL::cols((k & 1 ? qc : doc) + (32 * nb + 16 * ((k >> 1) / (DP / 32))) * TL::ROW_BYTES, (k >> 1) % (DP / 32), lane);
        },
        [&](auto i, const frag& x) __attribute__((always_inline)) {
          constexpr int ph = decltype(i)::value / N, k = decltype(i)::value % N, nb = ph & 1;
          if constexpr (ph < 2) {
            if constexpr ((k & 1) == 0) s[nb] = El<T>::mma(x, kf[k >> 1], k == 0 ? f32x16{} : s[nb]);
            else dp[nb] = El<T>::mma(x, vf[k >> 1], k == 1 ? f32x16{} : dp[nb]);
          } else {
            constexpr int st = (k >> 1) / (DP / 32), d = (k >> 1) % (DP / 32);
            if constexpr ((k & 1) == 0) dv[d] = El<T>::mma(x, pf[nb][st], dv[d]);
            else dk[d] = El<T>::mma(x, df[nb][st], dk[d]);
          }
          if constexpr (ph == 0) {  // block 0's statistics with its last products
            if constexpr (N >= 8 && k >= N - 4) stats(0, k - (N - 4));
            if constexpr (N < 8 && k == N - 1)
              for (int q = 0; q < 4; ++q) stats(0, q);
          }
          if constexpr (ph == 1 || ph == 2) {
#pragma unroll
            for (int q = 0; q < PER; ++q) weight(ph - 1, k * PER + q);
          }
          // four rows' are replaced by block 1's as soon as they have been used
          if constexpr (ph == 1 && (k + 1) * PER % 4 == 0) stats(1, (k + 1) * PER / 4 - 1);
        });
    return;
  }
#pragma unroll
  for (int nb = 0; nb < BR / 32; ++nb) {
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      if (16 * kk < dim) {  // what is past it is left out
        s = El<T>::mma(TL::rows(qr + 32 * nb * TL::ROW_BYTES, kk), kf[kk], s);
        dp = El<T>::mma(TL::rows(dor + 32 * nb * TL::ROW_BYTES, kk), vf[kk], dp);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned at = f + 4 * (32 * nb + 8 * i);
      const f32x4 lc = lds_get<f32x4>(at), de = lds_get<f32x4>(at + 4 * BR);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * i + j;
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lc[j]));
        dp[r] = s[r] * (dp[r] - de[j]);
        if constexpr (SCALED<T>) dp[r] *= times;
        if constexpr (MASKED) {
          const bool sees = key < lds_get<int>(at + 8 * BR + 4 * j);
          s[r] = sees ? s[r] : 0.f;
          dp[r] = sees ? dp[r] : 0.f;
        }
      }
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const frag p = as_frag<T>(s, st), ds = as_frag<T>(dp, st);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        dv[d] = El<T>::mma(TL::cols(doc + (32 * nb + 16 * st) * TL::ROW_BYTES, d, lane), p, dv[d]);
        dk[d] = El<T>::mma(TL::cols(qc + (32 * nb + 16 * st) * TL::ROW_BYTES, d, lane), ds, dk[d]);
      }
    }
  }
}

// ---- backward, dK and dV -----------------------------------------------------------------------------------------------
// S = Q K^T is not transposed here: a lane owns ONE key and 16 of 32 rows, so P and dS are the B operands of
// dV^T = dO^T P and dK^T = Q^T dS.  Runs after the dQ kernels, which write delta.

// tiles of BR rows of one problem, staged by NT threads: the workgroup's, or a wave's
template <typename T, int DP, int BR, int NT>
struct RowTiles {
  static constexpr int TILE = BR * Tile<T, DP>::ROW_BYTES;
  typedef Stage<T, DP, BR, NT> ST;
  const MhaArgs& A;
  const int b, hk, n, R, e0, per_pass, me;
  const int blind;  // rows in front that see no key: they repeat the first that sees one, as rows past the end the last
  const bool even;  // G divides the rows of a pass: a thread's rows are the same query head's, and their tokens a step apart
  const T *qp, *dop;
  ST sq, sdo;
  float st_l = 0.f, st_d = 0.f, st_top = 0.f;
  int st_see = 0;

  __device__ __forceinline__ RowTiles(const MhaArgs& A, int b, int hk, int n)
      : A(A), b(b), hk(hk), n(n), R(A.G * A.Tq), e0(ST::elem() < A.D ? ST::elem() : 0), per_pass(ST::RPI / A.G), me(threadIdx.x % NT),
        blind(A.causal && A.Tq > A.Tk ? A.G * (A.Tq - A.Tk) : 0), even(ST::RPI % A.G == 0) {
    const int t0 = token_of(A, ST::row()), h0 = hk * A.G + ST::row() - t0 * A.G;
    qp = at<T>(A.q, A.qs, b, t0, h0) + e0;
    dop = at<T>(A.dout, A.dos, b, t0, h0) + e0;
  }
  __device__ __forceinline__ void fetch(int it) {
    if (even && it * BR >= blind && (it + 1) * BR <= R) {
#pragma unroll
      for (int i = 0; i < ST::N; ++i) {
        sq.r[i] = *reinterpret_cast<const u32x4*>(qp + (long)(it * ST::N + i) * (per_pass * A.qs[1]));
        sdo.r[i] = *reinterpret_cast<const u32x4*>(dop + (long)(it * ST::N + i) * (per_pass * A.dos[1]));
      }
    } else {
      auto row_of = [&](const void* p, const long(&st)[3], int r) {
        const int t = token_of(A, it * BR + r);
        return at<T>(p, st, b, t, hk * A.G + it * BR + r - t * A.G);
      };
      sq.gather([&](int r) { return row_of(A.q, A.qs, r); }, e0, blind - it * BR, R - it * BR);
      sdo.gather([&](int r) { return row_of(A.dout, A.dos, r); }, e0, blind - it * BR, R - it * BR);
    }
    const int row = it * BR + me;
    if (me < BR && row < R) {  // as they are: a use here would wait for every load above
      const int t = token_of(A, row);
      const long s = ((long)b * A.H + hk * A.G + row - t * A.G) * A.Tq + t;
      st_l = A.lse[s];
      st_d = A.delta[s];
      if constexpr (SCALED<T>) st_top = A.delta[(long)A.B * A.H * A.Tq + s];
      st_see = A.causal ? min(n, t + A.Tk - A.Tq + 1) : n;
    } else {
      st_l = -INFINITY;
      st_d = st_top = 0.f;
      st_see = 0;
    }
  }
  // Q rows, dO rows, then L log2(e), delta, the keys each row sees; (SCALED) each row's max |dO|, the tile's
  __device__ __forceinline__ void put(unsigned t) const {
    sq.store(t);
    sdo.store(t + TILE);
    if (me < BR) {
      const unsigned f = t + 2 * TILE + 4 * me;
      lds_put(f, st_l == -INFINITY ? INFINITY : fmaf(st_l, LOG2E, SCALED<T> ? -SHIFT : 0.f));  // sees nothing, or is not there: P = 0
      lds_put(f + 4 * BR, st_d);
      lds_put(f + 8 * BR, st_see);
    }
    if constexpr (SCALED<T>) {
      static_assert(BR <= 64, "the rows' maximum is one wave's");
      if (me < 64) {
        float top = st_see > 0 ? st_top : 0.f;
        if (me < BR) lds_put(t + 2 * TILE + 12 * BR + 4 * me, top);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        if (me == 0) lds_put(t + 2 * TILE + 16 * BR, top);
      }
    }
  }
};

// a wave's 32 keys: operands and sums; key lane & 31 is this lane's
template <typename T, int DP>
struct GradKeys {
  typename El<T>::frag k[DP / 16], v[DP / 16];
  f32x16 dk[DP / 32], dv[DP / 32];
  // SCALED, of the lane's key: dS is 2^12 P times (dP - delta) times this; the maximum so far of the rows that see the key
  float times = exp2f(-SHIFT), top = 0.f;

  __device__ __forceinline__ void start(const MhaArgs& A, int b, int hk, int key, bool real, int h) {
    load_frags<T, DP>(k, real ? at<T>(A.k, A.ks, b, key, hk) : nullptr, A.D, h);
    load_frags<T, DP>(v, real ? at<T>(A.v, A.vs, b, key, hk) : nullptr, A.D, h);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = f32x16{};
  }
  template <int BR, bool MASKED>
  __device__ __forceinline__ void tile(unsigned qt, float c, int key, int D, int lane) {
    constexpr int TILE = BR * Tile<T, DP>::ROW_BYTES;
    if constexpr (SCALED<T>) {
      const unsigned f = qt + 2 * TILE;
      float now = 0.f;
      if constexpr (MASKED) {
#pragma unroll 4
        for (int r = 0; r < BR; r += 4) {
          const f32x4 x = lds_get<f32x4>(f + 12 * BR + 4 * r);
          const u32x4 sees = lds_get<u32x4>(f + 8 * BR + 4 * r);
#pragma unroll
          for (int j = 0; j < 4; ++j) now = fmaxf(now, key < (int)sees[j] ? x[j] : 0.f);
        }
      } else {
        now = lds_get<float>(f + 16 * BR);
      }
      if (__any(now > top)) {
        const float next = now > top ? ds_scale(now) * exp2f(-SHIFT) : times, by = next / times;
        if (__any(by != 1.f)) {
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[d][r] *= by;
        }
        times = next;
        top = fmaxf(top, now);
      }
    }
    dkv_tile<T, DP, BR, MASKED>(qt, qt + TILE, qt + 2 * TILE, k, v, dk, dv, c, times, key, D, lane);
  }
  __device__ __forceinline__ void finish(bool real) {
    if constexpr (SCALED<T>) {
      const float back = exp2f(-SHIFT) / times;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          dk[d][r] *= back;
          dv[d][r] *= exp2f(-SHIFT);
        }
    }
    if (!real)  // a key that is not there: its lane's products are of zeros and of rows that do not see it
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = f32x16{};
  }
};

// the row tiles of BR that keys key0 .. key1 - 1 need: from the first that sees one of them; in those before `all` some row
// does not see some of them; none where the sequence ends before them
struct Walk {
  int it0, it1, all;
  __device__ __forceinline__ Walk(const MhaArgs& A, int n, int key0, int key1, int BR) {
    const long R = (long)A.G * A.Tq, off = A.Tk - A.Tq;
    it0 = A.causal ? (int)(min(max(0L, key0 - off) * A.G, R) / BR) : 0;
    it1 = key0 < n ? (int)((R + BR - 1) / BR) : it0;
    all = A.causal ? (int)((min(max(0L, key1 - 1 - off) * A.G, R) + BR - 1) / BR) : 0;
  }
};

// Many keys: 128 of a problem to a workgroup, 32 to a wave, walking the rows in tiles of BR.  With causal order key tile i
// is seen by fewer rows the later it is: a workgroup takes tiles i and N - 1 - i, whose rows add up to the same number for
// every i.  (The two calls above: 379 us, 0.73 PFLOP/s, and 70 us.)  kv_splits > 1: a kv_splits-th of each tile's rows,
// summed by a further launch.
template <typename T, int DP, int BR>
__global__ __launch_bounds__(THREADS, backward_waves<T>(DP)) void mha_dkv_kernel(MhaArgs A) {
  constexpr int BK = 32 * WAVES, BUF = dkv_buffer<T, DP, BR>();
  extern __shared__ char shared[];  // [2][BUF]
  const unsigned lds = lds_base(shared);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const int ntile = (A.Tk + BK - 1) / BK;
  int problem, place0;
  if (!place(A.B * A.Hkv, (A.causal ? (ntile + 1) / 2 : ntile) * A.kv_splits, problem, place0)) return;
  const int split = place0 % A.kv_splits;
  place0 /= A.kv_splits;
  const int b = problem / A.Hkv, hk = problem % A.Hkv;
  const int n = A.lens ? min(max(A.lens[b], 0), A.Tk) : A.Tk;
  const float c = A.scale * LOG2E;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const int tile = pass == 0 ? place0 : ntile - 1 - place0;
    if (pass == 1 && (!A.causal || tile == place0)) break;
    const int key = tile * BK + 32 * wave + (lane & 31);
    GradKeys<T, DP> w;
    w.start(A, b, hk, key, key < n, h);
    const Walk x(A, n, tile * BK, (tile + 1) * BK, BR);
    const int it0 = x.it0 + (int)((long)(x.it1 - x.it0) * split / A.kv_splits);
    const int it1 = x.it0 + (int)((long)(x.it1 - x.it0) * (split + 1) / A.kv_splits);
    RowTiles<T, DP, BR, THREADS> rows(A, b, hk, n);
    if (it0 < it1) {
      rows.fetch(it0);
      rows.put(lds);
    }
    mta_wait_vmem();  // the keys' operands too: a wait for them inside the loop would wait for the next tile as well
    __syncthreads();
    auto walk = [&](auto masked, int from, int to) {
#pragma unroll 1
      for (int it = from; it < to; ++it) {
        if (it + 1 < it1) rows.fetch(it + 1);
        w.template tile<BR, decltype(masked)::value>(lds + ((it - it0) & 1) * BUF, c, key, A.D, lane);
        if (it + 1 < it1) rows.put(lds + ((it + 1 - it0) & 1) * BUF);
        __syncthreads();
      }
    };
    const int all = min(it1, max(it0, x.all));
    walk(std::true_type{}, it0, all);
    walk(std::false_type{}, all, it1);
    w.finish(key < n);
    if (key >= A.Tk) continue;
    T* ok = at<T>(A.dk, A.dks, b, key, hk);
    T* ov = at<T>(A.dv, A.dvs, b, key, hk);
    const long each = (long)A.B * A.Hkv * A.Tk * A.D;
    float* part = A.part + (A.dq_splits > 1 ? (long)A.dq_splits * A.B * A.Hkv * A.G * A.Tq * A.D : 0) + 2 * split * each +
                  ((long)problem * A.Tk + key) * A.D;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = 32 * d + 8 * i + 4 * h;
        if (col >= A.D) continue;
        const f32x4 a = {w.dk[d][4 * i], w.dk[d][4 * i + 1], w.dk[d][4 * i + 2], w.dk[d][4 * i + 3]};
        const f32x4 e = {w.dv[d][4 * i], w.dv[d][4 * i + 1], w.dv[d][4 * i + 2], w.dv[d][4 * i + 3]};
        if (A.kv_splits > 1) {
          *reinterpret_cast<f32x4*>(part + col) = a;
          *reinterpret_cast<f32x4*>(part + each + col) = e;
        } else {
          store4<T>(ok + col, a[0] * A.scale, a[1] * A.scale, a[2] * A.scale, a[3] * A.scale);
          store4<T>(ov + col, e[0], e[1], e[2], e[3]);
        }
      }
  }
}

// Few keys: 32 of a problem to a workgroup, whose waves share the rows, each through LDS of its own, and add their sums.
template <typename T, int DP>
__global__ __launch_bounds__(THREADS, backward_waves<T>(DP)) void mha_dkv_few_kernel(MhaArgs A) {
  constexpr int BUF = dkv_buffer<T, DP, 32>();
  extern __shared__ char shared[];  // [wave][BUF]
  const unsigned lds = lds_base(shared);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  int problem, tile;
  if (!place(A.B * A.Hkv, (A.Tk + 31) / 32, problem, tile)) return;
  const int b = problem / A.Hkv, hk = problem % A.Hkv;
  const int n = A.lens ? min(max(A.lens[b], 0), A.Tk) : A.Tk;
  const int key = tile * 32 + (lane & 31);
  GradKeys<T, DP> w;
  w.start(A, b, hk, key, key < n, h);
  const Walk x(A, n, tile * 32, tile * 32 + 32, 32);
  int it = x.it0 + wave;
  RowTiles<T, DP, 32, 64> rows(A, b, hk, n);
  const unsigned qt = lds + wave * BUF;
  if (it < x.it1) rows.fetch(it);
  for (; it < x.it1; it += WAVES) {
    rows.put(qt);
    wave_order();
    if (it + WAVES < x.it1) rows.fetch(it + WAVES);
    if (it < x.all) w.template tile<32, true>(qt, A.scale * LOG2E, key, A.D, lane);
    else w.template tile<32, false>(qt, A.scale * LOG2E, key, A.D, lane);
    wave_order();
  }
  w.finish(key < n);
  const int real = min(key, A.Tk - 1);
  T* ok = at<T>(A.dk, A.dks, b, real, hk);
  T* ov = at<T>(A.dv, A.dvs, b, real, hk);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) {
    const f32x4 a = join_waves(reinterpret_cast<float*>(shared), w.dk[d], wave, lane);
    const f32x4 e = join_waves(reinterpret_cast<float*>(shared), w.dv[d], wave, lane);
    const int col = 32 * d + 8 * wave + 4 * h;
    if (key >= A.Tk || col >= A.D) continue;
    store4<T>(ok + col, a[0] * A.scale, a[1] * A.scale, a[2] * A.scale, a[3] * A.scale);
    store4<T>(ov + col, e[0], e[1], e[2], e[3]);
  }
}

// Sums over split axes, all of a call in one launch: part (splits, problems, rows, D) every `step` floats -> out, times
// `scale`; row r of problem (b, hk) is token r / G of head hk * G + r % G.
struct Sum {
  const float* part;
  void* out;
  long s[3], step, rows, items;  // items: 4-element pieces
  int splits, G;
  float scale;
};
struct Sums {
  Sum a[3];
  int n, Hkv, D;
};
template <typename T>
__global__ __launch_bounds__(THREADS) void mha_sum_kernel(Sums S) {
  long i = (long)blockIdx.x * THREADS + threadIdx.x;
  int k = 0;
  while (k < S.n && i >= S.a[k].items) i -= S.a[k++].items;
  if (k == S.n) return;
  const Sum& a = S.a[k];
  const int quads = S.D / 4, d = (int)(i % quads) * 4;
  const long row = i / quads, r = row % a.rows;
  const int problem = (int)(row / a.rows), b = problem / S.Hkv, hk = problem % S.Hkv;
  const float* p = a.part + row * S.D + d;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(p + s * a.step);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += x[j];
  }
  T* o = static_cast<T*>(a.out) + b * a.s[0] + r / a.G * a.s[1] + (hk * a.G + r % a.G) * a.s[2] + d;
  store4<T>(o, sum[0] * a.scale, sum[1] * a.scale, sum[2] * a.scale, sum[3] * a.scale);
}

// ---- rotary positions of packed q, k -----------------------------------------------------------------------------------
// x (tokens of `seq`-long sequences, row stride ld): heads x D of interleaved pairs (2 i, 2 i + 1) turned by
// sign * position * base^(-2 i / D), in place.  The angle's product is in 64 bits: positions are not bounded here.
template <typename T>
__global__ __launch_bounds__(THREADS) void rope_kernel(T* x, long tokens, int seq, long ld, int heads, int D, double base,
                                                       float sign) {
  const int half = D / 2;
  const long i = (long)blockIdx.x * THREADS + threadIdx.x;
  if (i >= tokens * half) return;
  const long tok = i / half;
  const int d = (int)(i % half);
  const double turn = (double)(tok % seq) * exp2(-2.0 * d / D * log2(base)) * 0.15915494309189535;  // / (2 pi)
  const float a = (float)(turn - floor(turn)) * 6.283185307179586f;
  const float cs = cosf(a), sn = sinf(a) * sign;
  T* p = x + tok * ld + 2 * d;
  for (int hd = 0; hd < heads; ++hd, p += D) {
    const float u = (float)p[0], v = (float)p[1];
    p[0] = (T)(u * cs - v * sn);
    p[1] = (T)(v * cs + u * sn);
  }
}

// 0, or why a kernel was not started: 2 more threads than a launch holds (2^32 - 1), 3 the LDS, 4 the launch itself
template <typename... P>
int start(void (*kernel)(P...), long grid, int lds, hipStream_t st, P... args) {
  if (grid < 1 || grid > 0xffffffffL / THREADS) return 2;
  const void* f = reinterpret_cast<const void*>(kernel);
  if (lds > 64 * 1024 && hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return 3;
  void* p[] = {&args...};
  return hipLaunchKernel(f, dim3((unsigned)grid), dim3(THREADS), p, lds, st) == hipSuccess ? 0 : 4;
}
int launch(void (*kernel)(MhaArgs), long grid, int lds, const MhaArgs& A, hipStream_t st) { return start<MhaArgs>(kernel, grid, lds, st, A); }

// keys of a tile of the many-row kernels, rows of one of the many-key kernel
template <typename T>
constexpr int BLOCK = 64 * 2 / (int)sizeof(T);

// Whether `rows` (keys) of each of P problems are taken by 32 to a workgroup, whose four waves share the other axis, instead
// of 128: where 128 leave some of the card's 256 compute units idle.  Against ranges of the other axis joined by a further
// launch (us): forward, 4 x 512 tokens, 8 heads of 32, bf16 23 -> 6.4; 2 x 1024 causal, 4 of 128 43 -> 16; fp32 3 x 777
// causal, 6 of 40 58 -> 37; one head of 8192 tokens, 128 wide, 76 -> 82.
bool few(long P, long rows) { return rows <= 32 || P * ((rows + 127) / 128) < 256; }
// Backward: in 16 bits, where the other axis is at most 2048; a wave's own tiles of 32 keep its products less busy than
// tiles of 64 that four share.  us in bf16 against ranges, P problems of n tokens: dim 32, 16 of 512 13 / 21, 8 of 2048
// 39 / 49; dim 64, 16 of 585 causal 24 / 44, 8 of 1500 causal 40 / 55, 8 of 2048 62 / 67; dim 128, 16 of 585 causal 41 / 59, 8 of
// 1024 51 / 57.  It costs where one or two problems are long (dim 64, 1 of 2048 46 / 32) and at dims past 64, one workgroup
// on a unit, where 256 do not hold all (8 of 2048 166 / 103, 32 of 512 64 / 58).  In float16 past dim 64 the dK / dV kernel
// spills 140 registers: short axes only there (16 of 256 32 / 37, 16 of 512 causal 48 / 71; but 16 of 64 25 / 20, 8 of
// 1024 72 / 62, 8 of 2048 235 / 114).  In fp32 the registers for both do not suffice: 3 x 777, 6 of 40 141 -> 191.
template <typename T>
bool few_backward(long P, long rows, long other, int dp, bool causal) {
  if (sizeof(T) != 2 || P * ((rows + 127) / 128) >= 256) return false;
  if (SCALED<T> && dp > 64) return other <= (causal ? 512 : 256) && P * ((rows + 31) / 32) <= 256;
  return other <= 2048;
}

// Ranges that `tiles` tiles of a sum are split into: one while `groups` workgroups fill the card, else as many as find a
// place at once, `waves` workgroups on a unit, of at least `least` tiles.
void ranges(long groups, long tiles, long least, int waves, int& splits, int& per) {
  splits = 1;
  per = (int)(tiles < 1 ? 1 : tiles);
  if (groups >= 256 || tiles < 2 * least) return;
  const long places = 256 * waves;
  long p = (tiles * groups + places - 1) / places;
  if (p < least) p = least;
  per = (int)p;
  splits = (int)((tiles + p - 1) / p);
}

// the splits of a call, and the workspace (floats) that they need
template <typename T>
long plan(MhaArgs& A, bool backward) {
  const long R = (long)A.G * A.Tq, P = (long)A.B * A.Hkv;
  const int dp = A.D <= 32 ? 32 : A.D <= 64 ? 64 : 128;
  A.splits = A.dq_splits = A.kv_splits = 1;
  if (!backward) {
    if (few(P, R)) ranges(P * ((R + 31) / 32), (A.Tk + 31) / 32, 2 * WAVES, forward_waves<T>(dp), A.splits, A.split_tiles);
    return A.splits > 1 ? A.splits * P * R * (A.D + 2) : 0;
  }
  constexpr int BN = BLOCK<T>;
  const long kt = (A.Tk + 127) / 128;
  int per;
  if (!few_backward<T>(P, R, A.Tk, dp, A.causal))
    ranges(P * ((R + 127) / 128), (A.Tk + BN - 1) / BN, 2, backward_waves<T>(dp), A.dq_splits, A.dq_split_tiles);
  if (!few_backward<T>(P, A.Tk, R, dp, A.causal))
    ranges(P * (A.causal ? (kt + 1) / 2 : kt), (R + BN - 1) / BN, 4, backward_waves<T>(dp), A.kv_splits, per);
  return (A.dq_splits > 1 ? A.dq_splits * P * R * A.D : 0) + (A.kv_splits > 1 ? 2L * A.kv_splits * P * A.Tk * A.D : 0);
}

template <typename T, int DP>
int fwd(const MhaArgs& A, hipStream_t st) {
  constexpr int BN = BLOCK<T>, ROW = DP * (int)sizeof(T), OWN = WAVES * 2 * 32 * ROW;
  const long R = (long)A.G * A.Tq, P = (long)A.B * A.Hkv;
  if (!few(P, R)) return launch(mha_fwd_kernel<T, DP, BN>, grid_of(P, (R + 127) / 128), 4 * BN * ROW, A, st);
  const int rc = launch(mha_few_kernel<T, DP>, grid_of(P, (R + 31) / 32 * A.splits), OWN > 20 * 1024 ? OWN : 20 * 1024, A, st);
  return rc == 0 && A.splits > 1 ? launch(mha_join_kernel<T>, (R * P + WAVES - 1) / WAVES, 0, A, st) : rc;
}

template <typename T, int DP>
int bwd(const MhaArgs& A, hipStream_t st) {
  constexpr int BN = BLOCK<T>, ROW = DP * (int)sizeof(T), OWN = WAVES * 2 * 32 * ROW + WAVES * 32 * 4;
  constexpr int BUF = dkv_buffer<T, DP, BN>(), OWN_BUF = WAVES * dkv_buffer<T, DP, 32>();
  const long R = (long)A.G * A.Tq, P = (long)A.B * A.Hkv, kt = (A.Tk + 127) / 128;
  int rc = -1;
  if constexpr (sizeof(T) == 2)
    if (few_backward<T>(P, R, A.Tk, DP, A.causal))
      rc = launch(mha_dq_few_kernel<T, DP>, grid_of(P, (R + 31) / 32), OWN > JOIN_BYTES ? OWN : JOIN_BYTES, A, st);
  if (rc < 0) rc = launch(mha_dq_kernel<T, DP, BN>, grid_of(P, (R + 127) / 128 * A.dq_splits), 4 * BN * ROW, A, st);
  if (rc) return rc;
  rc = -1;
  if constexpr (sizeof(T) == 2)
    if (few_backward<T>(P, A.Tk, R, DP, A.causal))
      rc = launch(mha_dkv_few_kernel<T, DP>, grid_of(P, (A.Tk + 31L) / 32), OWN_BUF > JOIN_BYTES ? OWN_BUF : JOIN_BYTES, A, st);
  if (rc < 0) rc = launch(mha_dkv_kernel<T, DP, BN>, grid_of(P, (A.causal ? (kt + 1) / 2 : kt) * A.kv_splits), 2 * BUF, A, st);
  if (rc) return rc;
  Sums S{};
  S.Hkv = A.Hkv;
  S.D = A.D;
  long items = 0;
  auto add = [&](const float* part, void* out, const long(&strides)[3], int splits, long step, long rows, int G, float scale) {
    Sum& a = S.a[S.n++];
    a = Sum{part, out, {strides[0], strides[1], strides[2]}, step, rows, P * rows * (A.D / 4), splits, G, scale};
    items += a.items;
  };
  const float* part = A.part;
  if (A.dq_splits > 1) {
    add(part, A.dq, A.dqs, A.dq_splits, P * R * A.D, R, A.G, A.scale);
    part += A.dq_splits * P * R * A.D;
  }
  if (A.kv_splits > 1) {
    const long all = P * A.Tk * A.D;
    add(part, A.dk, A.dks, A.kv_splits, 2 * all, A.Tk, 1, A.scale);
    add(part + all, A.dv, A.dvs, A.kv_splits, 2 * all, A.Tk, 1, 1.f);
  }
  return S.n ? start<Sums>(mha_sum_kernel<T>, (items + THREADS - 1) / THREADS, 0, st, S) : 0;
}

template <typename T>
int run(const MhaArgs& A, bool backward, hipStream_t st) {
  if (A.D <= 32) return backward ? bwd<T, 32>(A, st) : fwd<T, 32>(A, st);
  if (A.D <= 64) return backward ? bwd<T, 64>(A, st) : fwd<T, 64>(A, st);
  return backward ? bwd<T, 128>(A, st) : fwd<T, 128>(A, st);
}

bool sizes_ok(const MhaArgs* A) {
  return A->D >= 8 && A->D <= 128 && A->D % 8 == 0 && A->G >= 1 && A->Hkv >= 1 && A->H == A->G * A->Hkv &&
         (long)A->G * A->Tq + 256 < 0x7fffffffL && A->Tk < 0x7fffff00;
}

}  // namespace

// sets the call's splits and returns the floats of workspace (A->part) that it needs; negative: unsupported
extern "C" long mta_mha_plan(int dtype, int backward, MhaArgs* A) {
  if (!sizes_ok(A)) return -1;
  switch (dtype) {
    case MHA_BF16: return plan<__bf16>(*A, backward);
    case MHA_F16: return plan<_Float16>(*A, backward);
    case MHA_F32: return plan<float>(*A, backward);
  }
  return -1;
}

// forward: o and lse; backward: dq, dk, dv (and delta).  The splits are mta_mha_plan's.
extern "C" int mta_mha(int dtype, int backward, MhaArgs* A, hipStream_t st) {
  if (!sizes_ok(A)) return 1;
  // row / G for rows below 2^31: with 2^(s-1) < G <= 2^s the error of ceil(2^(31+s) / G) times a row stays below 2^(31+s)
  unsigned s = 0;
  while ((1u << s) < (unsigned)A->G) ++s;
  A->gshift = 31 + s;
  A->gmul = (unsigned)(((1ull << A->gshift) + A->G - 1) / A->G);
  switch (dtype) {
    case MHA_BF16: return run<__bf16>(*A, backward, st);
    case MHA_F16: return run<_Float16>(*A, backward, st);
    case MHA_F32: return run<float>(*A, backward, st);
  }
  return 1;
}

// Whether two tensors (strides >= 0) have an element in common: whole numbers x, each in its range, with
// sum stride * x = b.at - a.at, where a dimension of `a` counts up and one of `b` down, and equal strides are one x.  By
// descending stride, x is taken only where the smaller strides can make up the rest, which for dimensions that lie within
// each other are two values or three.  1 also where the search does not end within its steps.
extern "C" int mta_mha_meet(const MhaBox* a, const MhaBox* b) {
  struct Axis {
    long stride, lo, hi;
  } axes[8];
  int n = 0;
  auto add = [&](long stride, long lo, long hi) {
    if (lo == hi) return;
    int i = 0;
    while (i < n && axes[i].stride > stride) ++i;
    if (i == n || axes[i].stride != stride) {
      for (int j = n++; j > i; --j) axes[j] = axes[j - 1];
      axes[i] = Axis{stride, 0, 0};
    }
    axes[i].lo += lo;
    axes[i].hi += hi;
  };
  for (int k = 0; k < 4; ++k) {
    if (a->sizes[k] == 0 || b->sizes[k] == 0) return 0;
    if (a->strides[k]) add(a->strides[k], 0, a->sizes[k] - 1);
    if (b->strides[k]) add(b->strides[k], 1 - b->sizes[k], 0);
  }
  long least[9] = {}, most[9] = {};  // of axes i ..
  for (int i = n - 1; i >= 0; --i) {
    least[i] = least[i + 1] + axes[i].stride * axes[i].lo;
    most[i] = most[i + 1] + axes[i].stride * axes[i].hi;
  }
  int steps = 1 << 16;
  auto down = [](long x, long y) { return x / y - (x % y != 0 && x < 0); };  // y > 0
  auto search = [&](auto&& self, int i, long rest) -> bool {
    if (i == n) return rest == 0;
    const Axis& x = axes[i];
    long from = -down(most[i + 1] - rest, x.stride), to = down(rest - least[i + 1], x.stride);
    from = from > x.lo ? from : x.lo;
    to = to < x.hi ? to : x.hi;
    for (long v = from; v <= to; ++v)
      if (--steps < 0 || self(self, i + 1, rest - x.stride * v)) return true;
    return false;
  };
  return search(search, 0, b->at - a->at);
}

extern "C" int mta_rope(int dtype, void* x, long tokens, int seq, long ld, int heads, int D, double base, int inverse,
                        hipStream_t st) {
  const long n = tokens * (D / 2);
  if (n <= 0) return 0;
  const long grid = (n + THREADS - 1) / THREADS;
  const float s = inverse ? -1.f : 1.f;
  if (dtype == MHA_BF16) return start(rope_kernel<__bf16>, grid, 0, st, (__bf16*)x, tokens, seq, ld, heads, D, base, s);
  if (dtype == MHA_F32) return start(rope_kernel<float>, grid, 0, st, (float*)x, tokens, seq, ld, heads, D, base, s);
  return 1;
}
