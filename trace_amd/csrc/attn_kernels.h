// Attention and its backward pass (gfx950): the kernels behind trace_attention / trace_attention_backward.
//
//   S = scale q k^T over the visible pairs,  lse_i = log sum_j exp S_ij,  out_i = sum_j exp(S_ij - lse_i) v_j
//   P = exp(S - lse),  delta_i = dout_i . out_i,  dS = P (dout v^T - delta)
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
//
// One pass over the keys with a running maximum and sum; nothing of size Lq x Lk leaves the registers.  Every product is
// a 32x32 matrix instruction, and its operands are chosen so that no result is ever shuffled between lanes: S is
// computed transposed (rows = keys, columns = queries), which leaves lane l with query l & 31 and half of the tile's
// keys -- exactly the second operand of out^T = V^T P^T once the 16 keys of an instruction are taken in the order
// 8a + 4h + i -> slot 8h + 4a + i (h: lane half).  The first operands V^T, K^T, Q^T, dO^T come from LDS images that are
// written transposed and with their keys in that order (TileX); operands read along the head come from TileR.
#pragma once
#include "layer_types.h"

namespace trace {

struct AttnView {
  long sb, sl, sh;      // strides in elements: batch, token, head
};

struct AttnArgs {
  const void *q, *k, *v, *out_in, *dout;
  void *out, *dq, *dk, *dv;
  const float* lse_in;
  float* lse;                        // (B, Hq, Lq)
  float* delta;                      // (B, Hq, Lq), written by the dq kernel, read by the dk / dv kernel
  AttnView vq, vk, vv, vo, vdo, vdq, vdk, vdv;
  int B, Lq, Lk, Hq, Hk, G, D;       // G = Hq / Hk query heads share a key head
  float scale, scale_log2;           // scale, scale * log2(e)
  int causal;
  const int* query_start;            // (B) or null
  const int* key_lengths;            // (B) or null
  const unsigned char* key_mask;     // (B, Lk) or null
  long mask_stride;
  int vec;                           // every pointer and stride 16-byte aligned, D % 8 == 0
  int waves_q, waves_k;              // waves of a workgroup over queries (forward, dq), over keys (dk / dv)
  int splits_q;                      // shares of the keys (attn_dq_kernel), results in part_q: (splits_q, rows, padded D)
  float* part_q;
  int splits;                        // ranges of keys (forward), shares of the queries (attn_dkv_kernel)
  float *part_ml, *part_o;           // their partial results: (rows, splits, 2), (rows, splits, padded D) or
                                     // (splits, {dk, dv}, rows, padded D)
  long items;                        // work items of the launch
};
constexpr int ATTN_MAX_SPLITS = 256;

enum class AttnPass { forward, few, dq, dkv, short_backward };
template <typename T>
int attn_run(AttnPass pass, const AttnArgs& a, hipStream_t st);

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;

// ---- LDS images of a tile of ROWS tokens x DP head elements -----------------------------------------------------
// TileR: token-major; the 16 bytes of padding put the 16-byte pieces of 16 consecutive rows on different banks.
template <typename T, int DP>
struct TileR {
  static constexpr int S = DP + 16 / (int)sizeof(T);
  static __device__ __forceinline__ int frag(int row, int c, int half) { return row * S + c * 16 + half * 8; }
};
// TileX: transposed, element (d, token) with the tokens of each group of 16 in slot order.  The group's two blocks of
// eight are exchanged with those of other groups by the d >> 4 term: rows 16 apart would otherwise meet on the same banks
// when eight lanes write eight head elements each (rows are padded, so reads along 32 rows do not conflict).
template <typename T, int ROWS>
struct TileX {
  static constexpr int S = ROWS + 16 / (int)sizeof(T);
  static constexpr int M = ROWS / 8 - 1;
  static __device__ __forceinline__ int frag(int d, int c, int half) { return d * S + (((c * 2 + half) ^ ((d >> 4) & M)) << 3); }
  // tokens 4 quad .. 4 quad + 3
  static __device__ __forceinline__ int quad(int d, int quad) {
    const int h = quad & 1, a = (quad >> 1) & 1, c = quad >> 2;
    return d * S + (((c * 2 + h) ^ ((d >> 4) & M)) << 3) + a * 4;
  }
};

// A staging unit is 4 tokens x 8 head elements: unit u of a tile covers tokens 4 (u / (DP/8)) .. + 3.
template <typename T>
struct Unit {
  typename Elem<T>::V8 r[4];
  // Tokens row .. row + 3 of a head at base, head elements d .. d + 7.  valid: bit i = token row + i counts (others become
  // zero); rows: tokens that exist (>= 1); whole: uniform, all of the tile counts and vec holds.  Tokens that do not exist are never
  // read: their place is taken by the last one there is.  With 16-byte loads every lane loads: no branches around loads.
  __device__ __forceinline__ void load(const T* base, long sl, int row, int rows, int d, int D, unsigned valid, bool vec,
                                       bool whole) {
    typedef typename Elem<T>::V8 V8;
    if (whole) {
      const T* p = base + (long)row * sl + d;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const V8*>(p + i * sl);
    } else if (vec) {
      const T* p = base + (d < D ? d : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const V8*>(p + (long)min(row + i, rows - 1) * sl);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d >= D || !((valid >> i) & 1)) r[i] = V8{};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r[i] = load8<T>(base + (long)min(row + i, rows - 1) * sl + d, (valid >> i) & 1 ? D - d : 0, false);
    }
  }
  template <int DP>
  __device__ __forceinline__ void put_r(T* tile, int u) const {
    const int quad = u / (DP / 8), dc = u % (DP / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<typename Elem<T>::V8*>(tile + (quad * 4 + i) * TileR<T, DP>::S + dc * 8) = r[i];
  }
  template <int DP, int ROWS>
  __device__ __forceinline__ void put_x(T* tile, int u) const {
    const int quad = u / (DP / 8), dc = u % (DP / 8);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      typename Elem<T>::V4 t;
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = r[i][j];
      *reinterpret_cast<typename Elem<T>::V4*>(tile + TileX<T, ROWS>::quad(dc * 8 + j, quad)) = t;
    }
  }
};

template <typename T>
__device__ __forceinline__ const typename Elem<T>::V8 frag_at(const T* tile, int at) {
  return *reinterpret_cast<const typename Elem<T>::V8*>(tile + at);
}

// Registers 8c .. 8c + 7 of a 32x32 result.
__device__ __forceinline__ f32v8 part8(const f32x16& s, int c) {
  f32v8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = s[8 * c + i];
  return v;
}

// An fp32 value as the second operand of a product (P and dS): the matrix instructions of the 16-bit types take no wider one, so it is
// the sum of two, and the product takes two instructions.  bf16 rounds both to nearest, fp16 towards zero (one instruction for two
// elements): what is lost is at most 2^-16 or 2^-20 of the value, against the 2^-8 or 2^-11 of one operand, which would add as much to
// the error of a result as its own rounding to the type does (long causal forward, bf16: 1.95e-3 of the result in all, with two
// 1.52e-3).  All of a step's products take the first operand before the second: no two in a row add to the same registers.
template <typename T>
struct Wide {
  typename Elem<T>::V8 high, low;
  __device__ __forceinline__ explicit Wide(const f32v8& x);
  // c[i] += frag(i) x
  template <int N, typename F>
  __device__ __forceinline__ void mma_all(f32x16 (&c)[N], F frag) const {
    typename Elem<T>::V8 a[N];
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = frag(i);
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = Elem<T>::mma32(a[i], high, c[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = Elem<T>::mma32(a[i], low, c[i]);
  }
  __device__ __forceinline__ f32x16 mma(const typename Elem<T>::V8& a, f32x16 c) const {
    return Elem<T>::mma32(a, low, Elem<T>::mma32(a, high, c));
  }
};
template <>
__device__ __forceinline__ Wide<__bf16>::Wide(const f32v8& x) {
  struct {
    bf16v2 pair[4];
  } h, l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32v2 v = {x[2 * i], x[2 * i + 1]};
    h.pair[i] = __builtin_convertvector(v, bf16v2);
    l.pair[i] = __builtin_convertvector((f32v2{v[0] - (float)h.pair[i][0], v[1] - (float)h.pair[i][1]}), bf16v2);
  }
  high = __builtin_bit_cast(bf16v8, h);
  low = __builtin_bit_cast(bf16v8, l);
}
template <>
__device__ __forceinline__ Wide<_Float16>::Wide(const f32v8& x) {
  struct {
    f16v2 pair[4];
  } h, l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h.pair[i] = __builtin_bit_cast(f16v2, __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]));
    l.pair[i] = __builtin_bit_cast(
        f16v2, __builtin_amdgcn_cvt_pkrtz(x[2 * i] - (float)h.pair[i][0], x[2 * i + 1] - (float)h.pair[i][1]));
  }
  high = __builtin_bit_cast(f16v8, h);
  low = __builtin_bit_cast(f16v8, l);
}
template <>
struct Wide<float> {
  f32v8 x;
  __device__ __forceinline__ explicit Wide(const f32v8& v) : x(v) {}
  template <int N, typename F>
  __device__ __forceinline__ void mma_all(f32x16 (&c)[N], F frag) const {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = Elem<float>::mma32(frag(i), x, c[i]);
  }
  __device__ __forceinline__ f32x16 mma(const f32v8& a, f32x16 c) const { return Elem<float>::mma32(a, x, c); }
};

// fp16: P and dS are taken as 16 P and 16 dS.  A row of n keys holds P of about 1 / n, which from n = 2^14 on, and dS sooner,
// would fall among fp16's subnormals.
template <typename T>
constexpr float P_SHIFT = 0.f;
template <>
inline constexpr float P_SHIFT<_Float16> = 4.f;
template <typename T>
constexpr float P_UNSHIFT = 1.f;
template <>
inline constexpr float P_UNSHIFT<_Float16> = 0.0625f;

// |dS| is up to half the largest |dout . v| and so has no bound that fp16 could hold: where 16 dS passes FIT_LIMIT, a power of two
// (`fit`, 1 until then, the same in all lanes of a wave) takes the largest down to 2^14 .. 2^15, and the sums so far with it.  The result
// is divided by it again, in fp32.  The second operand then ends at 2^-38 of the largest.  All but a maximum and a
// comparison is in the branch.
template <typename T>
constexpr bool FIT = false;
template <>
inline constexpr bool FIT<_Float16> = true;
constexpr float FIT_LIMIT = 32768.f;
__device__ __forceinline__ float fit_for(float most) {
  return __builtin_bit_cast(float, (268u - ((__builtin_bit_cast(unsigned, most) >> 23) & 255u)) << 23);      // 2^(14 - exponent)
}
// The largest magnitude; zero if that is infinite: such a row's or column's results are lost, and others' scale must not go by it.
template <typename V>
__device__ __forceinline__ float most_of(V x) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / sizeof(float)); ++i) m = fmaxf(m, fabsf(x[i]));
  return m < INFINITY ? m : 0.f;
}
__device__ __forceinline__ float wave_most(float m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, m)));
}
// The values ds of a step, made to fit; acc holds sums of what came before.  (By value: a template's parameter does not keep f32v8's
// alignment.)
template <typename V, int N>
__device__ __forceinline__ V make_fit(V ds, f32x16 (&acc)[N], float& fit) {
  const float most = most_of(ds);
  if (__any(most * fit > FIT_LIMIT)) {
    const float now = fit_for(wave_most(most));
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][r] *= now / fit;
    fit = now;
  }
  if (fit != 1.f) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / sizeof(float)); ++i) ds[i] *= fit;
  }
  return ds;
}

// One bit per key of the tile at key0: below the sequence's length and not masked.  The same in every wave.
__device__ __forceinline__ unsigned long long key_bits(const AttnArgs& a, int b, int key0, int len) {
  const int key = key0 + (int)(threadIdx.x & 63);
  bool on = key < len;
  if (on && a.key_mask) on = a.key_mask[(long)b * a.mask_stride + key] != 0;
  return __ballot(on);
}

// Whether this lane's key of result register r counts: bit 8 (r / 4) + r % 4 of the 32 keys' word for lanes 0 .. 31, four
// further for the others.  The word is uniform, so this is scalar work and one select a register.
__device__ __forceinline__ bool key_on(unsigned word, int r) {
  const int key = 8 * (r / 4) + r % 4;
  const int low = (int)(word << (31 - key)) >> 31, high = (int)(word << (27 - key)) >> 31;
  return __builtin_amdgcn_inverse_ballot_w64(((unsigned long long)(unsigned)high << 32) | (unsigned)low);
}
__device__ __forceinline__ unsigned word_of(unsigned long long bits, int t) {
  return __builtin_amdgcn_readfirstlane((unsigned)(bits >> (32 * t)));
}

__device__ __forceinline__ int key_limit(const AttnArgs& a, int b) {
  if (!a.key_lengths) return a.Lk;
  const int n = a.key_lengths[b];
  return n < 0 ? 0 : (n < a.Lk ? n : a.Lk);
}

// Query i sees key j iff j <= i + start.  Without causality every key is at or before the start.
__device__ __forceinline__ long causal_start(const AttnArgs& a, int b) {
  if (!a.causal) return (long)a.Lk;
  return a.query_start ? (long)a.query_start[b] : (long)a.Lk - a.Lq;
}

// Keys of a tile in LDS.  fp32: 32, which lets three waves a SIMD run instead of two (L = 52, D = 64, 40960 heads: forward
// 760 -> 690 us, dq 1298 -> 1008 us).
template <typename T>
constexpr int KEY_TILE = sizeof(T) == 4 ? 32 : 64;

// Leaves one range's result of a row for attn_join_kernel: maximum and sum, and the unnormalised output (not written where
// nothing was seen).  Rows are ordered (batch, key head, query, head of the group).
template <typename T, int DP>
__device__ __forceinline__ void put_partial(const AttnArgs& a, long row, int split, float m, float l, const f32x16 (&o)[DP / 32]) {
  const int half = (threadIdx.x & 63) >> 5;
  row = row * a.splits + split;
  if (half == 0) reinterpret_cast<f32v2*>(a.part_ml)[row] = f32v2{m, l};
  if (l == 0.f) return;
  float* p = a.part_o + row * DP;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32v4*>(p + dt * 32 + g * 8 + half * 4) =
          f32v4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
}

// ---- forward ------------------------------------------------------------------------------------------------------
// One workgroup = 32 NW queries of one head, one wave = 32 of them; the keys pass in tiles.  8192 tokens, 16 on 4 heads of 128,
// bf16, causal: 427 .. 455 us, 907 .. 966 TFLOP/s of its three products (P V takes two), where a large product reaches 1119; the matrix
// pipe is busy 48 % of the time, and a wave reads 32 KB of LDS for each 32 x 64 scores (331 us with P in one operand, at the error
// told at Wide).  Two waves a SIMD (603 us at one, then) and loads between the barriers, not a tile ahead in
// registers (which took a fifth more of them for the same time).
// With few workgroups the tiles are cut into `splits` ranges, which attn_join_kernel joins.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? 2 : DP <= 64 ? 3 : 1) void attn_fwd_kernel(AttnArgs a) {
  typedef typename Elem<T>::V8 V8;
  constexpr int KT = KEY_TILE<T>, NT = NW * 64, NC = DP / 16, ND = DP / 32;
  constexpr int UN = KT / 4 * (DP / 8), UPT = (2 * UN + NT - 1) / NT;
  constexpr unsigned long long FULL = ~0ull >> (64 - KT);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const kt = reinterpret_cast<T*>(lds);
  T* const vx = kt + KT * TileR<T, DP>::S;
  const long item = xcd_item(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  const int tiles = (a.Lq + 32 * NW - 1) / (32 * NW);
  const int split = (int)(item % a.splits);
  const int tile = tiles - 1 - (int)(item / a.splits % tiles);       // causal: the longest first
  const int hq = (int)((item / a.splits / tiles) % a.Hq);
  const int b = (int)(item / a.splits / tiles / a.Hq);
  const int hk = hq / a.G;
  const int i = tile * 32 * NW + wave * 32 + col;         // this lane's query
  const bool vec = a.vec != 0;

  V8 qf[NC];
  {
    const T* p = (const T*)a.q + b * a.vq.sb + hq * a.vq.sh + (long)i * a.vq.sl;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = c * 16 + half * 8;
      qf[c] = load8<T>(p + d, i < a.Lq ? a.D - d : 0, vec);
    }
  }
  const int len = key_limit(a, b);
  const long start = causal_start(a, b);
  const int last_row = min(tile * 32 * NW + 32 * NW, a.Lq) - 1;
  const long seen = last_row + start + 1;                 // keys the last query of the workgroup sees
  const int end = (int)max(0L, min((long)len, seen));
  const long sees = (long)i + start;                      // last key this lane's query sees
  const long all_tiles = (end + KT - 1) / KT;             // this workgroup's share of the key tiles
  const int from = (int)(all_tiles * split / a.splits) * KT;
  const int stop = (int)min((long)end, all_tiles * (split + 1) / a.splits * KT);

  const T* kb = (const T*)a.k + b * a.vk.sb + hk * a.vk.sh;
  const T* vb = (const T*)a.v + b * a.vv.sb + hk * a.vv.sh;
  const bool whole = vec && a.D == DP && 2 * UN % NT == 0;
  auto load_unit = [&](Unit<T>& to, int n, int key0, unsigned long long bits) {
    const int u = tid + n * NT;
    const bool is_v = u >= UN;
    const int w = is_v ? u - UN : u;
    const int quad = w / (DP / 8), d = w % (DP / 8) * 8;
    const unsigned ok = u < 2 * UN ? (unsigned)(bits >> (quad * 4)) & 15u : 0u;
    const long sl = is_v ? a.vv.sl : a.vk.sl;
    to.load(is_v ? vb : kb, sl, key0 + quad * 4, a.Lk, d, a.D, ok, vec, whole && bits == FULL);
  };
  auto put_unit = [&](const Unit<T>& from, int n) {
    const int u = tid + n * NT;
    if (u < UN) from.template put_r<DP>(kt, u);
    else if (u < 2 * UN) from.template put_x<DP, KT>(vx, u - UN);
  };
  auto stage = [&](int key0, unsigned long long bits) {
#pragma unroll 2
    for (int n = 0; n < UPT; ++n) {
      Unit<T> t;
      load_unit(t, n, key0, bits);
      put_unit(t, n);
    }
  };

  f32x16 o[ND] = {};
  float m = -INFINITY, l = 0.f;                            // l: the sum over this lane half's keys
  unsigned long long bits = key_bits(a, b, from, end) & FULL;
  for (int key0 = from; key0 < stop; key0 += KT) {
    const unsigned long long here = bits;
    if (key0 + KT < stop) bits = key_bits(a, b, key0 + KT, end) & FULL;
    if (here == 0ull) continue;                            // the same in every wave
    __syncthreads();
    stage(key0, here);
    __syncthreads();
    f32x16 s[KT / 32] = {};
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
      for (int c = 0; c < NC; ++c) s[t] = Elem<T>::mma32(frag_at<T>(kt, TileR<T, DP>::frag(t * 32 + col, c, half)), qf[c], s[t]);
    if (here != FULL) {
#pragma unroll
      for (int t = 0; t < KT / 32; ++t) {
        const unsigned word = word_of(here, t);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = key_on(word, r) ? s[t][r] : -INFINITY;
      }
    }
    if (a.causal && key0 + KT - 1 > sees - col) {          // sees - col: what the wave's first query sees
      const int room = (int)max(-64L, min(64L, sees - key0)) - 4 * half;
#pragma unroll
      for (int t = 0; t < KT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * 32 + 8 * (r / 4) + r % 4 > room) s[t][r] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mn = fmaxf(m, top * a.scale_log2);
    const float use = mn == -INFINITY ? 0.f : mn;          // nothing visible yet: every exponential below is 0
    const float alpha = __builtin_amdgcn_exp2f(m - use);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale_log2, -use));
        sum += s[t][r];
      }
    l = fmaf(l, alpha, sum);
    if (__any(alpha != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Wide<T> p(part8(s[t], c));
        p.mma_all(o, [&](int dt) { return frag_at<T>(vx, TileX<T, KT>::frag(dt * 32 + col, t * 2 + c, half)); });
      }
  }
  l += __shfl_xor(l, 32, 64);
  if (i >= a.Lq) return;
  if (a.splits > 1) {
    put_partial<T, DP>(a, (((long)b * a.Hk + hk) * a.Lq + i) * a.G + hq % a.G, split, m, l, o);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* op = (T*)a.out + b * a.vo.sb + hq * a.vo.sh + (long)i * a.vo.sl;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = dt * 32 + g * 8 + half * 4;
      const f32v4 w = {o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv, o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv};
      if (d < a.D) store4<T>(op + d, w, a.D - d, vec);
    }
  if (half == 0) a.lse[((long)b * a.Hq + hq) * a.Lq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// ---- forward of few queries over many keys ---------------------------------------------------------------------------
// The queries of all heads that share a key head are the columns of one tile: column n = i G + g.  A workgroup is one wave
// with 32 columns and one of `splits` ranges of the sequence's keys, so a cache is read once and by the whole chip however
// few its queries are; attn_join_kernel joins the ranges.  HBM-bound: per 32 keys a wave has 32 D elements of k (straight to the
// operand's registers) and of v (transposed through LDS of its own, no barriers) in flight while it works on the last 32.
// 8 sequences of up to 8192 keys, 32 on 8 heads of 128, bf16: 38 us, 5.3 TB/s (532 us in tiles of 32 queries a head).
template <typename T, int DP>
__global__ __launch_bounds__(64) void attn_few_kernel(AttnArgs a) {
  typedef typename Elem<T>::V8 V8;
  constexpr int KT = 32, NC = DP / 16, ND = DP / 32, UPT = KT / 4 * (DP / 8) / 64 > 0 ? KT / 4 * (DP / 8) / 64 : 1;
  __shared__ __attribute__((aligned(16))) T vx[DP * TileX<T, KT>::S];
  const long item = xcd_item(a.items);
  if (item >= a.items) return;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int N = a.Lq * a.G, tiles = (N + 31) / 32;
  const int split = (int)(item % a.splits);
  const int tile = (int)((item / a.splits) % tiles);
  const long pair = item / a.splits / tiles;
  const int hk = (int)(pair % a.Hk), b = (int)(pair / a.Hk);
  const int n = tile * 32 + col;
  const int i = n / a.G, hq = hk * a.G + n % a.G;
  const bool vec = a.vec != 0;
  V8 qf[NC];
  {
    const T* p = (const T*)a.q + b * a.vq.sb + hq * a.vq.sh + (long)i * a.vq.sl;
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = load8<T>(p + c * 16 + half * 8, n < N ? a.D - c * 16 - half * 8 : 0, vec);
  }
  const long start = causal_start(a, b);
  const long sees = (long)i + start;
  const int last_i = min(tile * 32 + 31, N - 1) / a.G;
  const int len = (int)max(0L, min((long)key_limit(a, b), last_i + start + 1));
  const int each = ((len + a.splits - 1) / a.splits + KT - 1) / KT * KT;
  const int from = (int)min((long)len, (long)split * each), end = min(len, from + each);
  const T* kb = (const T*)a.k + b * a.vk.sb + hk * a.vk.sh;
  const T* vb = (const T*)a.v + b * a.vv.sb + hk * a.vv.sh;
  V8 kf[NC];
  Unit<T> un[UPT];
  const bool whole = vec && a.D == DP && KT / 4 * (DP / 8) % 64 == 0;
  auto fetch = [&](int key0, unsigned bits) {
    const int key = key0 + col;
    const T* p = kb + (long)key * a.vk.sl;
    const bool on = (bits >> col) & 1;
#pragma unroll
    for (int c = 0; c < NC; ++c) kf[c] = load8<T>(p + c * 16 + half * 8, on ? a.D - c * 16 - half * 8 : 0, vec);
#pragma unroll
    for (int m = 0; m < UPT; ++m) {
      const int u = lane + m * 64, quad = u / (DP / 8), d = u % (DP / 8) * 8;
      const unsigned ok = quad < KT / 4 ? (bits >> (quad * 4)) & 15u : 0u;
      un[m].load(vb, a.vv.sl, key0 + quad * 4, a.Lk, d, a.D, ok, vec, whole && bits == ~0u);
    }
  };
  f32x16 o[ND] = {};
  float m = -INFINITY, l = 0.f;
  unsigned bits = (unsigned)key_bits(a, b, from, end);
  if (from < end) fetch(from, bits);                        // an empty range may have no memory behind it
  for (int key0 = from; key0 < end; key0 += KT) {
    const unsigned here = bits;
    f32x16 s = {};
#pragma unroll
    for (int c = 0; c < NC; ++c) s = Elem<T>::mma32(kf[c], qf[c], s);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the last tile's reads of vx come first
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < UPT; ++e)
      if (lane + e * 64 < KT / 4 * (DP / 8)) un[e].template put_x<DP, KT>(vx, lane + e * 64);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (key0 + KT < end) {
      bits = (unsigned)key_bits(a, b, key0 + KT, end);
      fetch(key0 + KT, bits);
    }
    if (here == 0u) continue;
    if (here != ~0u) {
      const unsigned word = word_of(here, 0);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = key_on(word, r) ? s[r] : -INFINITY;
    }
    if (a.causal && key0 + KT - 1 > start) {                // start: what query 0 sees
      const int room = (int)max(-64L, min(64L, sees - key0)) - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + r % 4 > room) s[r] = -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mn = fmaxf(m, top * a.scale_log2);
    const float use = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - use);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, -use));
      sum += s[r];
    }
    l = fmaf(l, alpha, sum);
    if (__any(alpha != 1.f)) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Wide<T> p(part8(s, c));
      p.mma_all(o, [&](int dt) { return frag_at<T>(vx, TileX<T, KT>::frag(dt * 32 + col, c, half)); });
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (n >= N) return;
  if (a.splits == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* op = (T*)a.out + b * a.vo.sb + hq * a.vo.sh + (long)i * a.vo.sl;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = dt * 32 + g * 8 + half * 4;
        const f32v4 w = {o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv, o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv};
        if (d < a.D) store4<T>(op + d, w, a.D - d, vec);
      }
    if (half == 0) a.lse[((long)b * a.Hq + hq) * a.Lq + i] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
    return;
  }
  put_partial<T, DP>(a, pair * N + n, split, m, l, o);
}

// One workgroup joins the `splits` partial results of one query: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.
// Lane groups of DP take every (256 / DP)-th range.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  constexpr int GR = 256 / DP;
  __shared__ float weight[ATTN_MAX_SPLITS];
  __shared__ float sums[256];
  const long row = blockIdx.x;                             // (b Hk + hk) N + n
  const int N = a.Lq * a.G, n = (int)(row % N);
  const long pair = row / N;
  const int hk = (int)(pair % a.Hk), b = (int)(pair / a.Hk), i = n / a.G, hq = hk * a.G + n % a.G;
  const f32v2* ml = reinterpret_cast<const f32v2*>(a.part_ml) + row * a.splits;
  const int tid = threadIdx.x, lane = tid & 63;
  // every wave finds the maximum and the sum for itself
  float top = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, ml[s][0]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  const float use = top == -INFINITY ? 0.f : top;
  float l = 0.f;
  for (int s = lane; s < a.splits; s += 64) {
    const f32v2 v = ml[s];
    const float w = v[1] == 0.f ? 0.f : __builtin_amdgcn_exp2f(v[0] - use);
    l += v[1] == 0.f ? 0.f : w * v[1];
    if (tid < 64) weight[s] = v[1] == 0.f ? -1.f : w;      // -1: nothing was written there
  }
  l = wave_sum(l);
  __syncthreads();
  const int d = tid % DP, g = tid / DP;
  float t = 0.f;
#pragma unroll 8
  for (int s = g; s < a.splits; s += GR) {                  // loads without a branch, so that eight are under way at a time
    const float w = weight[s], x = a.part_o[(row * a.splits + s) * DP + d];
    t += w >= 0.f || w != w ? w * x : 0.f;
  }
  sums[tid] = t;
  __syncthreads();
  if (g > 0 || d >= a.D) return;
#pragma unroll
  for (int k = 1; k < GR; ++k) t += sums[k * DP + d];
  ((T*)a.out)[b * a.vo.sb + hq * a.vo.sh + (long)i * a.vo.sl + d] = (T)(l == 0.f ? 0.f : t / l);
  if (d == 0) a.lse[((long)b * a.Hq + hq) * a.Lq + i] = l == 0.f ? -INFINITY : (top + log2f(l)) * LN2;
}

// The same for up to ATTN_ROW_SPLITS ranges of many rows: a lane has four head elements of one row and every range of it
// (16384 rows of 64 in 4 ranges: a quarter of the time of a workgroup a row).
constexpr int ATTN_ROW_SPLITS = 16;
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_rows_kernel(AttnArgs a) {
  constexpr int PER = DP / 4;
  const long rows = (long)a.B * a.Hq * a.Lq;
  const long at = (long)blockIdx.x * 256 + threadIdx.x, row = at / PER;
  const int d = (int)(at % PER) * 4;
  if (row >= rows || d >= a.D) return;
  const f32v2* ml = reinterpret_cast<const f32v2*>(a.part_ml) + row * a.splits;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[s][0]);
  const float use = top == -INFINITY ? 0.f : top;
  float l = 0.f;
  f32v4 t = {};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const f32v2 v = ml[s];
    const f32v4 x = *reinterpret_cast<const f32v4*>(a.part_o + (row * a.splits + s) * DP + d);
    const bool on = v[1] != 0.f;                           // else: nothing was written there
    const float w = __builtin_amdgcn_exp2f(v[0] - use);
    l += on ? w * v[1] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] += on ? w * x[e] : 0.f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] *= inv;
  const long pair = row / ((long)a.Lq * a.G);
  const int n = (int)(row % ((long)a.Lq * a.G)), i = n / a.G;
  const int hk = (int)(pair % a.Hk), b = (int)(pair / a.Hk), hq = hk * a.G + n % a.G;
  store4<T>((T*)a.out + b * a.vo.sb + hq * a.vo.sh + (long)i * a.vo.sl + d, t, a.D - d, a.vec);
  if (d == 0) a.lse[((long)b * a.Hq + hq) * a.Lq + i] = l == 0.f ? -INFINITY : (top + log2f(l)) * LN2;
}

// ---- backward: dq (and delta) ---------------------------------------------------------------------------------------
// One workgroup = 32 NW queries of one head, keys in tiles of KT: S^T and dP^T = V dO^T share the layout of the forward,
// dq^T += K^T dS^T.  delta = dout . out is formed here first and left for the dk / dv kernel.  With few workgroups the key tiles
// are cut into `splits_q` shares, whose fp32 results attn_sum_q_kernel adds in order.  2 x 4001 tokens, 16 on 4 heads of 128,
// bf16, causal: 394 us, 665 TFLOP/s of its four products (dS K takes two); 350 us with dS in one operand.  The next tile in registers
// spilled, and took a quarter longer.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? 2 : DP <= 32 ? 3 : DP <= 64 ? 2 : 1) void attn_dq_kernel(AttnArgs a) {
  typedef typename Elem<T>::V8 V8;
  constexpr int KT = KEY_TILE<T>, NT = NW * 64, NC = DP / 16, ND = DP / 32;
  constexpr int UN = KT / 4 * (DP / 8), UPT = (2 * UN + NT - 1) / NT;
  constexpr unsigned long long FULL = ~0ull >> (64 - KT);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const kt = reinterpret_cast<T*>(lds);
  T* const vt = kt + KT * TileR<T, DP>::S;
  T* const kx = vt + KT * TileR<T, DP>::S;
  const long item = xcd_item(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  const int tiles = (a.Lq + 32 * NW - 1) / (32 * NW);
  const int split = (int)(item % a.splits_q);
  const int tile = tiles - 1 - (int)(item / a.splits_q % tiles);
  const int hq = (int)((item / a.splits_q / tiles) % a.Hq);
  const int b = (int)(item / a.splits_q / tiles / a.Hq);
  const int hk = hq / a.G;
  const int i = tile * 32 * NW + wave * 32 + col;
  const bool vec = a.vec != 0;
  const long row = ((long)b * a.Hq + hq) * a.Lq + i;

  const float lse = i < a.Lq ? a.lse_in[row] : -INFINITY;
  const bool live = lse != -INFINITY;                     // a row that sees nothing has no gradient, whatever it holds
  const float lse2 = live ? fmaf(lse, LOG2E, -P_SHIFT<T>) : INFINITY;
  V8 qf[NC], gf[NC];
  float delta = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int d = c * 16 + half * 8, n = live ? a.D - d : 0;
    qf[c] = load8<T>((const T*)a.q + b * a.vq.sb + hq * a.vq.sh + (long)i * a.vq.sl + d, n, vec);
    gf[c] = load8<T>((const T*)a.dout + b * a.vdo.sb + hq * a.vdo.sh + (long)i * a.vdo.sl + d, n, vec);
    const V8 of = load8<T>((const T*)a.out_in + b * a.vo.sb + hq * a.vo.sh + (long)i * a.vo.sl + d, n, vec);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[c][j], (float)of[j], delta);
  }
  delta += __shfl_xor(delta, 32, 64);
  if (half == 0 && i < a.Lq && split == 0) a.delta[row] = delta;

  const int len = key_limit(a, b);
  const long start = causal_start(a, b);
  const int last_row = min(tile * 32 * NW + 32 * NW, a.Lq) - 1;
  const int end = (int)max(0L, min((long)len, last_row + start + 1));
  const long sees = (long)i + start;
  const long all_tiles = (end + KT - 1) / KT;             // this workgroup's share of the key tiles
  const int from = (int)(all_tiles * split / a.splits_q) * KT;
  const int stop = (int)min((long)end, all_tiles * (split + 1) / a.splits_q * KT);
  const T* kb = (const T*)a.k + b * a.vk.sb + hk * a.vk.sh;
  const T* vb = (const T*)a.v + b * a.vv.sb + hk * a.vv.sh;
  const bool whole = vec && a.D == DP && 2 * UN % NT == 0;
  auto load_unit = [&](Unit<T>& to, int n, int key0, unsigned long long bits) {
    const int u = tid + n * NT;
    const bool is_v = u >= UN;
    const int w = is_v ? u - UN : u;
    const int quad = w / (DP / 8), d = w % (DP / 8) * 8;
    const unsigned ok = u < 2 * UN ? (unsigned)(bits >> (quad * 4)) & 15u : 0u;
    const long sl = is_v ? a.vv.sl : a.vk.sl;
    to.load(is_v ? vb : kb, sl, key0 + quad * 4, a.Lk, d, a.D, ok, vec, whole && bits == FULL);
  };
  auto put_unit = [&](const Unit<T>& from, int n) {
    const int u = tid + n * NT;
    if (u < UN) {
      from.template put_r<DP>(kt, u);
      from.template put_x<DP, KT>(kx, u);
    } else if (u < 2 * UN) {
      from.template put_r<DP>(vt, u - UN);
    }
  };
  auto stage = [&](int key0, unsigned long long bits) {
#pragma unroll 2
    for (int n = 0; n < UPT; ++n) {
      Unit<T> t;
      load_unit(t, n, key0, bits);
      put_unit(t, n);
    }
  };
  f32x16 acc[ND] = {};
  float fit = 1.f;
  unsigned long long bits = key_bits(a, b, from, end) & FULL;
  for (int key0 = from; key0 < stop; key0 += KT) {
    const unsigned long long here = bits;
    if (key0 + KT < stop) bits = key_bits(a, b, key0 + KT, end) & FULL;
    if (here == 0ull) continue;                            // the same in every wave
    __syncthreads();
    stage(key0, here);
    __syncthreads();
    const bool beyond = a.causal && key0 + KT - 1 > sees - col;
#pragma unroll
    for (int t = 0; t < KT / 32; ++t) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int c = 0; c < NC; ++c) s = Elem<T>::mma32(frag_at<T>(kt, TileR<T, DP>::frag(t * 32 + col, c, half)), qf[c], s);
#pragma unroll
      for (int c = 0; c < NC; ++c) dp = Elem<T>::mma32(frag_at<T>(vt, TileR<T, DP>::frag(t * 32 + col, c, half)), gf[c], dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, -lse2)) * (dp[r] - delta);
      if (here != FULL) {
        const unsigned word = word_of(here, t);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = key_on(word, r) ? s[r] : 0.f;
      }
      if (beyond) {
        const int room = (int)max(-64L, min(64L, sees - key0)) - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * 32 + 8 * (r / 4) + r % 4 > room) s[r] = 0.f;
      }
      if (FIT<T>) s = make_fit(s, acc, fit);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Wide<T> ds(part8(s, c));
        ds.mma_all(acc, [&](int dt) { return frag_at<T>(kx, TileX<T, KT>::frag(dt * 32 + col, t * 2 + c, half)); });
      }
    }
  }
  if (i >= a.Lq) return;
  const float unfit = FIT<T> ? 1.f / fit : 1.f;
  if (a.splits_q > 1) {
    float* p = a.part_q + (split * ((long)a.B * a.Hq * a.Lq) + row) * DP;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32v4*>(p + dt * 32 + g * 8 + half * 4) =
            f32v4{acc[dt][4 * g] * unfit, acc[dt][4 * g + 1] * unfit, acc[dt][4 * g + 2] * unfit, acc[dt][4 * g + 3] * unfit};
    return;
  }
  const float back = a.scale * P_UNSHIFT<T> * unfit;
  T* p = (T*)a.dq + b * a.vdq.sb + hq * a.vdq.sh + (long)i * a.vdq.sl;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = dt * 32 + g * 8 + half * 4;
      const f32v4 w = {acc[dt][4 * g] * back, acc[dt][4 * g + 1] * back, acc[dt][4 * g + 2] * back,
                       acc[dt][4 * g + 3] * back};
      if (d < a.D) store4<T>(p + d, w, a.D - d, vec);
    }
}

// dq from the fp32 shares of the dq kernel; a lane has four head elements of one query.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_sum_q_kernel(AttnArgs a) {
  constexpr int PER = DP / 4;
  const long rows = (long)a.B * a.Hq * a.Lq;
  const long at = (long)blockIdx.x * 256 + threadIdx.x, row = at / PER;
  const int d = (int)(at % PER) * 4;
  if (row >= rows || d >= a.D) return;
  f32v4 t = {};
#pragma unroll 4
  for (int s = 0; s < a.splits_q; ++s) {
    const f32v4 x = *reinterpret_cast<const f32v4*>(a.part_q + (s * rows + row) * DP + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] += x[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) t[e] *= a.scale * P_UNSHIFT<T>;
  const int i = (int)(row % a.Lq), hq = (int)(row / a.Lq % a.Hq), b = (int)(row / a.Lq / a.Hq);
  store4<T>((T*)a.dq + b * a.vdq.sb + hq * a.vdq.sh + (long)i * a.vdq.sl + d, t, a.D - d, a.vec);
}

// ---- backward: dk, dv ------------------------------------------------------------------------------------------------
// With few workgroups the list of (head, query tile) is cut into `splits` shares, whose fp32 results attn_sum_kernel adds in order.
// V_LDS: 16-bit heads of 128 leave no room for the values beside both accumulators at two waves a SIMD.
template <typename T, int DP>
constexpr bool DKV_V_LDS = sizeof(T) == 2 && DP == 128;

// One workgroup = 32 NW keys of one key head, one wave = 32 of them; the queries of every head that shares it pass in
// tiles of 32.  S and dP = dO V^T here have queries as rows: dv^T += dO^T P, dk^T += Q^T dS.  The sums over heads
// and queries stay in one accumulator in a fixed order: no atomics, the same bits every time.  2 x 4001 tokens, 16 on 4 heads
// of 128, bf16, causal: 563 us, 700 TFLOP/s of its six products (dO P and Q dS take two); 461 us with P and dS in one operand, 1440 us
// without shares and at one wave a SIMD.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 || DP <= 64 ? 2 : 1) void attn_dkv_kernel(AttnArgs a) {
  typedef typename Elem<T>::V8 V8;
  constexpr bool V_LDS = DKV_V_LDS<T, DP>;
  constexpr int QT = 32, NT = NW * 64, NC = DP / 16, ND = DP / 32;
  constexpr int UN = QT / 4 * (DP / 8), UPT = (2 * UN + NT - 1) / NT;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const qt = reinterpret_cast<T*>(lds);
  T* const gt = qt + QT * TileR<T, DP>::S;
  T* const qx = gt + QT * TileR<T, DP>::S;
  T* const gx = qx + DP * TileX<T, QT>::S;
  float* const lse2s = reinterpret_cast<float*>(gx + DP * TileX<T, QT>::S);
  float* const deltas = lse2s + QT;
  T* const vt = reinterpret_cast<T*>(deltas + QT);        // V_LDS: the workgroup's values
  const long item = xcd_item(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  const int tiles = (a.Lk + 32 * NW - 1) / (32 * NW);
  const int split = (int)(item % a.splits);
  const int tile = (int)(item / a.splits % tiles);        // causal: the first keys are seen by the most queries
  const int hk = (int)((item / a.splits / tiles) % a.Hk);
  const int b = (int)(item / a.splits / tiles / a.Hk);
  const int key0 = tile * 32 * NW;
  const int j = key0 + wave * 32 + col;                   // this lane's key
  const bool vec = a.vec != 0;
  const long start = causal_start(a, b);
  const int len = (int)max(0L, min((long)key_limit(a, b), a.Lq + start));       // keys that no query sees count as absent
  const bool on = j < len && (!a.key_mask || a.key_mask[(long)b * a.mask_stride + j] != 0);
  V8 kf[NC], vf[V_LDS ? 1 : NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int d = c * 16 + half * 8, n = on ? a.D - d : 0;
    kf[c] = load8<T>((const T*)a.k + b * a.vk.sb + hk * a.vk.sh + (long)j * a.vk.sl + d, n, vec);
    const V8 t = load8<T>((const T*)a.v + b * a.vv.sb + hk * a.vv.sh + (long)j * a.vv.sl + d, n, vec);
    // a lane reads back only what it writes here: no barrier
    if (V_LDS) *reinterpret_cast<V8*>(vt + TileR<T, DP>::frag(wave * 32 + col, c, half)) = t;
    else vf[V_LDS ? 0 : c] = t;
  }
  const bool all_on = __all(on);
  const int first = (int)max(0L, min((long)a.Lq, (long)key0 - start)) / QT * QT;      // queries before see none of these keys
  const int per_head = first < a.Lq && key0 < len ? (a.Lq - first + QT - 1) / QT : 0;
  // this workgroup's share of the (head, query tile) list
  const long list = (long)per_head * a.G;
  const int begin = (int)(list * split / a.splits), total = (int)(list * (split + 1) / a.splits) - begin;
  f32x16 dk[ND] = {}, dv[ND] = {};
  float fit = 1.f;
  const bool whole = vec && a.D == DP && 2 * UN % NT == 0;
  auto load_unit = [&](Unit<T>& to, float (&seen)[4], int n, int hq, int q0) {
    const int u = tid + n * NT;
    const bool is_g = u >= UN;
    const int w = is_g ? u - UN : u;
    const int quad = w / (DP / 8), d = w % (DP / 8) * 8;
    const int left = u < 2 * UN ? a.Lq - q0 - quad * 4 : 0;
    const unsigned ok = left >= 4 ? 15u : left > 0 ? (1u << left) - 1 : 0u;
    const float* lse = a.lse_in + ((long)b * a.Hq + hq) * a.Lq + q0 + quad * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) seen[e] = e < left ? lse[e] : -INFINITY;
    const long sb = is_g ? a.vdo.sb : a.vq.sb, sh = is_g ? a.vdo.sh : a.vq.sh, sl = is_g ? a.vdo.sl : a.vq.sl;
    to.load((const T*)(is_g ? a.dout : a.q) + b * sb + hq * sh, sl, q0 + quad * 4, a.Lq, d, a.D, ok, vec,
            whole && q0 + QT <= a.Lq);
  };
  auto put_unit = [&](Unit<T>& from, const float (&seen)[4], int n) {
    const int u = tid + n * NT;
#pragma unroll
    for (int e = 0; e < 4; ++e)                           // rows that see nothing count as absent, whatever they hold
      if (seen[e] == -INFINITY) from.r[e] = V8{};
    if (u < UN) {
      from.template put_r<DP>(qt, u);
      from.template put_x<DP, QT>(qx, u);
    } else if (u < 2 * UN) {
      from.template put_r<DP>(gt, u - UN);
      from.template put_x<DP, QT>(gx, u - UN);
    }
  };
  auto stage = [&](int hq, int q0) {
#pragma unroll 2
    for (int n = 0; n < UPT; ++n) {
      Unit<T> t;
      float s[4];
      load_unit(t, s, n, hq, q0);
      put_unit(t, s, n);
    }
    if (tid < QT) {
      const long at = ((long)b * a.Hq + hq) * a.Lq + q0 + tid;
      const float x = q0 + tid < a.Lq ? a.lse_in[at] : -INFINITY;
      const float y = q0 + tid < a.Lq ? a.delta[at] : 0.f;
      lse2s[tid] = x == -INFINITY ? INFINITY : fmaf(x, LOG2E, -P_SHIFT<T>);
      deltas[tid] = x == -INFINITY ? 0.f : y;
    }
  };
  int hq = hk * a.G, q0 = first;
  if (total > 0) {
    hq += begin / per_head;
    q0 += begin % per_head * QT;
  }
  for (int n_tile = 0; n_tile < total; ++n_tile, q0 += QT) {
    if (q0 >= a.Lq) {
      q0 = first;
      ++hq;
    }
    __syncthreads();
    stage(hq, q0);
    __syncthreads();
    if ((long)key0 + wave * 32 > q0 + QT - 1 + start) continue;       // none of the wave's keys is seen
    const bool partial = (long)key0 + wave * 32 + 31 > q0 + start || !all_on;
    // rows of the tile before this one do not see the lane's key
    const int sees_from = on ? (int)max(-64L, min(64L, j - start - q0)) - 4 * half : 64;
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int c = 0; c < NC; ++c) s = Elem<T>::mma32(frag_at<T>(qt, TileR<T, DP>::frag(col, c, half)), kf[c], s);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const V8 v = V_LDS ? frag_at<T>(vt, TileR<T, DP>::frag(wave * 32 + col, c, half)) : vf[V_LDS ? 0 : c];
      dp = Elem<T>::mma32(frag_at<T>(gt, TileR<T, DP>::frag(col, c, half)), v, dp);
    }
    // 16 queries at a time: P and dS of the others take no operands' registers yet
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      f32v8 p8, ds8;
#pragma unroll
      for (int g = 2 * c; g < 2 * c + 2; ++g) {
        const f32v4 ls = *reinterpret_cast<const f32v4*>(lse2s + 8 * g + 4 * half);
        const f32v4 de = *reinterpret_cast<const f32v4*>(deltas + 8 * g + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, -ls[e]));
          float ds = p * (dp[r] - de[e]);
          if (partial && 8 * g + e < sees_from) p = ds = 0.f;
          p8[r - 8 * c] = p;
          ds8[r - 8 * c] = ds;
        }
      }
      const Wide<T> p(p8);
      p.mma_all(dv, [&](int dt) { return frag_at<T>(gx, TileX<T, QT>::frag(dt * 32 + col, c, half)); });
      if (FIT<T>) ds8 = make_fit(ds8, dk, fit);
      const Wide<T> ds(ds8);
      ds.mma_all(dk, [&](int dt) { return frag_at<T>(qx, TileX<T, QT>::frag(dt * 32 + col, c, half)); });
    }
  }
  if (j >= a.Lk) return;
  const float unfit = FIT<T> ? 1.f / fit : 1.f;
  if (a.splits > 1) {
    const long rows = (long)a.B * a.Hk * a.Lk, row = ((long)b * a.Hk + hk) * a.Lk + j;
    float* pk = a.part_o + (2 * split * rows + row) * DP;
    float* pv = pk + rows * DP;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = dt * 32 + g * 8 + half * 4;
        *reinterpret_cast<f32v4*>(pk + d) =
            f32v4{dk[dt][4 * g] * unfit, dk[dt][4 * g + 1] * unfit, dk[dt][4 * g + 2] * unfit, dk[dt][4 * g + 3] * unfit};
        *reinterpret_cast<f32v4*>(pv + d) = f32v4{dv[dt][4 * g], dv[dt][4 * g + 1], dv[dt][4 * g + 2], dv[dt][4 * g + 3]};
      }
    return;
  }
  const float back = a.scale * P_UNSHIFT<T> * unfit;
  T* pk = (T*)a.dk + b * a.vdk.sb + hk * a.vdk.sh + (long)j * a.vdk.sl;
  T* pv = (T*)a.dv + b * a.vdv.sb + hk * a.vdv.sh + (long)j * a.vdv.sl;
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = dt * 32 + g * 8 + half * 4;
      if (d >= a.D) continue;
      const f32v4 w = {dk[dt][4 * g] * back, dk[dt][4 * g + 1] * back, dk[dt][4 * g + 2] * back,
                       dk[dt][4 * g + 3] * back};
      const f32v4 x = {dv[dt][4 * g] * P_UNSHIFT<T>, dv[dt][4 * g + 1] * P_UNSHIFT<T>, dv[dt][4 * g + 2] * P_UNSHIFT<T>,
                       dv[dt][4 * g + 3] * P_UNSHIFT<T>};
      store4<T>(pk + d, w, a.D - d, vec);
      store4<T>(pv + d, x, a.D - d, vec);
    }
}

// ---- backward of short sequences -------------------------------------------------------------------------------------
// At most 32 QB queries and 32 KB keys: one workgroup does a whole key head, so that every tensor crosses HBM once and S, dP
// are formed once (5 products instead of 7).  Wave (qi, ki) forms the 32x32 block of S^T and dP^T of its queries and keys;
// P, then dS, pass through LDS, in fp32, to the waves that own the 32x32 tiles of dv^T, dk^T and dq^T.  All tiles are token-major
// (TileN): an operand that runs along the tokens is read element by element, lanes side by side.  dk and dv stay in registers
// over the query heads of the group.  fp32, L = 52, D = 64: loads and stores alone take 1024 us of the 1680, the matrix
// instructions 745; the two workgroups that a CU's LDS holds do not overlap them.
template <typename T, int W>
struct TileN {
  static constexpr int S = W + 8;      // rows 4 apart start half the banks apart, rows 1 apart 16 or 32 bytes
};
// eight fp32 elements along a row, in slot order (contraction along the row)
__device__ __forceinline__ f32v8 frag_slots(const float* p, int half) {
  const f32v4 u = *reinterpret_cast<const f32v4*>(p + 4 * half), v = *reinterpret_cast<const f32v4*>(p + 8 + 4 * half);
  return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
}
// eight rows in slot order, one column (contraction along the tokens); p: row 0 of the group of 16, this lane's column
template <typename T>
__device__ __forceinline__ typename Elem<T>::V8 frag_rows(const T* p, int stride, int half) {
  typename Elem<T>::V8 v;
#pragma unroll
  for (int s = 0; s < 8; ++s) v[s] = p[(8 * (s / 4) + 4 * half + s % 4) * stride];
  return v;
}

// Waves a SIMD that the registers are cut to: what measured best (10240 sequences of 52 steps, 4 heads of 64: bf16 774 us, fp32 1680;
// of 24 steps, bf16: 325 us at two waves, 391 at one).  Where more waves would spill they are slower, by half and more.
template <typename T, int DP, int QB, int KB>
constexpr int SHORT_WAVES = sizeof(T) == 2 ? (DP == 32 ? 3 : DP == 64 ? 2 : 1) : (DP == 32 || (DP == 64 && QB * KB == 4) ? 2 : 1);

// MANY: where dS has to be made fit, the sums of other heads may have to as well.  (It takes registers: fp16, 4096 sequences of 30 on
// 4 heads of 128: 332 us without, 445 with.)
template <typename T, int DP, int QB, int KB, bool MANY>
__global__ __launch_bounds__(QB * KB * 64, (SHORT_WAVES<T, DP, QB, KB>)) void attn_short_backward_kernel(AttnArgs a) {
  typedef typename Elem<T>::V8 V8;
  constexpr int NW = QB * KB, NT = NW * 64, NC = DP / 16, ND = DP / 32, S = TileN<T, DP>::S, XS = TileN<float, 32 * KB>::S;
  constexpr int UQ = 8 * QB * (DP / 8), UK = 8 * KB * (DP / 8);          // staging units of a query / key tile
  constexpr int KTILES = (KB * ND + NW - 1) / NW, QTILES = (QB * ND + NW - 1) / NW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  T* const qt = reinterpret_cast<T*>(lds);
  T* const gt = qt + 32 * QB * S;
  T* const kt = gt + 32 * QB * S;
  float* const xt = reinterpret_cast<float*>(kt + 32 * KB * S);          // P, then dS: (query, key)
  float* const most_s = xt + 32 * QB * XS;                               // FIT: of each wave, what passes the limit
  const long item = xcd_item(a.items);
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
  const int hk = (int)(item % a.Hk), b = (int)(item / a.Hk);
  const int qi = wave % QB, ki = wave / QB;
  const bool vec = a.vec != 0, whole_d = vec && a.D == DP;
  const long start = causal_start(a, b);
  const int len = (int)max(0L, min((long)key_limit(a, b), a.Lq + start));       // keys behind count as absent
  const unsigned long long bits = key_bits(a, b, 0, len);
  const int i = qi * 32 + col;                                           // this lane's query
  const T* kb = (const T*)a.k + b * a.vk.sb + hk * a.vk.sh;
  const T* vb = (const T*)a.v + b * a.vv.sb + hk * a.vv.sh;
  // All loads of a head are under way before the first is waited for, and none hangs on another's result: rows that do not
  // exist are read from the last one that does, and what must not count is made zero on its way to LDS.
  constexpr int UKT = (UK + NT - 1) / NT, UQT = (2 * UQ + NT - 1) / NT;
  V8 vf[NC];
  Unit<T> ku[UKT];
  {
    const int j = ki * 32 + col;
    const T* p = vb + (long)min(j, a.Lk - 1) * a.vv.sl;
#pragma unroll
    for (int c = 0; c < NC; ++c) vf[c] = load8<T>(p + c * 16 + half * 8, a.D - c * 16 - half * 8, vec);
#pragma unroll
    for (int n = 0; n < UKT; ++n) {
      const int u = min(tid + n * NT, UK - 1), quad = u / (DP / 8), d = u % (DP / 8) * 8;
      ku[n].load(kb, a.vk.sl, quad * 4, a.Lk, d, a.D, 15u, vec, whole_d && 32 * KB <= a.Lk);
    }
  }
  f32x16 dk[KTILES] = {}, dv[KTILES] = {};
  float fit = 1.f;                                                       // the same in every wave
  for (int g = 0; g < a.G; ++g) {
    const int hq = hk * a.G + g;
    const float* lse_row = a.lse_in + ((long)b * a.Hq + hq) * a.Lq;
    V8 of[NC];
    Unit<T> un[UQT];
    float seen[UQT][4];
    const float lse_i = lse_row[min(i, a.Lq - 1)];
    {
      const T* p = (const T*)a.out_in + b * a.vo.sb + hq * a.vo.sh + (long)min(i, a.Lq - 1) * a.vo.sl;
#pragma unroll
      for (int c = 0; c < NC; ++c) of[c] = load8<T>(p + c * 16 + half * 8, a.D - c * 16 - half * 8, vec);
    }
#pragma unroll
    for (int n = 0; n < UQT; ++n) {
      const int u = min(tid + n * NT, 2 * UQ - 1);
      const bool is_g = u >= UQ;
      const int w = is_g ? u - UQ : u, quad = w / (DP / 8), d = w % (DP / 8) * 8;
      const T* base = is_g ? (const T*)a.dout + b * a.vdo.sb + hq * a.vdo.sh : (const T*)a.q + b * a.vq.sb + hq * a.vq.sh;
      un[n].load(base, is_g ? a.vdo.sl : a.vq.sl, quad * 4, a.Lq, d, a.D, 15u, vec, whole_d && 32 * QB <= a.Lq);
#pragma unroll
      for (int e = 0; e < 4; ++e) seen[n][e] = lse_row[min(quad * 4 + e, a.Lq - 1)];
    }
    if (g > 0) {
      __syncthreads();                                                   // the last head's tiles are done with
    } else {
#pragma unroll
      for (int n = 0; n < UKT; ++n) {
        const int u = tid + n * NT, quad = u / (DP / 8), d = u % (DP / 8) * 8;
        if (u >= UK) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<V8*>(kt + (quad * 4 + e) * S + d) = (bits >> (quad * 4 + e)) & 1 ? ku[n].r[e] : V8{};
      }
      if (!((bits >> (ki * 32 + col)) & 1)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) vf[c] = V8{};
      }
    }
    // queries that see nothing, and those past the end, count as absent, whatever they hold
    const bool live = i < a.Lq && lse_i != -INFINITY;
    const float lse2 = live ? fmaf(lse_i, LOG2E, -P_SHIFT<T>) : INFINITY;
#pragma unroll
    for (int n = 0; n < UQT; ++n) {
      const int u = tid + n * NT;
      const bool is_g = u >= UQ;
      const int w = is_g ? u - UQ : u, quad = w / (DP / 8), d = w % (DP / 8) * 8;
      if (u >= 2 * UQ) continue;
      T* to = (is_g ? gt : qt) + quad * 4 * S + d;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<V8*>(to + e * S) = quad * 4 + e < a.Lq && seen[n][e] != -INFINITY ? un[n].r[e] : V8{};
    }
    __syncthreads();
    f32x16 s = {}, dp = {};
    float delta = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int at = c * 16 + half * 8;
      s = Elem<T>::mma32(*reinterpret_cast<const V8*>(kt + (ki * 32 + col) * S + at), *reinterpret_cast<const V8*>(qt + i * S + at), s);
      const V8 gf = *reinterpret_cast<const V8*>(gt + i * S + at);
      dp = Elem<T>::mma32(vf[c], gf, dp);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf((float)gf[j], (float)of[c][j], delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    delta = live ? delta : 0.f;
    {
      const unsigned word = word_of(bits, ki);
      const int room = (int)max(-64L, min(64L, i + start - ki * 32)) - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale_log2, -lse2));
        const bool on = key_on(word, r) && 8 * (r / 4) + r % 4 <= room;
        s[r] = on ? p : 0.f;
        dp[r] = on ? p * (dp[r] - delta) : 0.f;
      }
    }
    auto put = [&](const f32x16& x) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32v4*>(xt + i * XS + ki * 32 + 8 * q + 4 * half) = f32v4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
    };
    if (FIT<T>) {
      float most = most_of(dp);
      if (__any(most * fit > FIT_LIMIT)) most = wave_most(most);
      if (lane == 0) most_s[wave] = most;
    }
    // tile t of a gradient: token block t / ND, head elements 32 (t % ND) .. + 31
    put(s);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < KTILES; ++n) {
      const int t = wave + n * NW;
      if (KB * ND % NW == 0 || t < KB * ND) {
#pragma unroll
        for (int c = 0; c < 2 * QB; ++c)
          dv[n] = Wide<T>(frag_rows<float>(xt + c * 16 * XS + t / ND * 32 + col, XS, half))
                      .mma(frag_rows<T>(gt + c * 16 * S + t % ND * 32 + col, S, half), dv[n]);
      }
    }
    if (FIT<T>) {
      float most = most_s[0];
#pragma unroll
      for (int w = 1; w < NW; ++w) most = fmaxf(most, most_s[w]);
      if (most * fit > FIT_LIMIT) {
        const float now = fit_for(most);
        if (MANY) {
#pragma unroll
          for (int n = 0; n < KTILES; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[n][r] *= now / fit;
        }
        fit = now;
      }
      if (fit != 1.f) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] *= fit;
      }
    }
    const float back = a.scale * P_UNSHIFT<T> / fit;
    __syncthreads();
    put(dp);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < KTILES; ++n) {
      const int t = wave + n * NW;
      if (KB * ND % NW == 0 || t < KB * ND) {
#pragma unroll
        for (int c = 0; c < 2 * QB; ++c)
          dk[n] = Wide<T>(frag_rows<float>(xt + c * 16 * XS + t / ND * 32 + col, XS, half))
                      .mma(frag_rows<T>(qt + c * 16 * S + t % ND * 32 + col, S, half), dk[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < QTILES; ++n) {
      const int t = wave + n * NW;
      if (QB * ND % NW == 0 || t < QB * ND) {
        f32x16 dq = {};
#pragma unroll
        for (int c = 0; c < 2 * KB; ++c)
          dq = Wide<T>(frag_slots(xt + (t / ND * 32 + col) * XS + c * 16, half))
                   .mma(frag_rows<T>(kt + c * 16 * S + t % ND * 32 + col, S, half), dq);
        const int row = t / ND * 32 + col;
        T* p = (T*)a.dq + b * a.vdq.sb + hq * a.vdq.sh + (long)row * a.vdq.sl;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int d = t % ND * 32 + q * 8 + half * 4;
          if (row < a.Lq && d < a.D)
            store4<T>(p + d, f32v4{dq[4 * q] * back, dq[4 * q + 1] * back, dq[4 * q + 2] * back, dq[4 * q + 3] * back},
                      a.D - d, vec);
        }
      }
    }
  }
  const float back = a.scale * P_UNSHIFT<T> / fit;
#pragma unroll
  for (int n = 0; n < KTILES; ++n) {
    const int t = wave + n * NW, row = t / ND * 32 + col;
    if (t >= KB * ND || row >= a.Lk) continue;
    T* pk = (T*)a.dk + b * a.vdk.sb + hk * a.vdk.sh + (long)row * a.vdk.sl;
    T* pv = (T*)a.dv + b * a.vdv.sb + hk * a.vdv.sh + (long)row * a.vdv.sl;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = t % ND * 32 + q * 8 + half * 4;
      if (d >= a.D) continue;
      store4<T>(pk + d, f32v4{dk[n][4 * q] * back, dk[n][4 * q + 1] * back, dk[n][4 * q + 2] * back, dk[n][4 * q + 3] * back},
                a.D - d, vec);
      store4<T>(pv + d, f32v4{dv[n][4 * q] * P_UNSHIFT<T>, dv[n][4 * q + 1] * P_UNSHIFT<T>, dv[n][4 * q + 2] * P_UNSHIFT<T>,
                              dv[n][4 * q + 3] * P_UNSHIFT<T>}, a.D - d, vec);
    }
  }
}

// dk and dv from the fp32 shares of the dk / dv kernel; a lane has four head elements of one key.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_sum_kernel(AttnArgs a) {
  constexpr int PER = DP / 4;
  const long rows = (long)a.B * a.Hk * a.Lk;
  const long at = (long)blockIdx.x * 256 + threadIdx.x, row = at / PER;
  const int d = (int)(at % PER) * 4;
  if (row >= rows || d >= a.D) return;
  f32v4 dk = {}, dv = {};
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.part_o + (2 * s * rows + row) * DP + d;
    const f32v4 x = *reinterpret_cast<const f32v4*>(p), y = *reinterpret_cast<const f32v4*>(p + rows * DP);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dk[e] += x[e];
      dv[e] += y[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    dk[e] *= a.scale * P_UNSHIFT<T>;
    dv[e] *= P_UNSHIFT<T>;
  }
  const int j = (int)(row % a.Lk), hk = (int)(row / a.Lk % a.Hk), b = (int)(row / a.Lk / a.Hk);
  store4<T>((T*)a.dk + b * a.vdk.sb + hk * a.vdk.sh + (long)j * a.vdk.sl + d, dk, a.D - d, a.vec);
  store4<T>((T*)a.dv + b * a.vdv.sb + hk * a.vdv.sh + (long)j * a.vdv.sl + d, dv, a.D - d, a.vec);
}

}  // namespace trace
