// Rotary positions over the axes of a token grid, and the LayerNorm of every head's queries and keys in front of them, for the packed
// projection rows of the vision transformer (beside MONAI's learned position embedding, dose_pyfer.py:55-67).
//
//   h = (x - mean) * rstd over the d channels of one head;  u = h w + b (w, b shared by all heads: one pair for q, one for k)
//   pair i of the head is turned by angle(token, i) = position[token][axis(i)] * base^(-e(i) / pairs(axis)):
//     (a, b) -> (a cos - b sin, a sin + b cos)
//   backward: g' = the pairs of gy turned by -angle;  gu = g' w;  gx = rstd (gu - mean(gu) - h mean(gu h));  dw = sum g' h;  db = sum g'
//
// Bound: HBM.  A value is read once and written once (the backward pass reads x and gy, writes gx; the row statistics are recomputed from
// the x that is in registers anyway, so nothing but x is kept between the passes).
// Split: a lane owns 8 PAIRS of one head (16 channels, whole 16-byte pieces next to its neighbours'), so that a turn needs no other lane and a
// head is d / 16 lanes whose sums are two or three shuffles.  Cosines and sines belong to a token, not to a head: a block computes those of its
// tokens once into LDS and all heads of q and k share them.  Angles are formed in 64 bits (position * frequency, reduced to a fraction of a
// turn) because a far position times a frequency has no fraction left in 32.
// Measured: turning 27 648 bf16 rows of 12 heads of 64 (85 MB in and out) 15.6 us; with the norm, 13 801 fp32 rows of 16 heads of 64: forward
// 21.4 us (113 MB), backward 37 + 4 us for the weights' sums (170 MB), 27 648 bf16 rows of 12 heads of 64: 20.3 (85 MB), 39.4 + 4 (127 MB); a large
// copy moves 4.9 TB/s, what a kernel before left in the cache comes faster.  1024 rows (12 heads of 128): 7.0 and 12.5 + 3.9 us for about 3 us of
// bytes: the angles and a barrier stand in front of the loads, and the weights' sums are a launch of their own.
#include "common.h"
#include <math.h>

#define STREAM ((hipStream_t)stream)

namespace {

constexpr int MAXPAIRS = 64;
struct RotPlan {
  double freq[MAXPAIRS];             // turns per unit of position
  int axis[MAXPAIRS];
  int pairs, interleaved, naxes, kind;      // pairs < d / 2: the rest of a head keeps its place.  kind: 0 int32, 1 int64, 2 float positions
  const void* pos; int64_t posb;     // elements between two sequences' positions (0: one table for all)
};
struct QkArgs {
  const void *x, *g; void* y;
  int64_t xb, xt, gb, gt, yb, yt;    // element strides of sequence and token
  const float *wq, *bq, *wk, *bk;
  float* part;
  const int* lens;                   // backward: valid tokens of every sequence (NULL: all); what lies behind has no gradient, whatever it holds
  float eps, sgn;
  int hq, hk, tok;
  int64_t N, tokens;
};

// 16 bytes
template <typename T> __device__ __forceinline__ void ld_piece(const T* p, float* v);
template <> __device__ __forceinline__ void ld_piece<float>(const float* p, float* v) {
  const v4f a = *(const v4f*)p;
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = a[i];
}
template <> __device__ __forceinline__ void ld_piece<bf16_t>(const bf16_t* p, float* v) {
  const v4u u = *(const v4u*)p;
#pragma unroll
  for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void ld_piece<f16_t>(const f16_t* p, float* v) {
  const v8h u = *(const v8h*)p;
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (float)u[i];
}
template <typename T> __device__ __forceinline__ void st_piece(T* p, const float* v);
template <> __device__ __forceinline__ void st_piece<float>(float* p, const float* v) { *(v4f*)p = (v4f){v[0], v[1], v[2], v[3]}; }
template <> __device__ __forceinline__ void st_piece<bf16_t>(bf16_t* p, const float* v) {
  v4u u;
#pragma unroll
  for (int i = 0; i < 4; i++) u[i] = (unsigned)f2bf(v[2 * i]) | ((unsigned)f2bf(v[2 * i + 1]) << 16);
  *(v4u*)p = u;
}
template <> __device__ __forceinline__ void st_piece<f16_t>(f16_t* p, const float* v) {
  v8h u;
#pragma unroll
  for (int i = 0; i < 8; i++) u[i] = (f16_t)v[i];
  *(v8h*)p = u;
}

template <int D> struct Lanes { static constexpr int LG = D / 16, LGP = D == 96 ? 8 : D / 16; };

// Which of a head's D / 2 pairs lane c owns: 16-byte pieces c, c + LG, c + 2 LG ..., so that the lanes of a head read consecutive pieces and
// the two members of a pair are both the lane's own (8 consecutive channels per lane instead: 33 -> 21 us forward, 53 -> 37 us backward for fp32
// rows of 16 heads of 64, 13 801 tokens).  PW pairs come with a piece (of each half of the head, or, interleaved, inside it); all types of one
// kernel use the ownership of the storage type T.
template <typename T, int D, bool IN> struct Own {
  static constexpr int EPP = 16 / (int)sizeof(T), PW = IN ? EPP / 2 : EPP, LG = Lanes<D>::LG;
  __device__ __forceinline__ static int pair(int c, int e) { return PW * (c + LG * (e / PW)) + e % PW; }
  __device__ __forceinline__ static int chan(int c, int k) {      // channel of v[k]: k < 8 the first members of the pairs, then the second
    const int p = pair(c, k & 7);
    return IN ? 2 * p + (k >> 3) : p + (k >> 3) * (D / 2);
  }
  // the lane's 16 channels of a row of U (U = T: whole pieces; a wider U: what lies in a piece of T, in pieces of its own)
  template <typename U> __device__ __forceinline__ static void load(const U* p, int c, float* v) {
    constexpr int UP = 16 / (int)sizeof(U), R = sizeof(U) / sizeof(T) > 0 ? EPP / UP : 1;
    static_assert(UP <= EPP, "");
#pragma unroll
    for (int k = 0; k < 16 / EPP; k++) {
      float t[EPP];
      // half layout: the first 8 / EPP pieces from the first half of the head, the others from the second
      const int piece = IN ? c + LG * k : c + LG * (k % (8 / EPP)), base = IN ? 0 : (k / (8 / EPP)) * (D / 2);
#pragma unroll
      for (int r = 0; r < R; r++) ld_piece(p + base + piece * EPP + r * UP, t + r * UP);
      put(t, k, v);
    }
  }
  __device__ __forceinline__ static void store(T* p, int c, const float* v) {
#pragma unroll
    for (int k = 0; k < 16 / EPP; k++) {
      float t[EPP];
      const int piece = IN ? c + LG * k : c + LG * (k % (8 / EPP)), base = IN ? 0 : (k / (8 / EPP)) * (D / 2);
#pragma unroll
      for (int i = 0; i < EPP; i++) t[i] = IN ? v[(k * (EPP / 2) + i / 2) + 8 * (i & 1)] : v[k * EPP + i];
      st_piece(p + base + piece * EPP, t);
    }
  }
  __device__ __forceinline__ static void put(const float* t, int k, float* v) {
#pragma unroll
    for (int i = 0; i < EPP; i++) {
      if (IN) v[(k * (EPP / 2) + i / 2) + 8 * (i & 1)] = t[i]; else v[k * EPP + i] = t[i];
    }
  }
};

template <int LGP> __device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LGP / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// sequence and place of the token t tokens behind (b0, r0)
__device__ __forceinline__ void locate(int64_t N, int64_t b0, int64_t r0, int t, int64_t& b, int64_t& r) {
  b = b0; r = r0 + t;
  while (r >= N) { r -= N; b++; }
}

// cosines and sines of tokens [t0, t0 + n) into LDS [n][D / 2]
template <int D> __device__ __forceinline__ void fill_angles(const RotPlan& R, int64_t N, int64_t b0, int64_t r0, int n, float sgn, float2* cs) {
  for (int i = threadIdx.x; i < n * (D / 2); i += 256) {
    const int t = i / (D / 2), p = i % (D / 2);
    float s = 0.f, c = 1.f;
    if (p < R.pairs) {
      int64_t b, r;
      locate(N, b0, r0, t, b, r);
      const int64_t at = b * R.posb + r * R.naxes + R.axis[p];
      const double x = R.kind == 0 ? (double)((const int*)R.pos)[at] : R.kind == 1 ? (double)((const int64_t*)R.pos)[at] : (double)((const float*)R.pos)[at];
      const double turns = x * R.freq[p];
      sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    }
    cs[i] = make_float2(c, s * sgn);
  }
}

template <int D> __device__ __forceinline__ void head_stats(const float* v, bool on, float eps, float& mean, float& rstd) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e++) s += v[e];
  mean = head_sum<Lanes<D>::LGP>(on ? s : 0.f) * (1.f / D);
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e++) q += (v[e] - mean) * (v[e] - mean);
  rstd = 1.f / sqrtf(head_sum<Lanes<D>::LGP>(on ? q : 0.f) * (1.f / D) + eps);
}

template <typename T, int D, bool NORM, bool IN>
__global__ void __launch_bounds__(256) k_qk_rotary_fwd(const QkArgs a, const RotPlan R) {
  constexpr int LG = Lanes<D>::LG, LGP = Lanes<D>::LGP;
  using O = Own<T, D, IN>;
  extern __shared__ __attribute__((aligned(16))) float2 cs[];
  const int64_t t0 = (int64_t)blockIdx.x * a.tok, b0 = t0 / a.N, r0 = t0 - b0 * a.N;
  const int n = (int)min((int64_t)a.tok, a.tokens - t0), c = threadIdx.x % LGP;
  const bool on = c < LG;
  if (R.pairs) { fill_angles<D>(R, a.N, b0, r0, n, a.sgn, cs); __syncthreads(); }
#pragma unroll
  for (int part = 0; part < 2; part++) {
    const int heads = part ? a.hk : a.hq;
    float w[16], bi[16];
    if (NORM && on && heads) { O::load(part ? a.wk : a.wq, c, w); O::load(part ? a.bk : a.bq, c, bi); }
    for (int i = threadIdx.x / LGP; i < n * heads; i += 256 / LGP) {
      const int t = i / heads, h = i - t * heads + (part ? a.hq : 0);
      int64_t b, r;
      locate(a.N, b0, r0, t, b, r);
      float v[16];
      if (on) O::load((const T*)a.x + b * a.xb + r * a.xt + h * D, c, v);
      if (NORM) {
        float mean, rstd;
        head_stats<D>(v, on, a.eps, mean, rstd);
#pragma unroll
        for (int e = 0; e < 16; e++) v[e] = (v[e] - mean) * rstd * w[e] + bi[e];
      }
      if (R.pairs && on) {
        const float2* q = cs + t * (D / 2);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float2 z = q[O::pair(c, e)];
          const float x0 = v[e], x1 = v[8 + e];
          v[e] = fmaf(x0, z.x, -(x1 * z.y)); v[8 + e] = fmaf(x0, z.y, x1 * z.x);
        }
      }
      if (on) O::store((T*)a.y + b * a.yb + r * a.yt + h * D, c, v);
    }
  }
}

// G: type of the incoming gradient (fp32 where the attention's backward pass keeps the gradient of q and k unrounded for this kernel)
template <typename T, typename G, int D, bool NORM, bool IN>
__global__ void __launch_bounds__(256) k_qk_rotary_bwd(const QkArgs a, const RotPlan R) {
  constexpr int LG = Lanes<D>::LG, LGP = Lanes<D>::LGP;
  using O = Own<T, D, IN>;
  extern __shared__ __attribute__((aligned(16))) float2 cs[];
  const int c = threadIdx.x % LGP;
  const bool on = c < LG;
  float dw[2][16], db[2][16];
#pragma unroll
  for (int p = 0; p < 2; p++)
#pragma unroll
    for (int e = 0; e < 16; e++) { dw[p][e] = 0.f; db[p][e] = 0.f; }
  // (with a norm a block walks over token chunks and adds the weight gradients up in registers: one partial row per block)
  for (int64_t t0 = (int64_t)blockIdx.x * a.tok; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.tok) {
    const int64_t b0 = t0 / a.N, r0 = t0 - b0 * a.N;
    const int n = (int)min((int64_t)a.tok, a.tokens - t0);
    if (R.pairs) { __syncthreads(); fill_angles<D>(R, a.N, b0, r0, n, -1.f, cs); __syncthreads(); }
#pragma unroll
    for (int part = 0; part < 2; part++) {
      const int heads = part ? a.hk : a.hq;
      float w[16];
      if (NORM && on && heads) O::load(part ? a.wk : a.wq, c, w);
      for (int i = threadIdx.x / LGP; i < n * heads; i += 256 / LGP) {
        const int t = i / heads, h = i - t * heads + (part ? a.hq : 0);
        int64_t b, r;
        locate(a.N, b0, r0, t, b, r);
        float g[16], v[16];
        if (a.lens && r >= a.lens[b]) {      // (a head's lanes together.  Padding enters no product: 0 * NaN, or 0 * rstd of a row of zeros, is no zero)
#pragma unroll
          for (int e = 0; e < 16; e++) g[e] = 0.f;
          if (on) O::store((T*)a.y + b * a.yb + r * a.yt + h * D, c, g);
          continue;
        }
        if (on) {
          O::load((const G*)a.g + b * a.gb + r * a.gt + h * D, c, g);
          if (NORM) O::load((const T*)a.x + b * a.xb + r * a.xt + h * D, c, v);
        }
        if (R.pairs && on) {
          const float2* q = cs + t * (D / 2);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float2 z = q[O::pair(c, e)];
            const float g0 = g[e], g1 = g[8 + e];
            g[e] = fmaf(g0, z.x, -(g1 * z.y)); g[8 + e] = fmaf(g0, z.y, g1 * z.x);
          }
        }
        if (NORM) {
          float mean, rstd, s1 = 0.f, s2 = 0.f;
          head_stats<D>(v, on, a.eps, mean, rstd);
          if (on) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
              v[e] = (v[e] - mean) * rstd;
              dw[part][e] += g[e] * v[e]; db[part][e] += g[e];
              g[e] *= w[e];
              s1 += g[e]; s2 += g[e] * v[e];
            }
          }
          s1 = head_sum<LGP>(s1) * (1.f / D); s2 = head_sum<LGP>(s2) * (1.f / D);
#pragma unroll
          for (int e = 0; e < 16; e++) g[e] = rstd * (g[e] - s1 - v[e] * s2);
        }
        if (on) O::store((T*)a.y + b * a.yb + r * a.yt + h * D, c, g);
      }
    }
  }
  if (NORM) {
    __shared__ float red[4][4][D];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        float s = dw[p][e], u = db[p][e];
#pragma unroll
        for (int o = 32; o >= LGP; o >>= 1) { s += __shfl_xor(s, o, 64); u += __shfl_xor(u, o, 64); }
        const int ch = O::chan(c, e);
        if (lane < LGP && on) { red[wv][2 * p][ch] = s; red[wv][2 * p + 1][ch] = u; }
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 4 * D; i += 256) {
      const int k = i / D, ch = i % D;
      a.part[(int64_t)blockIdx.x * 4 * D + i] = (red[0][k][ch] + red[1][k][ch]) + (red[2][k][ch] + red[3][k][ch]);
    }
  }
}

// dw[i] = sum over the partial rows, in a fixed order: 32 row strips per column, each added in 64 bits with four loads in flight
__global__ void __launch_bounds__(1024) k_qk_dw_sum(const float* __restrict__ part, float* __restrict__ dw, int rows, int cols) {
  __shared__ double red[32][32];
  const int cc = threadIdx.x & 31, col = blockIdx.x * 32 + cc, strip = threadIdx.x >> 5;
  double s = 0.0;
  if (col < cols) {
    int r = strip;
    for (; r + 96 < rows; r += 128) {
      const float* p = part + (int64_t)r * cols + col;
      const float x0 = p[0], x1 = p[32 * cols], x2 = p[64 * cols], x3 = p[96 * cols];
      s += ((double)x0 + (double)x1) + ((double)x2 + (double)x3);
    }
    for (; r < rows; r += 32) s += (double)part[(int64_t)r * cols + col];
  }
  red[strip][cc] = s;
  __syncthreads();
  if (strip == 0 && col < cols) {
    double t[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int k = 0; k < 32; k++) t[k & 3] += red[k][cc];
    dw[col] = (float)((t[0] + t[1]) + (t[2] + t[3]));
  }
}

int make_plan(const char* name, RotPlan& R, const void* pos, int pos_kind, int64_t posb, int naxes, const int* sec, double base, int interleaved, int d) {
  R.pairs = 0; R.interleaved = interleaved != 0; R.naxes = naxes; R.kind = pos_kind; R.pos = pos; R.posb = posb;
  if (!pos) return 0;
  if (naxes < 1 || naxes > 4) DP_FAIL("%s: %d position axes (1 to 4)", name, naxes);
  if (pos_kind < 0 || pos_kind > 2) DP_FAIL("%s: position type %d", name, pos_kind);
  if (!(base > 1.0) || !(base < 1e30)) DP_FAIL("%s: base %g", name, base);
  for (int ax = 0; ax < naxes; ax++) {
    if (sec[ax] < 0 || sec[ax] > d / 2) DP_FAIL("%s: %d pairs for axis %d of a head of %d", name, sec[ax], ax, d);
    if (R.pairs + sec[ax] > d / 2) DP_FAIL("%s: more rotated pairs than a head of %d has", name, d);
    R.pairs += sec[ax];
  }
  // (64 powers are 3 us of host time: the table of the configuration that this thread used last is kept)
  static thread_local struct { double base; int sec[4]; int naxes; double freq[MAXPAIRS]; int axis[MAXPAIRS]; } kept = {0.0, {0, 0, 0, 0}, 0, {}, {}};
  bool same = kept.base == base && kept.naxes == naxes;
  for (int ax = 0; ax < naxes && same; ax++) same = kept.sec[ax] == sec[ax];
  if (!same) {
    int n = 0;
    for (int ax = 0; ax < naxes; ax++)
      for (int e = 0; e < sec[ax]; e++) { kept.freq[n] = pow(base, -(double)e / sec[ax]) / 6.283185307179586476925287; kept.axis[n++] = ax; }
    for (int ax = 0; ax < 4; ax++) kept.sec[ax] = ax < naxes ? sec[ax] : 0;
    kept.base = base; kept.naxes = naxes;
  }
  for (int i = 0; i < R.pairs; i++) { R.freq[i] = kept.freq[i]; R.axis[i] = kept.axis[i];
  }
  return 0;
}

int check_rows(const char* name, const void* p, int64_t sb, int64_t st, int es) {
  if (((uintptr_t)p & 15) || (sb * es) % 16 || (st * es) % 16) DP_FAIL("%s: rows must be 16-byte aligned (strides %lld, %lld)", name, (long long)sb, (long long)st);
  return 0;
}

// tokens per block: enough of them that the angles (one per token and pair) spread over all threads, fewer where the grid would not
// fill the 256 CUs.  (One token a block: 28 us instead of 15.6 at 27 648 tokens, with the norm 46 and 103 instead of 22 and 37 at 13 801; eight
// at the 1024 tokens of two 128^3 volumes: 8.7 and 14.2 us instead of 7.2 and 12.6.)
int block_tokens(int64_t tokens) { return tokens >= 8192 ? 8 : tokens >= 2048 ? 4 : tokens >= 512 ? 2 : 1; }

}  // namespace

#define QK_DIMS(d, ...) do { if ((d) == 32) { constexpr int D = 32; __VA_ARGS__; } else if ((d) == 64) { constexpr int D = 64; __VA_ARGS__; } \
    else if ((d) == 96) { constexpr int D = 96; __VA_ARGS__; } else { constexpr int D = 128; __VA_ARGS__; } } while (0)

#define QK_IN(in, ...) do { if (in) { constexpr bool IN = true; __VA_ARGS__; } else { constexpr bool IN = false; __VA_ARGS__; } } while (0)

extern "C" int dp_qk_rotary_parts(int64_t tokens) {
  const int64_t nblk = (tokens + block_tokens(tokens) - 1) / block_tokens(tokens);
  return (int)(nblk < 512 ? nblk : 512);
}

extern "C" int dp_qk_rotary_fwd(const void* x, int64_t xb, int64_t xt, void* y, int64_t yb, int64_t yt, int B, int64_t N, int heads, int kv_heads, int d,
                                const float* wq, const float* bq, const float* wk, const float* bk, float eps, const void* pos, int pos_kind, int64_t posb,
                                int naxes, int s0, int s1, int s2, int s3, double base, int interleaved, int inverse, int dtype, void* stream) {
  if (B < 0 || N < 0 || heads < 0 || kv_heads < 0) DP_FAIL("qk_rotary_fwd: bad sizes B=%d N=%lld heads=%d + %d", B, (long long)N, heads, kv_heads);
  if (d != 32 && d != 64 && d != 96 && d != 128) DP_FAIL("qk_rotary_fwd: head dim %d not in {32, 64, 96, 128}", d);
  if (dtype != DP_F32 && dtype != DP_BF16 && dtype != DP_F16) DP_FAIL("qk_rotary_fwd: bad dtype %d", dtype);
  const bool norm = wq || wk;
  if (norm && ((heads && (!wq || !bq)) || (kv_heads && (!wk || !bk)))) DP_FAIL("qk_rotary_fwd: the norm needs weight and bias for q and for k");
  const int es = dtype == DP_F32 ? 4 : 2;
  if (check_rows("qk_rotary_fwd", x, xb, xt, es) || check_rows("qk_rotary_fwd", y, yb, yt, es)) return 1;
  if (((uintptr_t)wq | (uintptr_t)bq | (uintptr_t)wk | (uintptr_t)bk) & 15) DP_FAIL("qk_rotary_fwd: weights must be 16-byte aligned");
  RotPlan R;
  const int sec[4] = {s0, s1, s2, s3};
  if (make_plan("qk_rotary_fwd", R, pos, pos_kind, posb, naxes, sec, base, interleaved, d)) return 1;
  const int64_t tokens = (int64_t)B * N;
  if (tokens == 0 || heads + kv_heads == 0) return 0;
  if (!x || !y) DP_FAIL("qk_rotary_fwd: x or y missing");
  const int tok = block_tokens(tokens);
  if ((tokens + tok - 1) / tok > 0x7fffffff || (int64_t)tok * (heads + kv_heads) > 0x3fffffff) DP_FAIL("qk_rotary_fwd: too many rows");
  QkArgs a{x, nullptr, y, xb, xt, 0, 0, yb, yt, wq, bq, wk, bk, nullptr, nullptr, eps, inverse ? -1.f : 1.f, heads, kv_heads, tok, N, tokens};
  const size_t smem = R.pairs ? (size_t)tok * (d / 2) * sizeof(float2) : 0;
  const dim3 grid((unsigned)((tokens + tok - 1) / tok));
  DP_DISPATCH(dtype, QK_DIMS(d, QK_IN(R.interleaved, if (norm) hipLaunchKernelGGL((k_qk_rotary_fwd<T, D, true, IN>), grid, dim3(256), smem, STREAM, a, R);
                                                      else hipLaunchKernelGGL((k_qk_rotary_fwd<T, D, false, IN>), grid, dim3(256), smem, STREAM, a, R))));
  DP_CHECK_LAUNCH("qk_rotary_fwd"); return 0;
}

extern "C" int dp_qk_rotary_bwd_ragged(const void* x, int64_t xb, int64_t xt, const void* g, int64_t gb, int64_t gt, int g_f32, void* gx, int64_t gxb, int64_t gxt,
                                       float* part, float* dw, int B, int64_t N, int heads, int kv_heads, int d, const float* wq, const float* wk, float eps,
                                       const void* pos, int pos_kind, int64_t posb, int naxes, int s0, int s1, int s2, int s3, double base, int interleaved,
                                       const int32_t* lengths, int dtype, void* stream) {
  if (B < 0 || N < 0 || heads < 0 || kv_heads < 0) DP_FAIL("qk_rotary_bwd: bad sizes B=%d N=%lld heads=%d + %d", B, (long long)N, heads, kv_heads);
  if (d != 32 && d != 64 && d != 96 && d != 128) DP_FAIL("qk_rotary_bwd: head dim %d not in {32, 64, 96, 128}", d);
  if (dtype != DP_F32 && dtype != DP_BF16 && dtype != DP_F16) DP_FAIL("qk_rotary_bwd: bad dtype %d", dtype);
  const bool norm = wq || wk;
  if (norm && ((heads && !wq) || (kv_heads && !wk) || !dw || (B > 0 && N > 0 && (!part || !x)))) DP_FAIL("qk_rotary_bwd: the norm needs x, both weights, part and dw");
  const int es = dtype == DP_F32 ? 4 : 2;
  if ((norm && check_rows("qk_rotary_bwd", x, xb, xt, es)) || check_rows("qk_rotary_bwd", g, gb, gt, g_f32 ? 4 : es) || check_rows("qk_rotary_bwd", gx, gxb, gxt, es)) return 1;
  if (((uintptr_t)wq | (uintptr_t)wk) & 15) DP_FAIL("qk_rotary_bwd: weights must be 16-byte aligned");
  RotPlan R;
  const int sec[4] = {s0, s1, s2, s3};
  if (make_plan("qk_rotary_bwd", R, pos, pos_kind, posb, naxes, sec, base, interleaved, d)) return 1;
  const int64_t tokens = (int64_t)B * N;
  if (tokens == 0 || heads + kv_heads == 0) {
    if (norm) { hipLaunchKernelGGL(k_qk_dw_sum, dim3(cdiv(4 * d, 32)), dim3(1024), 0, STREAM, (const float*)part, dw, 0, 4 * d); DP_CHECK_LAUNCH("qk_rotary_bwd"); }
    return 0;
  }
  if (!g || !gx) DP_FAIL("qk_rotary_bwd: g or gx missing");
  const int tok = block_tokens(tokens);
  if ((tokens + tok - 1) / tok > 0x7fffffff || (int64_t)tok * (heads + kv_heads) > 0x3fffffff) DP_FAIL("qk_rotary_bwd: too many rows");
  QkArgs a{x, g, gx, xb, xt, gb, gt, gxb, gxt, wq, nullptr, wk, nullptr, part, lengths, eps, 1.f, heads, kv_heads, tok, N, tokens};
  const size_t smem = R.pairs ? (size_t)tok * (d / 2) * sizeof(float2) : 0;
  const int nblk = norm ? dp_qk_rotary_parts(tokens) : (int)((tokens + tok - 1) / tok);
#define QK_BWD(TG) DP_DISPATCH(dtype, QK_DIMS(d, QK_IN(R.interleaved, \
    if (norm) hipLaunchKernelGGL((k_qk_rotary_bwd<T, TG, D, true, IN>), dim3(nblk), dim3(256), smem, STREAM, a, R); \
    else hipLaunchKernelGGL((k_qk_rotary_bwd<T, TG, D, false, IN>), dim3(nblk), dim3(256), smem, STREAM, a, R))))
  if (g_f32) QK_BWD(float); else QK_BWD(T);
  DP_CHECK_LAUNCH("qk_rotary_bwd");
  if (norm) { hipLaunchKernelGGL(k_qk_dw_sum, dim3(cdiv(4 * d, 32)), dim3(1024), 0, STREAM, (const float*)part, dw, nblk, 4 * d); DP_CHECK_LAUNCH("qk_rotary_bwd(dw)"); }
  return 0;
}

extern "C" int dp_qk_rotary_bwd(const void* x, int64_t xb, int64_t xt, const void* g, int64_t gb, int64_t gt, int g_f32, void* gx, int64_t gxb, int64_t gxt,
                                float* part, float* dw, int B, int64_t N, int heads, int kv_heads, int d, const float* wq, const float* wk, float eps,
                                const void* pos, int pos_kind, int64_t posb, int naxes, int s0, int s1, int s2, int s3, double base, int interleaved,
                                int dtype, void* stream) {
  return dp_qk_rotary_bwd_ragged(x, xb, xt, g, gb, gt, g_f32, gx, gxb, gxt, part, dw, B, N, heads, kv_heads, d, wq, wk, eps, pos, pos_kind, posb, naxes, s0, s1,
                                 s2, s3, base, interleaved, nullptr, dtype, stream);
}
