// Attention over a sliding window whose first tokens stay visible, forward and backward: the form of the ViT's attention for token rows
// that are too long for the full one (attention.hip: finer patches, larger crops than the 512 .. 1152 tokens of dose_pyfer.py:55-67).
//
//   key j is seen by the query at position p  iff  p < n, j < n, j <= p + right and (j >= p - left or j < sinks)   (n: valid tokens)
//   O = softmax(scale Q K^T) V over the seen keys; a query that sees nothing, or lies outside [0, n), gives 0.
//   backward, from lse = log2 sum exp2(scale log2e s):  P = exp2(c s - lse), dV = P^T dO, dS = P (dO V^T - delta) scale, dQ = dS K,
//   dK = dS^T Q with delta = rowsum(dO O).  Two passes without atomics (dQ by query rows, dK / dV by key rows): 14 d flop per pair
//   instead of 10, and the same bits every time.
//
// Rows: the query heads that share a key head stand beside each other, row r = (token r / group, head r % group), so that one staged key
// tile serves all of them and a single token with a group of heads is one tile.
// Matrix tiles are 32 x 32 (k = 16).  The score tile is computed transposed (streamed rows x owned columns): a lane then holds one owned
// row's scores, and the accumulator registers are, pair by pair of 8-row groups, the B operand of the second product; its A operand is
// the streamed tile read k-major from LDS (ds_read_b64_tr_b16).  Running maximum and sum are one register per lane, fp32.
//
// Roundings below 32 bits: P and dS go through the second product in the storage type (the matrix cores take nothing wider there), each off by
// half a step of its own size; the row sum adds the rounded P, the ones that the product takes, so that numerator and normaliser agree; delta reads
// O as it was stored.  Everything that is added up stays fp32.  In the 2-norm, windows of 41 to 1153 keys: with its own rounding the result is off by
// 2.0 .. 2.2e-3 in bf16 (the last rounding alone: 1.7e-3) and dQ, dK, dV by 2.4e-3, of which the rounded O inside delta is 0.2 .. 0.6e-3; fp16 an
// eighth of each.
// Bound, heads of 64: in the forward kernel the vector instructions beside the products, in dQ the matrix cores and the LDS alike, in dK / dV the
// LDS (full attention over 8192 keys, shares of the time in which the unit works, forward / dQ / dK, dV: vector issue 66 / 60 / 50 %, matrix 44 / 54 / 53 %,
// LDS 44 / 54 / 66 %).  12 heads, 13 825 tokens, window 576 + 576, one sink, bf16, chip at work: 75, 95 and 124 us + 5 for the sinks' sums, 0.64, 0.76
// and 0.77 PFLOP/s (a large library product: 1.22); 64 keys more a row cost 1.07, 1.27 and 1.27 PFLOP/s (windows of 577 .. 2305 keys).  The rest is
// empty slots: 1308 blocks on the 1024 (forward) and 768 slots that the CUs have for them are 1.3 and 1.7 rounds, 2.8 waves a SIMD on average of 4,
// 2.4 of 3.  Tiles at the window's edges are 4 % more products than needed.
// 6 heads of 128, window 1152 + 1152: 123, 197, 306 us, 0.76, 0.71, 0.61 PFLOP/s.
#include "common.h"
#include <atomic>

#define STREAM ((hipStream_t)stream)

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int FAR = 1 << 30;            // no limit on this side of the window
typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mma32(const Frag8<bf16_t>& a, const Frag8<bf16_t>& b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a.u), __builtin_bit_cast(v8bf, b.u), c, 0, 0, 0);
}
__device__ __forceinline__ v16f mma32(const Frag8<f16_t>& a, const Frag8<f16_t>& b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a.u), __builtin_bit_cast(v8h, b.u), c, 0, 0, 0);
}
__device__ __forceinline__ v16f mma32(const Frag8<float>& a, const Frag8<float>& b, v16f c) {      // exact fp32 chain, same k slots
#pragma unroll
  for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}
// Results of matrix instructions, ready to be read by others.  The wait states are written out (18 behind a 16-pass fp32 instruction, 12 behind an
// 8-pass 16-bit one) and tied to the registers: where a branch stands between the matrix instruction and the first read, the compiler has counted
// them along the longer of two paths and read the last rows of a tile too early.
template <typename T> __device__ __forceinline__ void mma_ready(v16f& x) {
  if constexpr (sizeof(T) == 4) asm volatile("s_nop 15\n\ts_nop 1" : "+v"(x)); else asm volatile("s_nop 11" : "+v"(x));
}
template <typename T> __device__ __forceinline__ void mma_ready(v16f& x, v16f& y) {
  if constexpr (sizeof(T) == 4) asm volatile("s_nop 15\n\ts_nop 1" : "+v"(x), "+v"(y)); else asm volatile("s_nop 11" : "+v"(x), "+v"(y));
}
__device__ __forceinline__ v16f zero16() { v16f z; for (int i = 0; i < 16; i++) z[i] = 0.f; return z; }

template <typename T> __device__ __forceinline__ Frag8<T> ldg8(const T* p) { Frag8<T> f; f.u = *(const v4u*)p; return f; }
template <> __device__ __forceinline__ Frag8<float> ldg8<float>(const float* p) { return frag_ld_lds(p); }
// (pairs through vector conversions: one v_cvt_pk per two values)
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned pack_pair(float a, float b, bf16_t) { return __builtin_bit_cast(unsigned, __builtin_convertvector((v2f){a, b}, v2bf)); }
__device__ __forceinline__ unsigned pack_pair(float a, float b, f16_t) { return __builtin_bit_cast(unsigned, __builtin_convertvector((v2f){a, b}, v2h)); }
template <typename T> __device__ __forceinline__ Frag8<T> pack8(const float* p, T t) {
  Frag8<T> f;
#pragma unroll
  for (int i = 0; i < 4; i++) f.u[i] = pack_pair(p[2 * i], p[2 * i + 1], t);
  return f;
}
__device__ __forceinline__ Frag8<float> pack8(const float* p, float) {
  Frag8<float> f;
#pragma unroll
  for (int i = 0; i < 8; i++) f.v[i] = p[i];
  return f;
}
// sum of the 8 values of a fragment, added to l (two values an instruction; of the rounded values, the ones the second product takes)
// (the word is copied first: a bit cast of a vector's element itself always took element 0)
__device__ __forceinline__ float add8(const Frag8<bf16_t>& f, float l) {
#pragma unroll
  for (int i = 0; i < 4; i++) { const unsigned w = f.u[i]; l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, w), __builtin_bit_cast(v2bf, 0x3f803f80u), l, false); }
  return l;
}
__device__ __forceinline__ float add8(const Frag8<f16_t>& f, float l) {
#pragma unroll
  for (int i = 0; i < 4; i++) { const unsigned w = f.u[i]; l = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w), __builtin_bit_cast(v2h, 0x3c003c00u), l, false); }
  return l;
}
__device__ __forceinline__ float add8(const Frag8<float>& f, float l) {
#pragma unroll
  for (int i = 0; i < 8; i++) l += f.v[i];
  return l;
}
template <typename T> __device__ __forceinline__ float elem(const Frag8<T>& f, int i) {
  const unsigned short h = (unsigned short)(f.u[i >> 1] >> (16 * (i & 1)));
  return ld_f((const T*)&h);
}
template <> __device__ __forceinline__ float elem<float>(const Frag8<float>& f, int i) { return f.v[i]; }
__device__ __forceinline__ void st4(float* p, const float* v) { *(v4f*)p = (v4f){v[0], v[1], v[2], v[3]}; }
template <typename T> __device__ __forceinline__ void st4(T* p, const float* v) { *(uint2*)p = make_uint2(pack_pair(v[0], v[1], T{}), pack_pair(v[2], v[3], T{})); }

// over the two lanes that hold halves of one owned row
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T, int D> struct Cfg {
  static constexpr int ES = sizeof(T), PITCH = D * ES;         // bytes of a row in LDS: no padding, the copies below write 1 KB runs
  static constexpr int PPR = PITCH / 16, SW = PPR % 8 == 0 ? 7 : 3;
  static constexpr int KK = D / 16, DT = D / 32, CP = D + 4;   // k steps, output tiles, fp32 pitch of the merge tile
};

// Tiles go from memory to LDS without passing registers (buffer_load ... lds: 64 lanes x 16 bytes to consecutive LDS addresses).  What keeps
// the reads apart in the banks is the order of a row's 16-byte pieces: piece c of row r stands in place c ^ (r & SW), chosen by the
// address each lane loads from.  Heads of 64 in 16 bits: the LDS works for as many cycles as the reads have bytes over 128, so nothing waits (8
// cycles a matrix instruction in the forward kernel, 10 in dK / dV; the conflict counter shows half of every read of 8 or 16 bytes a lane all the
// same).  Heads of 128, rows of 256 bytes: 12 instead of 8, the transposing reads take twice their cycles.
// Rows behind `left` are out of the descriptor's range and arrive as zeros.
typedef int v4i __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4i rsrc_of(const void* p, unsigned bytes) {
  const uint64_t u = (uint64_t)(uintptr_t)p;
  return (v4i){__builtin_amdgcn_readfirstlane((int)u), __builtin_amdgcn_readfirstlane((int)(u >> 32)), __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
// In assembly (no register is loaded, so nothing can be reused too early) because the compiler would wait for every copy under way in front of
// each transposing LDS read, whatever tile it reads; the waits are written out in stream_tiles.  (s_nop: the descriptor may come from vector
// instructions, whose scalar results a buffer load must not read for five states; M0 needs one.)
__device__ __forceinline__ void lds_copy(v4i rs, char* lds, int off) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(off), "s"(rs) : "memory");
}
// DIRECT false: through registers, for tiles beyond the 64 KB of LDS that such a copy can address
template <typename T, int D, int ROWS, int NTH, bool DIRECT> struct Copy {
  using C = Cfg<T, D>;
  static constexpr int NP = ROWS * C::PPR / NTH;
  static_assert(NP * NTH == ROWS * C::PPR, "every piece of a tile has a thread");
  int off[NP], stride;       // stride: bytes between rows
  __device__ __forceinline__ Copy(int64_t st, int gid) : stride((int)st * C::ES) {
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int idx = gid + i * NTH, row = idx / C::PPR;
      off[i] = row * stride + (((idx % C::PPR) ^ (row & C::SW)) << 4);
    }
  }
  // rows first .. first + ROWS - 1 of `base`, of which `left` exist
  __device__ __forceinline__ void issue(const T* base, int64_t st, int first, int left, char* lds, int wave) const {
    const auto rs = rsrc_of(base + (int64_t)first * st, (unsigned)(min(left, ROWS) * stride));
#pragma unroll
    for (int i = 0; i < NP; i++)
      if (DIRECT) lds_copy(rs, lds + (i * NTH + wave * 64) * 16, off[i]);
    if (!DIRECT) {
      const auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)first * st), 0, min(left, ROWS) * stride, 0x00020000);
      v4u r[NP];
#pragma unroll
      for (int i = 0; i < NP; i++) r[i] = __builtin_amdgcn_raw_buffer_load_b128(rb, off[i], 0, 0);
#pragma unroll
      for (int i = 0; i < NP; i++) *(v4u*)(lds + (i * NTH + (threadIdx.x & (NTH - 1))) * 16) = r[i];
    }
  }
};
// this wave's copies have landed
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// this wave's LDS reads are done: their tile may be filled again
__device__ __forceinline__ void reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Operand fragments of a staged tile.  Lane addresses are formed once (with the wave's own part of LDS, `base`); tile, row and step are
// constants behind them: an exclusive-or below SW + 1, the rest added, so they end up in the read's offset field.
template <typename T, int D> struct Frags {
  using C = Cfg<T, D>;
  int row, fx, tr, tx;
  int ra[4], ca[2];      // 16-bit: the different lane addresses there are, kept in registers (formed anew for every step otherwise; heads of 128 have none to spare)
  __device__ __forceinline__ Frags(int lane, int base) {
    const int c32 = lane & 31, h = lane >> 5, r = lane & 15, f = c32 & C::SW;
    row = base + c32 * C::PITCH;
    fx = C::ES == 2 ? h ^ f : (2 * h) ^ f;
    if (C::ES == 2) {      // four rows of 16 channels per 16 lanes, transposed on the way
      const int tr_row = 4 * h + (r >> 2);
      tr = base + tr_row * C::PITCH + 8 * (r & 1);
      tx = (2 * ((lane >> 4) & 1) + ((r >> 1) & 1)) ^ (tr_row & C::SW);
    } else {
      tr = base + 4 * h * C::PITCH + 4 * (c32 & 3);
      tx = (c32 >> 2) ^ (4 * h);
    }
#pragma unroll
    for (int i = 0; i < (C::SW + 1) / 2; i++) { ra[i] = row + (((2 * i) ^ fx) << 4); if (D < 128) asm("" : "+v"(ra[i])); }
#pragma unroll
    for (int i = 0; i < (C::SW + 1) / 4; i++) { ca[i] = tr + (((4 * i) ^ tx) << 4); if (D < 128) asm("" : "+v"(ca[i])); }
  }
  // byte of piece p, swizzled by x
  __device__ __forceinline__ static int piece(int p, int x) { return (((p & C::SW) ^ x) << 4) + ((p & ~C::SW) << 4); }
  // row (lane & 31) of the 32 rows from r0 on, channels 16 kk + 8 (lane >> 5) .. + 7
  __device__ __forceinline__ Frag8<T> rows(const char* tile, int r0, int kk) const {
    const char* p = tile + r0 * C::PITCH;
    if constexpr (C::ES == 2) { Frag8<T> f; f.u = *(const v4u*)(p + ((2 * kk & ~C::SW) << 4) + ra[(2 * kk & C::SW) / 2]); return f; }
    else {
      const v4f a = *(const v4f*)(p + (row + piece(4 * kk, fx))), b = *(const v4f*)(p + (row + piece(4 * kk + 1, fx)));
      Frag8<T> f;
      f.v[0] = a[0]; f.v[1] = a[1]; f.v[2] = a[2]; f.v[3] = a[3]; f.v[4] = b[0]; f.v[5] = b[1]; f.v[6] = b[2]; f.v[7] = b[3];
      return f;
    }
  }
  // k-major: channel 32 dt + (lane & 31) of the 16 rows from r0 on, in the order of the accumulator registers (rows 4 h .. 4 h + 3 and
  // 8 + 4 h .. 8 + 4 h + 3 of lane half h)
  __device__ __forceinline__ Frag8<T> cols(const char* tile, int r0, int dt) const {
    const char* p = tile + r0 * C::PITCH;
    if constexpr (C::ES == 2) return tr_pair<8 * D, T>((const T*)(p + ((4 * dt & ~C::SW) << 4) + ca[(4 * dt & C::SW) / 4]));
    else {
      Frag8<T> f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const char* q = p + j * C::PITCH + 128 * dt + (tr + ((tx ^ j) << 4));
        f.v[j] = *(const float*)q; f.v[4 + j] = *(const float*)(q + 8 * C::PITCH);
      }
      return f;
    }
  }
};

// Waves per SIMD that the register budget is cut for.  Two (256 registers) also keep the matrix accumulators in plain VGPRs: with more the
// compiler puts them into AGPRs and copies them back and forth around every rescale and mask (24 instead of 9 vector instructions per
// matrix instruction in the forward kernel).  One where two would spill (fp32 dK / dV of 128, narrow: 22 registers spill even so, 92 bytes of scratch).
template <typename T, int D, bool WIDE> constexpr int waves_fwd() { return sizeof(T) == 4 && D >= 96 ? 1 : sizeof(T) == 2 && D == 128 && WIDE ? 3 : 2; }
template <typename T, int D> constexpr int waves_dq() { return sizeof(T) == 4 && D >= 96 ? 1 : 2; }
template <typename T, int D> constexpr int waves_kv() { return sizeof(T) == 4 && D >= 64 ? 1 : sizeof(T) == 2 && D == 64 ? 3 : 2; }

struct Mat { void* p; int64_t b, t, h; };      // element strides of sequence, token and head
struct WinArgs {
  Mat q, k, v, o, go, dq, dk, dv;
  float *lse, *delta, *part;      // delta: rowsum(dO O) * scale
  const int *starts, *lens;
  int kv, group, Nq, Nk, rows, left, right, sinks, start, tiles, nsplit, sink_tiles, nchunk, g_f32;
  float c, lag, scale;      // c = scale * log2(e); lag: LAG powers of two in units of a score
};
constexpr float LAG = 8.f;

// contiguous ranges of the (batch, key head, tile) space per XCD: the blocks of one XCD's L2 read the same keys
__device__ __forceinline__ int xcd_range(int id, int total) {
  const int q = total >> 3, rem = total & 7, x = id & 7;
  return x * q + min(x, rem) + (id >> 3);
}

struct Seq { int start, len; };
__device__ __forceinline__ Seq sequence(const WinArgs& a, int b) {
  Seq s;
  s.len = a.lens ? min(max(a.lens[b], 0), a.Nk) : a.Nk;
  s.start = a.starts ? min(max(a.starts[b], -FAR), FAR) : a.start;
  return s;
}

template <typename T, int D, bool WIDE> struct Shape {
  using C = Cfg<T, D>;
  // WIDE: four waves own 32 rows each and share every staged tile (one barrier per tile).  Otherwise all four own the same 32 rows, stream
  // different tiles through LDS of their own and are merged at the end: four times the blocks, a quarter of the chain.
  // (heads of 128: 32-key tiles and 168 registers, so that three blocks stay on a CU instead of two: 172 -> 156 us at 6 heads, window 1152)
  static constexpr int KS = (WIDE && C::ES == 2 && D < 128) ? 2 : 1, KT = 32 * KS, ROWS = WIDE ? 128 : 32, NTH = WIDE ? 256 : 64;
  // tiles in LDS per stream: wide, the next one arrives while one is worked on; narrow, one, and more blocks on a CU instead (2 x 1024 tokens, 12
  // heads of 64, window 513: 16.3 -> 12.8, 19.7 -> 16.2 and, with dK / dV at three waves, 21.3 -> 17.2 us; chains of 1153 keys: 27 -> 23, 32 -> 33,
  // 44 -> 45)
  static constexpr int NBUF = WIDE ? 2 : 1;
  static constexpr int tile = KT * C::PITCH, sets = (WIDE ? 1 : 4) * NBUF, stage = sets * 2 * tile;
  static constexpr bool DIRECT = stage <= 64 * 1024;
  static constexpr int merge = WIDE ? 0 : 4 * 32 * C::CP * 4, big = stage > merge ? stage : merge;
  static constexpr int fwd = big + (WIDE ? 0 : 2 * 4 * 32 * 4);
  // dK / dV: tiles of RT query rows and of the output's gradient, their lse and delta behind all tiles
  static constexpr int RS = (WIDE && C::ES == 2 && D < 128) ? 2 : 1, RT = 32 * RS, rtile = RT * C::PITCH, rstage = sets * 2 * rtile;
  // heads of 128 in 16 bits: the owned keys' values wait in LDS too, not in registers (two waves per SIMD instead of one)
  static constexpr bool VLDS = C::ES == 2 && D == 128;
  static constexpr int vals = rstage + sets * 512, kv_all = vals + (VLDS ? ROWS * C::PITCH : 0), kvb = kv_all > merge ? kv_all : merge;
  static_assert(fwd <= 160 * 1024 && kvb <= 160 * 1024, "LDS of a CU");
};

// the tiles of KT keys that rows at positions [p0, p1] see at all: `nsink` from key 0 on, then from tile w0 on, nt in all
struct Plan { int nsink, w0, nt; };
template <int KT> __device__ __forceinline__ Plan key_tiles(const WinArgs& a, int len, int p0, int p1) {
  Plan k{0, 0, 0};
  p0 = max(p0, 0); p1 = min(p1, len - 1);
  if (p0 > p1) return k;
  const int lo = max(0, p0 - a.left), hi = min(len - 1, p1 + a.right);
  k.w0 = lo / KT;
  k.nsink = min((min(a.sinks, len) + KT - 1) / KT, k.w0);
  k.nt = k.nsink + hi / KT - k.w0 + 1;
  return k;
}

// what one lane's query row may see: keys [.., hi] that are >= lo or a sink
struct Row { int r, i, g, p, lo, hi; bool live; };
__device__ __forceinline__ Row row_of(const WinArgs& a, const Seq& s, int r) {
  Row w;
  w.r = r;
  const int rc = min(r, a.rows - 1);
  w.i = rc / a.group; w.g = rc - w.i * a.group; w.p = s.start + w.i;
  w.live = r < a.rows && w.p >= 0 && w.p < s.len;
  w.hi = w.live ? min(w.p + a.right, s.len - 1) : -1;
  w.lo = w.live ? w.p - a.left : 0;
  return w;
}
// ... and what a wave's rows see of 32 keys: nothing, all of it, or some
struct Rows {
  int p0, p1; bool any;
  __device__ __forceinline__ Rows(const WinArgs& a, const Seq& s, int r0) : p0(s.start + r0 / a.group), p1(s.start + min(r0 + 31, a.rows - 1) / a.group), any(r0 < a.rows) {}
  __device__ __forceinline__ bool none(const WinArgs& a, int k0) const { return !any || k0 > p1 + a.right || (k0 + 31 < p0 - a.left && k0 >= a.sinks); }
  __device__ __forceinline__ bool all(const WinArgs& a, const Seq& s, int k0) const {
    return k0 + 31 <= min(p0 + a.right, s.len - 1) && (k0 >= p1 - a.left || k0 + 32 <= a.sinks);
  }
};

// LDS reads written above this line are issued before what follows: left alone, the compiler reads each operand right in front of its matrix
// instruction and waits out the LDS latency every time.  (fp32 operands take twice the registers: there the compiler's own order stays.)
#define READS_FIRST do { if (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0); } while (0)
// Loads of the prologue are waited for before the loop: otherwise the waits for them sit inside it and hold up the copies instead.
#define PROLOGUE_LOADED __builtin_amdgcn_s_waitcnt(0)

// s += X x, t += Y y over the head dimension: 32 rows from r0 on of two staged tiles against fragments x[k], y(k)
template <typename T, int D, int G, typename Y>
__device__ __forceinline__ void two_products(const Frags<T, D>& F, const char* x0, const char* y0, int r0, const Frag8<T>* x, Y y, v16f& s, v16f& t) {
#pragma unroll
  for (int g = 0; g < Cfg<T, D>::KK; g += G) {
    Frag8<T> xf[G], yf[G], yr[G];
#pragma unroll
    for (int i = 0; i < G; i++) { xf[i] = F.rows(x0, r0, g + i); yf[i] = F.rows(y0, r0, g + i); yr[i] = y(g + i); }
    READS_FIRST;
#pragma unroll
    for (int i = 0; i < G; i++) { s = mma32(xf[i], x[g + i], s); t = mma32(yf[i], yr[i], t); }
  }
}
// k steps whose operands are read together (an fp32 operand is twice the registers)
template <typename T, int D> constexpr int read_group() { return sizeof(T) == 4 ? 1 : D == 32 ? 2 : D == 96 ? 3 : 4; }

// scores of keys k0 .. k0 + 31 that the lane's row does not see -> `none`.  Behind the sinks a seen key is one range: one subtraction and one
// unsigned comparison a key.  (A row that is not live may keep any value: its column is thrown away.)
__device__ __forceinline__ void mask_keys(v16f& s, const Row& row, int k0, int h, int sinks, float none) {
  if (k0 < sinks) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int j = k0 + 8 * (i >> 2) + 4 * h + (i & 3);
      s[i] = (j <= row.hi && (j >= row.lo || j < sinks)) ? s[i] : none;
    }
    return;
  }
  const int off = k0 + 4 * h - row.lo;
  const unsigned span = (unsigned)(row.hi - row.lo);
#pragma unroll
  for (int i = 0; i < 16; i++) s[i] = (unsigned)(off + 8 * (i >> 2) + (i & 3)) <= span ? s[i] : none;
}

// The stream of a block's tiles: tile(t, i) issues the copies of tile t into buffer i, land(i) stores what came in registers, work(t, i)
// computes; i is a constant of the code (the loop holds both buffers' turns).  Wide: the copies of the next tile run while this one is worked on; a
// wave passes the barrier when its own copies have landed, so behind it everyone's have, and everyone is done with the buffer that is filled
// next.  Narrow: a wave by itself, every fourth tile.
template <int I> struct Buf { static constexpr int v = I; };
template <typename S, typename TILE, typename LAND, typename WORK>
__device__ __forceinline__ void stream_tiles(int t0, int t1, TILE tile, LAND land, WORK work) {
  int t = t0;
  if constexpr (S::NBUF == 2) {
    auto turn = [&](auto i) __attribute__((always_inline)) {
      loads_done();
      land(i);
      lds_barrier();
      if (t + 1 < t1) tile(t + 1, Buf<1 - decltype(i)::v>());
      work(t, i);
      t++;
    };
    if (t < t1) tile(t, Buf<0>());
    PROLOGUE_LOADED;
    while (t < t1) {
      turn(Buf<0>());
      if (t >= t1) break;
      turn(Buf<1>());
    }
  } else {
    for (; t < t1; t += 4) {
      reads_done();
      tile(t, Buf<0>());
      loads_done();
      land(Buf<0>());
      work(t, Buf<0>());
    }
  }
}

template <typename T> __device__ __forceinline__ void st4_grad(void* p, int64_t off, int f32, const float* v) {
  if (f32) st4((float*)p + off, v); else st4((T*)p + off, v);
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(256, (waves_fwd<T, D, WIDE>())) void k_win_fwd(const WinArgs a) {
  using C = Cfg<T, D>;
  using S = Shape<T, D, WIDE>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, h = lane >> 5;
  int flat = xcd_range(blockIdx.x, gridDim.x);
  const int split = flat % a.nsplit; flat /= a.nsplit;
  const int bh = flat / a.tiles, tile = flat % a.tiles, b = bh / a.kv, kvh = bh % a.kv, r0 = tile * S::ROWS;
  const Seq sq = sequence(a, b);
  const int wr0 = WIDE ? r0 + 32 * wv : r0;
  const Row row = row_of(a, sq, wr0 + c32);
  const Rows wave(a, sq, wr0);
  const T* Kb = (const T*)a.k.p + (int64_t)b * a.k.b + (int64_t)kvh * a.k.h;
  const T* Vb = (const T*)a.v.p + (int64_t)b * a.v.b + (int64_t)kvh * a.v.h;
  const T* Qr = (const T*)a.q.p + (int64_t)b * a.q.b + (int64_t)row.i * a.q.t + (int64_t)(kvh * a.group + row.g) * a.q.h;
  Frag8<T> qf[C::KK];
#pragma unroll
  for (int kk = 0; kk < C::KK; kk++) qf[kk] = ldg8(Qr + 16 * kk + 8 * h);
  v16f acc[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; dt++) acc[dt] = zero16();
  float lim = -INFINITY, mc = 0.f, l = 0.f;      // nothing seen yet: lim = -inf, mc = 0
  const Plan pl = key_tiles<S::KT>(a, sq.len, sq.start + r0 / a.group, sq.start + (min(r0 + S::ROWS, a.rows) - 1) / a.group);
  const int per = (pl.nt + a.nsplit - 1) / a.nsplit, t0 = split * per, t1 = min(pl.nt, t0 + per);
  const int own = WIDE ? 0 : wv * S::NBUF * 2 * S::tile;      // the wave's tiles
  const Frags<T, D> F(lane, own);
  auto key_of = [&](int t) { return (t < pl.nsink ? t : pl.w0 + t - pl.nsink) * S::KT; };

  auto step = [&](const char* ks, const char* vs, int u, int k0) __attribute__((always_inline)) {      // 32 keys, k0 the first of them, rows 32 u .. of the tile
    if (wave.none(a, k0)) return;
    v16f s = zero16();
    {
      constexpr int G = C::KK == 6 ? 3 : C::KK == 4 ? 4 : 2;
#pragma unroll
      for (int g = 0; g < C::KK; g += G) {
        Frag8<T> kf[G];
#pragma unroll
        for (int i = 0; i < G; i++) kf[i] = F.rows(ks, 32 * u, g + i);
        READS_FIRST;
#pragma unroll
        for (int i = 0; i < G; i++) s = mma32(kf[i], qf[g + i], s);
      }
    }
    Frag8<T> vf[C::DT];      // the values of the first 16 keys are on their way while the softmax is worked out
#pragma unroll
    for (int dt = 0; dt < C::DT; dt++) vf[dt] = F.cols(vs, 32 * u, dt);
    READS_FIRST;
    mma_ready<T>(s);
    if (!wave.all(a, sq, k0)) mask_keys(s, row, k0, h, a.sinks, -INFINITY);
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
    // The subtracted maximum lags behind: it moves when a score passes it by more than LAG (in powers of two), so that P <= 2^LAG -- the
    // relative precision of P, its sum and the products is the same -- and the first tiles do not rescale the accumulators one after another
    // (some row of 32 sees a new maximum in most of its first 40 tiles: 90 -> 81 us at the window of 1153 keys, heads of 64).
    // (Every row decides for itself: one that stays has alpha = 2^0, exactly 1, whatever the wave's other rows do.)
    mx = pair_max(mx);
    if (__builtin_amdgcn_ballot_w64(mx > lim)) {
      const float nc = mx > lim ? mx * a.c : mc, alpha = lim == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - nc);
      lim = mx > lim ? mx + a.lag : lim; mc = nc; l *= alpha;
#pragma unroll
      for (int dt = 0; dt < C::DT; dt++) acc[dt] *= alpha;
    }
#pragma unroll
    for (int st = 0; st < 2; st++) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; i++) p[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * st + i], a.c, -mc));
      const Frag8<T> pf = pack8(p, T{});
      l = add8(pf, l);
      Frag8<T> vn[C::DT];
      if (st == 0) {
#pragma unroll
        for (int dt = 0; dt < C::DT; dt++) vn[dt] = F.cols(vs, 32 * u + 16, dt);
        READS_FIRST;
      }
#pragma unroll
      for (int dt = 0; dt < C::DT; dt++) { acc[dt] = mma32(vf[dt], pf, acc[dt]); if (st == 0) vf[dt] = vn[dt]; }
    }
  };

  const int gid = WIDE ? tid : lane, wave_id = WIDE ? wv : 0;
  const Copy<T, D, S::KT, S::NTH, S::DIRECT> ck(a.k.t, gid), cv(a.v.t, gid);
  stream_tiles<S>(WIDE ? t0 : t0 + wv, t1,
    [&](int t, auto i) {
      const int k0 = key_of(t);
      char* at = smem + own + decltype(i)::v * 2 * S::tile;
      ck.issue(Kb, a.k.t, k0, sq.len - k0, at, wave_id); cv.issue(Vb, a.v.t, k0, sq.len - k0, at + S::tile, wave_id);
    },
    [](auto) {},
    [&](int t, auto i) {
      const int k0 = key_of(t);
      const char* at = smem + decltype(i)::v * 2 * S::tile;
#pragma unroll
      for (int u = 0; u < S::KS; u++) step(at, at + S::tile, u, k0 + 32 * u);
    });
  l = pair_sum(l);
#pragma unroll
  for (int dt = 0; dt < C::DT; dt++) mma_ready<T>(acc[dt]);
  if (WIDE) {
    if (row.r < a.rows) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* Or = (T*)a.o.p + (int64_t)b * a.o.b + (int64_t)row.i * a.o.t + (int64_t)(kvh * a.group + row.g) * a.o.h;
#pragma unroll
      for (int dt = 0; dt < C::DT; dt++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; j++) v[j] = row.live ? acc[dt][4 * q + j] * inv : 0.f;
          st4(Or + 32 * dt + 8 * q + 4 * h, v);
        }
      if (h == 0 && a.lse) a.lse[(int64_t)bh * a.rows + row.r] = row.live && l != 0.f ? mc + __builtin_amdgcn_logf(l) : INFINITY;
    }
    return;
  }

  if (!row.live) { l = 0.f; lim = -INFINITY; }
  float* part = (float*)smem;
  float* mw = (float*)(smem + S::big);
  float* lw = mw + 4 * 32;
  __syncthreads();      // every wave is done with its tiles
  if (h == 0) { mw[wv * 32 + c32] = lim == -INFINITY ? -INFINITY : mc; lw[wv * 32 + c32] = l; }
#pragma unroll
  for (int dt = 0; dt < C::DT; dt++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = row.live ? acc[dt][4 * q + j] : 0.f;
      st4(part + (wv * 32 + c32) * C::CP + 32 * dt + 8 * q + 4 * h, v);
    }
  __syncthreads();
  for (int idx = tid; idx < 32 * (D / 4); idx += 256) {
    const int rr = idx / (D / 4), c4 = idx % (D / 4), r = r0 + rr;
    if (r >= a.rows) break;      // (rows only grow with idx)
    float M = mw[rr];
#pragma unroll
    for (int w = 1; w < 4; w++) M = fmaxf(M, mw[w * 32 + rr]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float e = __builtin_amdgcn_exp2f(mw[w * 32 + rr] - Ms);
      const v4f x = *(const v4f*)(part + (w * 32 + rr) * C::CP + 4 * c4);
      L += lw[w * 32 + rr] * e;
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += x[j] * e;
    }
    if (a.nsplit > 1) {
      float* ws = a.part + ((int64_t)(bh * a.nsplit + split) * a.rows + r) * (D + 4);
      st4(ws + 4 * c4, v);
      if (c4 == 0) { ws[D] = M; ws[D + 1] = L; }
      continue;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int i = r / a.group, g = r - i * a.group;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] *= inv;
    st4((T*)a.o.p + (int64_t)b * a.o.b + (int64_t)i * a.o.t + (int64_t)(kvh * a.group + g) * a.o.h + 4 * c4, v);
    if (c4 == 0 && a.lse) a.lse[(int64_t)bh * a.rows + r] = L != 0.f ? Ms + __builtin_amdgcn_logf(L) : INFINITY;
  }
}

// few rows, many keys: the shares of the key tiles of one row, merged in share order.  A wave takes every fourth share; statistics of all
// shares (at most 64) sit in one register per lane.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_win_merge(const WinArgs a) {
  __shared__ float part[4][D];
  const int bh = blockIdx.y, r = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6, b = bh / a.kv, kvh = bh % a.kv;
  const float* ws = a.part + ((int64_t)bh * a.nsplit * a.rows + r) * (D + 4);
  const int64_t step = (int64_t)a.rows * (D + 4);
  const float m = lane < a.nsplit ? ws[lane * step + D] : -INFINITY, l = lane < a.nsplit ? ws[lane * step + D + 1] : 0.f;
  const float M = wave_max(m), Ms = M == -INFINITY ? 0.f : M, e = __builtin_amdgcn_exp2f(m - Ms), L = wave_sum(l * e);
  float v[2] = {0.f, 0.f};
  for (int s = wv; s < a.nsplit; s += 4) {
    const float f = __shfl(e, s, 64);
#pragma unroll
    for (int k = 0; k < (D + 63) / 64; k++) if (lane + 64 * k < D) v[k] += ws[s * step + lane + 64 * k] * f;
  }
#pragma unroll
  for (int k = 0; k < (D + 63) / 64; k++) if (lane + 64 * k < D) part[wv][lane + 64 * k] = v[k];
  __syncthreads();
  const int i = r / a.group, g = r - i * a.group;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* o = (T*)a.o.p + (int64_t)b * a.o.b + (int64_t)i * a.o.t + (int64_t)(kvh * a.group + g) * a.o.h;
  if (threadIdx.x < D) st_f(o + threadIdx.x, (part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x]) * inv);
  if (threadIdx.x == 0 && a.lse) a.lse[(int64_t)bh * a.rows + r] = L != 0.f ? Ms + __builtin_amdgcn_logf(L) : INFINITY;
}

// ------------------------------------------------------------------------------------------------ backward: dQ (and delta)
template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(256, (waves_dq<T, D>())) void k_win_dq(const WinArgs a) {
  using C = Cfg<T, D>;
  using S = Shape<T, D, WIDE>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, h = lane >> 5;
  const int flat = xcd_range(blockIdx.x, gridDim.x);
  const int bh = flat / a.tiles, tile = flat % a.tiles, b = bh / a.kv, kvh = bh % a.kv, r0 = tile * S::ROWS;
  const Seq sq = sequence(a, b);
  const int wr0 = WIDE ? r0 + 32 * wv : r0;
  const Row row = row_of(a, sq, wr0 + c32);
  const Rows wave(a, sq, wr0);
  const int head = kvh * a.group + row.g;
  const T* Kb = (const T*)a.k.p + (int64_t)b * a.k.b + (int64_t)kvh * a.k.h;
  const T* Vb = (const T*)a.v.p + (int64_t)b * a.v.b + (int64_t)kvh * a.v.h;
  const T* Qr = (const T*)a.q.p + (int64_t)b * a.q.b + (int64_t)row.i * a.q.t + (int64_t)head * a.q.h;
  const T* Gr = (const T*)a.go.p + (int64_t)b * a.go.b + (int64_t)row.i * a.go.t + (int64_t)head * a.go.h;
  const T* Or = (const T*)a.o.p + (int64_t)b * a.o.b + (int64_t)row.i * a.o.t + (int64_t)head * a.o.h;
  Frag8<T> qf[C::KK], gf[C::KK];
  float dl = 0.f;
#pragma unroll
  for (int kk = 0; kk < C::KK; kk++) {
    qf[kk] = ldg8(Qr + 16 * kk + 8 * h); gf[kk] = ldg8(Gr + 16 * kk + 8 * h);
    const Frag8<T> of = ldg8(Or + 16 * kk + 8 * h);
#pragma unroll
    for (int i = 0; i < 8; i++) dl += elem(of, i) * elem(gf[kk], i);
  }
  dl = pair_sum(dl) * a.scale;      // (from O as stored, half a step of it off: the forward pass keeps nothing wider)
  const float lse = row.live ? a.lse[(int64_t)bh * a.rows + row.r] : INFINITY;
  if (row.r < a.rows && h == 0 && (WIDE || wv == 0)) a.delta[(int64_t)bh * a.rows + row.r] = row.live ? dl : 0.f;
  v16f acc[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; dt++) acc[dt] = zero16();
  const Plan pl = key_tiles<S::KT>(a, sq.len, sq.start + r0 / a.group, sq.start + (min(r0 + S::ROWS, a.rows) - 1) / a.group);
  const int own = WIDE ? 0 : wv * S::NBUF * 2 * S::tile;      // the wave's tiles
  const Frags<T, D> F(lane, own);
  auto key_of = [&](int t) { return (t < pl.nsink ? t : pl.w0 + t - pl.nsink) * S::KT; };

  auto step = [&](const char* ks, const char* vs, int u, int k0) __attribute__((always_inline)) {
    if (wave.none(a, k0)) return;
    v16f s = zero16(), dp = zero16();
    two_products<T, D, read_group<T, D>()>(F, ks, vs, 32 * u, qf, [&](int k) { return gf[k]; }, s, dp);
    Frag8<T> kt[2][C::DT];
#pragma unroll
    for (int dt = 0; dt < C::DT; dt++) kt[0][dt] = F.cols(ks, 32 * u, dt);
    READS_FIRST;
    mma_ready<T>(s, dp);
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c, -lse)) * fmaf(dp[i], a.scale, -dl);
    if (!wave.all(a, sq, k0)) mask_keys(s, row, k0, h, a.sinks, 0.f);
#pragma unroll
    for (int st = 0; st < 2; st++) {
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; i++) p[i] = s[8 * st + i];
      const Frag8<T> pf = pack8(p, T{});
      if (st == 0) {
#pragma unroll
        for (int dt = 0; dt < C::DT; dt++) kt[1][dt] = F.cols(ks, 32 * u + 16, dt);
        READS_FIRST;
      }
#pragma unroll
      for (int dt = 0; dt < C::DT; dt++) acc[dt] = mma32(kt[st][dt], pf, acc[dt]);
    }
  };

  const int gid = WIDE ? tid : lane, wave_id = WIDE ? wv : 0;
  const Copy<T, D, S::KT, S::NTH, S::DIRECT> ck(a.k.t, gid), cv(a.v.t, gid);
  stream_tiles<S>(WIDE ? 0 : wv, pl.nt,
    [&](int t, auto i) {
      const int k0 = key_of(t);
      char* at = smem + own + decltype(i)::v * 2 * S::tile;
      ck.issue(Kb, a.k.t, k0, sq.len - k0, at, wave_id); cv.issue(Vb, a.v.t, k0, sq.len - k0, at + S::tile, wave_id);
    },
    [](auto) {},
    [&](int t, auto i) {
      const int k0 = key_of(t);
      const char* at = smem + decltype(i)::v * 2 * S::tile;
#pragma unroll
      for (int u = 0; u < S::KS; u++) step(at, at + S::tile, u, k0 + 32 * u);
    });
#pragma unroll
  for (int dt = 0; dt < C::DT; dt++) mma_ready<T>(acc[dt]);
  if (WIDE) {
    const int64_t qoff = (int64_t)b * a.dq.b + (int64_t)row.i * a.dq.t + (int64_t)head * a.dq.h;
    if (row.r < a.rows) {
#pragma unroll
      for (int dt = 0; dt < C::DT; dt++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; j++) v[j] = row.live ? acc[dt][4 * q + j] : 0.f;
          st4_grad<T>(a.dq.p, qoff + 32 * dt + 8 * q + 4 * h, a.g_f32, v);
        }
    }
    return;
  }
  float* part = (float*)smem;
  __syncthreads();
#pragma unroll
  for (int dt = 0; dt < C::DT; dt++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = row.live ? acc[dt][4 * q + j] : 0.f;
      st4(part + (wv * 32 + c32) * C::CP + 32 * dt + 8 * q + 4 * h, v);
    }
  __syncthreads();
  for (int idx = tid; idx < 32 * (D / 4); idx += 256) {
    const int rr = idx / (D / 4), c4 = idx % (D / 4), r = r0 + rr;
    if (r >= a.rows) break;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const v4f x = *(const v4f*)(part + (w * 32 + rr) * C::CP + 4 * c4);
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += x[j];
    }
    const int i = r / a.group, g = r - i * a.group;
    st4_grad<T>(a.dq.p, (int64_t)b * a.dq.b + (int64_t)i * a.dq.t + (int64_t)(kvh * a.group + g) * a.dq.h + 4 * c4, a.g_f32, v);
  }
}

// ------------------------------------------------------------------------------------------------ backward: dK, dV
// tokens [lo, hi) whose queries see any key of [jlo, jhi], jhi < len
struct Span { int lo, hi; };
__device__ __forceinline__ Span tokens_of(const WinArgs& a, const Seq& s, int jlo, int jhi) {
  const int p0 = max(jlo - a.right, 0), p1 = jlo < a.sinks ? s.len - 1 : min(jhi + a.left, s.len - 1);
  const int i0 = min(max(p0 - s.start, 0), a.Nq), i1 = min(p1 - s.start, a.Nq - 1);
  return Span{i0, max(i1 + 1, i0)};
}

template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(256, (waves_kv<T, D>())) void k_win_dkv(const WinArgs a) {
  using C = Cfg<T, D>;
  using S = Shape<T, D, WIDE>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), c32 = lane & 31, h = lane >> 5;
  // the rows of the first sink_tiles tiles are dealt to nchunk blocks each, added up afterwards
  const int ktiles = (a.Nk + S::ROWS - 1) / S::ROWS, per_bh = a.sink_tiles * a.nchunk + ktiles - a.sink_tiles;
  const int flat = xcd_range(blockIdx.x, gridDim.x), bh = flat / per_bh, e = flat % per_bh, b = bh / a.kv, kvh = bh % a.kv;
  const bool shared_rows = e < a.sink_tiles * a.nchunk && a.nchunk > 1;
  const int tile = e < a.sink_tiles * a.nchunk ? e / a.nchunk : e - a.sink_tiles * (a.nchunk - 1), chunk = shared_rows ? e % a.nchunk : 0;
  const int k0 = tile * S::ROWS;
  const Seq sq = sequence(a, b);
  const int j = k0 + (WIDE ? 32 * wv : 0) + c32;
  const bool live = j < sq.len;
  const T* Qb = (const T*)a.q.p + (int64_t)b * a.q.b + (int64_t)kvh * a.group * a.q.h;
  const T* Gb = (const T*)a.go.p + (int64_t)b * a.go.b + (int64_t)kvh * a.group * a.go.h;
  const float *lseb = a.lse + (int64_t)bh * a.rows, *dlb = a.delta + (int64_t)bh * a.rows;
  const int set0 = WIDE ? 0 : wv * S::NBUF, own = set0 * 2 * S::rtile;      // the wave's tiles
  const Frags<T, D> F(lane, own), FV(lane, WIDE ? wv * 32 * C::PITCH : 0);
  Frag8<T> kf[C::KK], vf[S::VLDS ? 1 : C::KK];
  {
    const int jc = live ? j : 0;       // (a key behind the sequence: any key, its column is thrown away)
    const T* Kr = (const T*)a.k.p + (int64_t)b * a.k.b + (int64_t)jc * a.k.t + (int64_t)kvh * a.k.h;
    const T* Vr = (const T*)a.v.p + (int64_t)b * a.v.b + (int64_t)jc * a.v.t + (int64_t)kvh * a.v.h;
#pragma unroll
    for (int kk = 0; kk < C::KK; kk++) {
      kf[kk] = ldg8(Kr + 16 * kk + 8 * h);
      // (narrow: the four waves own the same keys and write the same values; a wave reads behind its own writes)
      if constexpr (S::VLDS) *(v4u*)(smem + S::vals + FV.row + FV.piece(2 * kk, FV.fx)) = ldg8(Vr + 16 * kk + 8 * h).u;
      else vf[kk] = ldg8(Vr + 16 * kk + 8 * h);
    }
  }
  v16f ak[C::DT], av[C::DT];
#pragma unroll
  for (int dt = 0; dt < C::DT; dt++) { ak[dt] = zero16(); av[dt] = zero16(); }
  const Span mine = live ? tokens_of(a, sq, j, j) : Span{0x7fffffff, 0x7fffffff};
  const Span block = k0 < sq.len ? tokens_of(a, sq, k0, min(k0 + S::ROWS, sq.len) - 1) : Span{0, 0};
  // Tokens that see all keys of the wave need no mask, tokens that see none of them no work.  The first token that sees a key moves with the
  // key; the last does too, but for the sinks, which everyone behind sees.
  const int j0 = k0 + (WIDE ? 32 * wv : 0), j1 = min(j0 + 31, sq.len - 1), jn = max(j0, a.sinks);
  int all_lo = 0, all_hi = 0, any_lo = 0, any_hi = 0;
  if (j0 <= j1) {
    const Span first = tokens_of(a, sq, j0, j0), last = tokens_of(a, sq, j1, j1);
    any_lo = first.lo; any_hi = j0 < a.sinks ? first.hi : last.hi;
    all_lo = last.lo; all_hi = j0 + 31 != j1 ? 0 : jn <= j1 ? tokens_of(a, sq, jn, jn).hi : first.hi;
  }
  // tiles of RT tokens of one query head, the heads of the group one after the other
  const int per_head = (block.hi - block.lo + S::RT - 1) / S::RT, ntile = per_head * a.group;
  const int per = shared_rows ? (ntile + a.nchunk - 1) / a.nchunk : ntile, t0 = chunk * per, t1 = min(ntile, t0 + per);

  auto step = [&](const char* qs, const char* gs, const float* sl, const float* sd, int u, int i0) __attribute__((always_inline)) {      // 32 query rows, i0 the first token
    if (i0 >= any_hi || i0 + 32 <= any_lo) return;
    v16f s = zero16(), dp = zero16();
    if constexpr (S::VLDS) two_products<T, D, 2>(F, qs, gs, 32 * u, kf, [&](int k) { return FV.rows(smem + S::vals, 0, k); }, s, dp);
    else two_products<T, D, D == 64 && sizeof(T) == 2 ? 2 : read_group<T, D>()>(F, qs, gs, 32 * u, kf, [&](int k) { return vf[k]; }, s, dp);
    // (the k-major operands are read ahead where that leaves the waves per SIMD as they are)
    constexpr int AH = C::ES == 2 && D >= 64 ? 0 : C::DT;
    Frag8<T> gt[C::DT], qt[C::DT];
#pragma unroll
    for (int dt = 0; dt < AH; dt++) { gt[dt] = F.cols(gs, 32 * u, dt); qt[dt] = F.cols(qs, 32 * u, dt); }
    READS_FIRST;
    mma_ready<T>(s, dp);
    if (!(i0 >= all_lo && i0 + 32 <= all_hi)) {
      const int off = i0 + 4 * h - mine.lo;
      const unsigned span = (unsigned)(mine.hi - mine.lo);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const bool see = (unsigned)(off + 8 * (i >> 2) + (i & 3)) < span;
        s[i] = see ? s[i] : -INFINITY; dp[i] = see ? dp[i] : 0.f;
      }
    }
#pragma unroll
    for (int st = 0; st < 2; st++) {
      v4f ls[2], dl[2];
#pragma unroll
      for (int q = 0; q < 2; q++) { ls[q] = *(const v4f*)(sl + 32 * u + 16 * st + 8 * q + 4 * h); dl[q] = *(const v4f*)(sd + 32 * u + 16 * st + 8 * q + 4 * h); }
      READS_FIRST;
      float p[8], d[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * st + i], a.c, -ls[i >> 2][i & 3]));
        d[i] = p[i] * fmaf(dp[8 * st + i], a.scale, -dl[i >> 2][i & 3]);
      }
      const Frag8<T> pf = pack8(p, T{}), df = pack8(d, T{});
      Frag8<T> gn[C::DT], qn[C::DT];
      if (st == 0) {
#pragma unroll
        for (int dt = 0; dt < AH; dt++) { gn[dt] = F.cols(gs, 32 * u + 16, dt); qn[dt] = F.cols(qs, 32 * u + 16, dt); }
        READS_FIRST;
      }
#pragma unroll
      for (int dt = 0; dt < C::DT; dt++) {
        if (!AH) { gt[dt] = F.cols(gs, 32 * u + 16 * st, dt); qt[dt] = F.cols(qs, 32 * u + 16 * st, dt); }
        av[dt] = mma32(gt[dt], pf, av[dt]);
        ak[dt] = mma32(qt[dt], df, ak[dt]);
        if (AH && st == 0) { gt[dt] = gn[dt]; qt[dt] = qn[dt]; }
      }
    }
  };

  const int gid = WIDE ? tid : lane, wave_id = WIDE ? wv : 0;
  const Copy<T, D, S::RT, S::NTH, S::DIRECT> cq(a.q.t, gid), cg(a.go.t, gid);
  float ls = 0.f, dl = 0.f;
  auto stats_of = [&](int i) { return (float*)(smem + S::rstage + (set0 + i) * 512); };
  stream_tiles<S>(WIDE ? t0 : t0 + wv, t1,
    [&](int t, auto i) {
      // rows behind the block's tokens arrive as zeros, with zeros for lse and delta: P = 1 times a zero row of dO, dS = 0
      const int g = a.group == 1 ? 0 : t / per_head, i0 = block.lo + (t - g * per_head) * S::RT, left = block.hi - i0;
      char* at = smem + own + decltype(i)::v * 2 * S::rtile;
      cq.issue(Qb + (int64_t)g * a.q.h, a.q.t, i0, left, at, wave_id); cg.issue(Gb + (int64_t)g * a.go.h, a.go.t, i0, left, at + S::rtile, wave_id);
      const bool in = gid < min(left, S::RT);
      const int64_t r = (int64_t)(i0 + (in ? gid : 0)) * a.group + g;
      ls = in ? lseb[r] : 0.f; dl = in ? dlb[r] : 0.f;
    },
    [&](auto i) { if (gid < S::RT) { float* st = stats_of(decltype(i)::v); st[gid] = ls; st[64 + gid] = dl; } },
    [&](int t, auto i) {
      const int i0 = block.lo + (a.group == 1 ? t : t % per_head) * S::RT;
      const char* at = smem + decltype(i)::v * 2 * S::rtile;
      const float* st = stats_of(decltype(i)::v);
#pragma unroll
      for (int u = 0; u < S::RS; u++) step(at, at + S::rtile, st, st + 64, u, i0 + 32 * u);
    });

#pragma unroll
  for (int dt = 0; dt < C::DT; dt++) mma_ready<T>(ak[dt], av[dt]);
  float* ws = shared_rows ? a.part + (((int64_t)bh * a.sink_tiles + tile) * a.nchunk + chunk) * (2 * S::ROWS * D) : nullptr;
  const int64_t koff = (int64_t)b * a.dk.b + (int64_t)kvh * a.dk.h, voff = (int64_t)b * a.dv.b + (int64_t)kvh * a.dv.h;
  if (WIDE) {
    if (j < a.Nk) {
#pragma unroll
      for (int dt = 0; dt < C::DT; dt++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          float x[4], y[4];
#pragma unroll
          for (int i = 0; i < 4; i++) { x[i] = live ? ak[dt][4 * q + i] : 0.f; y[i] = live ? av[dt][4 * q + i] : 0.f; }
          const int ch = 32 * dt + 8 * q + 4 * h;
          if (shared_rows) { st4(ws + (j - k0) * D + ch, x); st4(ws + (S::ROWS + j - k0) * D + ch, y); }
          else { st4_grad<T>(a.dk.p, koff + (int64_t)j * a.dk.t + ch, a.g_f32, x); st4((T*)a.dv.p + voff + (int64_t)j * a.dv.t + ch, y); }
        }
    }
    return;
  }
  float* part = (float*)smem;
#pragma unroll
  for (int pass = 0; pass < 2; pass++) {
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < C::DT; dt++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = live ? (pass ? av[dt][4 * q + i] : ak[dt][4 * q + i]) : 0.f;
        st4(part + (wv * 32 + c32) * C::CP + 32 * dt + 8 * q + 4 * h, x);
      }
    __syncthreads();
    for (int idx = tid; idx < 32 * (D / 4); idx += 256) {
      const int rr = idx / (D / 4), c4 = idx % (D / 4), key = k0 + rr;
      if (key >= a.Nk) break;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const v4f x = *(const v4f*)(part + (w * 32 + rr) * C::CP + 4 * c4);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] += x[i];
      }
      if (shared_rows) st4(ws + (pass * S::ROWS + rr) * D + 4 * c4, v);
      else if (pass) st4((T*)a.dv.p + voff + (int64_t)key * a.dv.t + 4 * c4, v);
      else st4_grad<T>(a.dk.p, koff + (int64_t)key * a.dk.t + 4 * c4, a.g_f32, v);
    }
  }
}

// dK, dV of the keys whose rows were dealt to several blocks, added in block order
template <typename T, int D>
__global__ __launch_bounds__(256) void k_win_sink_sum(const WinArgs a, int keys) {      // keys: rows of a tile
  const int nb = (2 * keys * (D / 4) + 255) / 256, bt = blockIdx.x / nb, bh = bt / a.sink_tiles, tile = bt % a.sink_tiles, b = bh / a.kv, kvh = bh % a.kv;
  const int idx = (blockIdx.x % nb) * 256 + threadIdx.x, which = idx / (keys * (D / 4)), rest = idx % (keys * (D / 4)), key = tile * keys + rest / (D / 4), ch = 4 * (rest % (D / 4));
  if (which > 1 || key >= a.Nk) return;
  const float* p = a.part + (int64_t)bt * a.nchunk * (2 * keys * D) + (int64_t)which * keys * D + (rest / (D / 4)) * D + ch;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < a.nchunk; c++) {
    const v4f x = *(const v4f*)(p + (int64_t)c * (2 * keys * D));
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] += x[i];
  }
  if (which) st4((T*)a.dv.p + (int64_t)b * a.dv.b + (int64_t)kvh * a.dv.h + (int64_t)key * a.dv.t + ch, v);
  else st4_grad<T>(a.dk.p, (int64_t)b * a.dk.b + (int64_t)kvh * a.dk.h + (int64_t)key * a.dk.t + ch, a.g_f32, v);
}

// ------------------------------------------------------------------------------------------------ host
// (`done`: a bit per device on which this kernel's limit has been raised)
int raise_lds(const void* kern, size_t smem, const char* name, std::atomic<uint64_t>& done) {
  if (smem <= 48 * 1024) return 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 64;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return 0;
  hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != hipSuccess) { (void)hipGetLastError(); DP_FAIL("%s: cannot raise dynamic LDS to %zu: %s", name, smem, hipGetErrorString(e)); }
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return 0;
}

// Which kernel, how many blocks: decided by sizes alone.
// Wide where it gives every CU a block, narrow below (bf16, window 256 + 256, two sequences; forward / dQ / dK, dV in us, wide against narrow):
//   heads of 128:  96 wide blocks 21 / 27 / 38 against 15 / 20 / 22;  264: 27 / 37 / 51 against 34 / 43 / 51
//   heads of 64:  192: 15 / 18 / 22 against 13 / 16 / 17;  264: 16 / 19 / 23 against 17 / 23 / 26;  384: 20 / 25 / 29 against 22 / 29 / 31
//   (fp32 the two come within a twentieth of each other; heads of 32 and 96 go by the same rule, not measured on both sides.  The threshold does not
//   know how many blocks a CU holds: 4, 3 and 3 for heads of 64.)
// Few rows, many keys (fewer than 256 narrow blocks): the key tiles are shared out over about 512 blocks, each with four tiles a wave or more
// (a token of 12 heads on 4 key heads, 4 sequences of up to 32 769 keys, fp16: 22.1 + 4.3 us for the merge; over 256 blocks 22.9 + 4.0, over 1024
// 23.6 + 6.3).  Where a wave's chain is short the merge costs more than it saves, the more so the more rows there are: 2048 rows over 1024 keys
// 10.5 us, split 7.6 + 4.4; 4096 over 2048 16.4 against 10.6 + 6.7; 5000 over 2500 (heads of 128) 26.8 against 18.2 + 7.4 (the rule rests on these).
// Only the forward pass splits its keys: dQ of few queries over many keys runs on as many blocks as there are key heads and tiles of rows (the token
// above, four sequences of 32 769 keys: 16 blocks, 251 us; its dK / dV 82 us, the forward pass 21 + 5).
// Few key tiles: the rows that see one are dealt out in the same way (dK / dV of 1024 tokens, 12 heads of 64 on 4, every token before: 15.7 + 3.9
// us; one block a tile 31.9; 8 heads of 96 on 2, 1000 tokens: 19.0 + 4.0 against 49.5).
// Tiles that hold sinks: their rows are dealt to as many blocks as have the work of another tile (dK / dV of 13 825 tokens, heads of 64: 143 us;
// with one block a tile 519).
struct Launch { bool wide; int tiles, nsplit; bool kwide; int ktiles, sink_tiles, nchunk; };      // sink_tiles: key tiles whose rows are dealt out
Launch plan(int B, int kv, int group, int Nq, int Nk, int d, int left, int right, int sinks) {
  Launch p;
  const int64_t rows = Nq > 0 ? (int64_t)Nq * group : 1, bk = (int64_t)B * kv;
  p.wide = (rows + 127) / 128 * bk >= 256;
  p.tiles = (int)((rows + (p.wide ? 127 : 31)) / (p.wide ? 128 : 32));
  p.nsplit = 1;
  const int64_t span = left >= FAR || right >= FAR ? Nk : (int64_t)left + right + sinks + 32;
  const int64_t rounds = ((span < Nk ? span : Nk) + 127) / 128;      // 32-key tiles for each of the four waves
  if (!p.wide && p.tiles * bk < 256 && rounds >= 16 + rows * bk / 512) {
    int64_t n = 512 / (p.tiles * bk);
    if (n > rounds / 4) n = rounds / 4;
    p.nsplit = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
  }
  p.kwide = (int64_t)(Nk + 127) / 128 * bk >= 256;
  const int kb = p.kwide ? 128 : 32;
  p.ktiles = (Nk + kb - 1) / kb;
  p.sink_tiles = 0; p.nchunk = 1;
  if (Nk < 1) return p;
  const int64_t usual = left >= FAR || right >= FAR ? rows : ((int64_t)left + right + kb) * group;      // rows of a tile without sinks
  const int64_t seen = usual < rows ? usual : rows, tall = sinks > 0 && left < FAR ? rows / (usual < 128 ? 128 : usual) : 1, blocks = p.ktiles * bk;
  int64_t n = blocks < 256 ? 512 / blocks : 1;
  if (n > seen / 512) n = seen / 512;      // (four tiles of 32 rows for each of a block's four waves)
  int64_t st = p.ktiles;
  if (n > 1) { if (n < tall) n = tall < 8 ? tall : 8 > n ? 8 : n; }
  else { n = tall; st = ((sinks < Nk ? sinks : Nk) + kb - 1) / kb; }
  const int64_t most = (64ll << 20) / (bk * (st < 1 ? 1 : st) * 2 * kb * d);      // (256 MB of partial sums at most)
  if (n > most) n = most;
  p.nchunk = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
  if (p.nchunk > 1) p.sink_tiles = (int)st;
  return p;
}

int check(const char* name, int B, int heads, int kv, int Nq, int Nk, int d, int left, int right, int sinks, float scale, int dtype) {
  if (dtype != DP_F32 && dtype != DP_BF16 && dtype != DP_F16) DP_FAIL("%s: bad dtype %d", name, dtype);
  if (d != 32 && d != 64 && d != 96 && d != 128) DP_FAIL("%s: head dim %d not in {32, 64, 96, 128}", name, d);
  if (B < 0 || heads < 1 || kv < 1 || heads % kv || Nq < 0 || Nk < 0) DP_FAIL("%s: bad sizes B=%d heads=%d/%d Nq=%d Nk=%d", name, B, heads, kv, Nq, Nk);
  if (left < -1 || right < -1 || sinks < 0) DP_FAIL("%s: bad window left=%d right=%d sinks=%d", name, left, right, sinks);
  if (!(scale > 0.f) || !(scale < 1e30f)) DP_FAIL("%s: scale %g", name, (double)scale);
  if (Nk >= FAR / 2 || (int64_t)Nq * (heads / kv) >= FAR / 2 || (int64_t)B * kv * ((Nk > Nq * (int64_t)(heads / kv) ? Nk : Nq * (int64_t)(heads / kv)) / 32 + 64) >= FAR)
    DP_FAIL("%s: too many rows", name);
  return 0;
}
// n > 0: a matrix of n tokens that is copied to LDS by 32-bit offsets from its tile's first row
int check_mat(const char* name, const char* what, Mat& m, int es, int n = 0, int d = 0) {
  if (((uintptr_t)m.p & 15) || (m.b * es) % 16 || (m.t * es) % 16 || (m.h * es) % 16) DP_FAIL("%s: %s: rows must be 16-byte aligned", name, what);
  if (n > 1 && (m.t < d || m.t * es > (1 << 24))) DP_FAIL("%s: %s: token stride %lld (at least the head dim, at most 16 MB)", name, what, (long long)m.t);
  if (n == 1) m.t = d;
  return 0;
}

template <typename T, int D, bool WIDE> int run_fwd(const WinArgs& a, int B, hipStream_t st) {
  auto kern = k_win_fwd<T, D, WIDE>;
  constexpr size_t smem = Shape<T, D, WIDE>::fwd;
  static_assert(smem <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> done{0};
  if (raise_lds((const void*)kern, smem, "window_attention_fwd", done)) return 1;
  hipLaunchKernelGGL(kern, dim3(a.tiles * a.nsplit * B * a.kv), dim3(256), smem, st, a);
  DP_CHECK_LAUNCH("window_attention_fwd");
  if (a.nsplit > 1) {
    hipLaunchKernelGGL((k_win_merge<T, D>), dim3(a.rows, B * a.kv), dim3(256), 0, st, a);
    DP_CHECK_LAUNCH("window_attention_fwd(merge)");
  }
  return 0;
}
template <typename T, int D, bool WIDE> int run_dq(const WinArgs& a, int B, hipStream_t st) {
  auto kern = k_win_dq<T, D, WIDE>;
  constexpr size_t smem = Shape<T, D, WIDE>::big;
  static std::atomic<uint64_t> done{0};
  if (raise_lds((const void*)kern, smem, "window_attention_bwd", done)) return 1;
  hipLaunchKernelGGL(kern, dim3(a.tiles * B * a.kv), dim3(256), smem, st, a);
  DP_CHECK_LAUNCH("window_attention_bwd(dq)");
  return 0;
}
template <typename T, int D, bool WIDE> int run_dkv(const WinArgs& a, int B, int ktiles, hipStream_t st) {
  auto kern = k_win_dkv<T, D, WIDE>;
  constexpr size_t smem = Shape<T, D, WIDE>::kvb;
  static_assert(smem <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> done{0};
  if (raise_lds((const void*)kern, smem, "window_attention_bwd", done)) return 1;
  hipLaunchKernelGGL(kern, dim3((a.sink_tiles * (a.nchunk - 1) + ktiles) * B * a.kv), dim3(256), smem, st, a);
  DP_CHECK_LAUNCH("window_attention_bwd(dkv)");
  if (a.sink_tiles) {
    constexpr int keys = Shape<T, D, WIDE>::ROWS;
    hipLaunchKernelGGL((k_win_sink_sum<T, D>), dim3(cdiv(2 * keys * (D / 4), 256) * a.sink_tiles * B * a.kv), dim3(256), 0, st, a, keys);
    DP_CHECK_LAUNCH("window_attention_bwd(sinks)");
  }
  return 0;
}

}  // namespace

#define WIN_DIMS(d, ...) do { if ((d) == 32) { constexpr int D = 32; __VA_ARGS__; } else if ((d) == 64) { constexpr int D = 64; __VA_ARGS__; } \
    else if ((d) == 96) { constexpr int D = 96; __VA_ARGS__; } else { constexpr int D = 128; __VA_ARGS__; } } while (0)

extern "C" int64_t dp_window_attention_ws_elems(int B, int heads, int kv_heads, int Nq, int Nk, int d, int left, int right, int sinks, int backward) {
  if (B < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || Nq < 1 || Nk < 1 || left < -1 || right < -1 || sinks < 0) return 0;
  const int group = heads / kv_heads;
  const Launch p = plan(B, kv_heads, group, Nq, Nk, d, left < 0 ? FAR : left, right < 0 ? FAR : right, sinks);
  const int64_t bk = (int64_t)B * kv_heads;
  if (!backward) return p.nsplit > 1 ? bk * p.nsplit * Nq * group * (d + 4) : 0;
  return bk * p.sink_tiles * p.nchunk * 2 * (p.kwide ? 128 : 32) * d;
}

extern "C" int dp_window_attention_fwd(const void* q, int64_t qb, int64_t qt, int64_t qh, const void* k, int64_t kb, int64_t kt, int64_t kh, const void* v,
                                       int64_t vb, int64_t vt, int64_t vh, void* o, int64_t ob, int64_t ot, int64_t oh, float* lse, float* ws, int B,
                                       int heads, int kv_heads, int Nq, int Nk, int d, int left, int right, int sinks, int q_start, const int32_t* q_starts,
                                       const int32_t* lengths, float scale, int dtype, void* stream) {
  if (check("window_attention_fwd", B, heads, kv_heads, Nq, Nk, d, left, right, sinks, scale, dtype)) return 1;
  WinArgs a{};
  a.q = Mat{(void*)q, qb, qt, qh}; a.k = Mat{(void*)k, kb, kt, kh}; a.v = Mat{(void*)v, vb, vt, vh}; a.o = Mat{o, ob, ot, oh};
  const int es = dtype == DP_F32 ? 4 : 2;
  if (check_mat("window_attention_fwd", "q", a.q, es, B > 0 ? Nq : 0, d) || check_mat("window_attention_fwd", "k", a.k, es, B > 0 ? Nk : 0, d) || check_mat("window_attention_fwd", "v", a.v, es, B > 0 ? Nk : 0, d) ||
      check_mat("window_attention_fwd", "o", a.o, es)) return 1;
  if (B == 0 || Nq == 0) return 0;
  if (!q || !o || (Nk > 0 && (!k || !v))) DP_FAIL("window_attention_fwd: q, k, v or o missing");
  a.lse = lse; a.part = ws; a.starts = q_starts; a.lens = lengths;
  a.kv = kv_heads; a.group = heads / kv_heads; a.Nq = Nq; a.Nk = Nk; a.rows = Nq * a.group;
  a.left = left < 0 ? FAR : left < FAR ? left : FAR; a.right = right < 0 ? FAR : right < FAR ? right : FAR; a.sinks = sinks < FAR ? sinks : FAR;
  a.start = q_start < -FAR ? -FAR : q_start > FAR ? FAR : q_start;
  a.scale = scale; a.c = scale * LOG2E; a.lag = LAG / a.c;
  const Launch p = plan(B, kv_heads, a.group, Nq, Nk, d, a.left, a.right, a.sinks);
  a.tiles = p.tiles; a.nsplit = p.nsplit; a.nchunk = 1;
  if (p.nsplit > 1 && (!ws || ((uintptr_t)ws & 15))) DP_FAIL("window_attention_fwd: needs a 16-byte aligned workspace (dp_window_attention_ws_elems)");
  DP_DISPATCH(dtype, WIN_DIMS(d, return p.wide ? run_fwd<T, D, true>(a, B, STREAM) : run_fwd<T, D, false>(a, B, STREAM)));
  return 0;
}

extern "C" int dp_window_attention_bwd(const void* q, int64_t qb, int64_t qt, int64_t qh, const void* k, int64_t kb, int64_t kt, int64_t kh, const void* v,
                                       int64_t vb, int64_t vt, int64_t vh, const void* o, int64_t ob, int64_t ot, int64_t oh, const void* go, int64_t gb,
                                       int64_t gt, int64_t gh, const float* lse, float* delta, void* dq, int64_t dqb, int64_t dqt, int64_t dqh, void* dk,
                                       int64_t dkb, int64_t dkt, int64_t dkh, void* dv, int64_t dvb, int64_t dvt, int64_t dvh, int qk_f32, float* ws, int B,
                                       int heads, int kv_heads, int Nq, int Nk, int d, int left, int right, int sinks, int q_start, const int32_t* q_starts,
                                       const int32_t* lengths, float scale, int dtype, void* stream) {
  const char* name = "window_attention_bwd";
  if (check(name, B, heads, kv_heads, Nq, Nk, d, left, right, sinks, scale, dtype)) return 1;
  WinArgs a{};
  a.q = Mat{(void*)q, qb, qt, qh}; a.k = Mat{(void*)k, kb, kt, kh}; a.v = Mat{(void*)v, vb, vt, vh}; a.o = Mat{(void*)o, ob, ot, oh};
  a.go = Mat{(void*)go, gb, gt, gh}; a.dq = Mat{dq, dqb, dqt, dqh}; a.dk = Mat{dk, dkb, dkt, dkh}; a.dv = Mat{dv, dvb, dvt, dvh};
  const int es = dtype == DP_F32 ? 4 : 2, gs = qk_f32 ? 4 : es;
  if (check_mat(name, "q", a.q, es, B > 0 ? Nq : 0, d) || check_mat(name, "k", a.k, es, B > 0 ? Nk : 0, d) || check_mat(name, "v", a.v, es, B > 0 ? Nk : 0, d) || check_mat(name, "o", a.o, es) ||
      check_mat(name, "go", a.go, es, B > 0 ? Nq : 0, d) || check_mat(name, "dq", a.dq, gs) || check_mat(name, "dk", a.dk, gs) || check_mat(name, "dv", a.dv, es)) return 1;
  if (B == 0) return 0;
  if (Nq > 0 && (!q || !o || !go || !lse || !delta || !dq)) DP_FAIL("%s: q, o, go, lse, delta or dq missing", name);
  if (Nk > 0 && (!k || !v || !dk || !dv)) DP_FAIL("%s: k, v, dk or dv missing", name);
  a.lse = (float*)lse; a.delta = delta; a.part = ws; a.starts = q_starts; a.lens = lengths;
  a.kv = kv_heads; a.group = heads / kv_heads; a.Nq = Nq; a.Nk = Nk; a.rows = Nq * a.group;
  a.left = left < 0 ? FAR : left < FAR ? left : FAR; a.right = right < 0 ? FAR : right < FAR ? right : FAR; a.sinks = sinks < FAR ? sinks : FAR;
  a.start = q_start < -FAR ? -FAR : q_start > FAR ? FAR : q_start;
  a.scale = scale; a.c = scale * LOG2E; a.g_f32 = qk_f32 != 0;
  const Launch p = plan(B, kv_heads, a.group, Nq, Nk, d, a.left, a.right, a.sinks);
  a.tiles = p.tiles; a.nsplit = 1; a.sink_tiles = p.sink_tiles; a.nchunk = p.nchunk;
  if (p.sink_tiles && (!ws || ((uintptr_t)ws & 15))) DP_FAIL("%s: needs a 16-byte aligned workspace (dp_window_attention_ws_elems)", name);
  if (Nq > 0) {
    int rc = 0;
    DP_DISPATCH(dtype, WIN_DIMS(d, rc = p.wide ? run_dq<T, D, true>(a, B, STREAM) : run_dq<T, D, false>(a, B, STREAM)));
    if (rc) return rc;
  }
  if (Nk == 0) return 0;
  DP_DISPATCH(dtype, WIN_DIMS(d, return p.kwide ? run_dkv<T, D, true>(a, B, p.ktiles, STREAM) : run_dkv<T, D, false>(a, B, p.ktiles, STREAM)));
  return 0;
}
