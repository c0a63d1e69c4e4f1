// Self-attention with document masks, causal and prefix masks, capped scores
// and linear distance biases, for any length; forward and backward, bf16 or
// fp16 operands, head sizes up to 128, shared key heads.
//
//   z_ij = scale q_i.k_j;  z = cap tanh(z / cap);  z -= slope_h |i - j|
//   (i, j) attended:  doc_i == doc_j >= 0  and  (not causal or j <= i or
//                     j < prefix)
//   p = softmax of z over the attended j (all 0 if there is none),  o = p v
//   D_i = go_i.o_i;  dp = go v^T;  dz = p (dp - D) (1 - tanh^2)
//   dq = scale dz k,  dk = scale dz^T q,  dv = p^T go
//
// All three kernels have one shape.  A wave owns 32 tokens (queries in the
// forward and dq kernels, keys in the dk/dv kernel) whose operands stay in
// registers, and tiles of 64 tokens of the other side stream through LDS,
// double-buffered: the next tile's loads are issued before a tile is worked on
// and land in the other buffer after it.  A workgroup's four waves own 128
// tokens (KS = 1), or 64 with two waves on each 32, one for either half of
// every tile, joined through LDS at the end (KS = 2; KS = 8: eight waves own
// 128 like that).  Products are 32x32x16 MFMAs with the streamed side as the
// left operand, so that a lane's column of the result belongs to one owned
// token and its 16 registers to streamed tokens: the softmax is a reduction
// over registers plus one exchange between the wave's halves, and the rounded
// probabilities already lie as the right operand of the second product.  That
// operand's k order is
//     slot 8h + j  <->  token 4h + (j & 3) + 8 (j >> 2)       (h: lane / 32)
// instead of the plain one; the left operand, read transposed from the same LDS
// tile (ds_read_b64_tr_b16: four tokens of 16 columns a lane group), uses the
// same order, so nothing moves between lanes.
//
// In fp16 the backward rounds 2^15 p instead of p (the factor leaves dv again
// in fp32): a uniform row of 16K tokens has p = 2^-14, below which fp16 loses a
// bit for every halving.  dz is as small as the gradients are and has no bound
// above: every owned token has a power of two for it that falls as its largest
// dz so far asks for (`Lift`), and leaves its sum at the end.  11 x 3913
// tokens, go around 0.02: relative error of dq and dk 0.00030, and 0.00042
// without.  2 x 1999 tokens, 16 heads of size 128: dq 137 us, 129 without;
// dk/dv 2 % more.
//
// dz is a small difference where few tokens share a row, and an error of D is
// one of the whole row.  Taken from the rounded o it would be as large as dz's
// own rounding, so the forward keeps what rounding took from o (in 16 bits).
// That leaves the rounding of p in o, which matters where a handful of tokens
// are all: sequences of up to 64 get D as the sum of p dp, in fp32, in a pass
// of its own.  Relative error of dq, bf16: 6 causal tokens 0.0032 from the
// rounded o, 0.0025 with the rest, 0.0023 from the sum; documents of 150
// 0.0026, 0.0024.  0.0017 is the rounding of the result alone.  The rest costs
// 3 + 3 us of 176 where bytes count most (32 x 512 tokens, 12 heads, 64); the
// sum 23 of 290 for 512 x 64 (kept in registers over a barrier instead of
// computed ahead: 9 more); in every tile it would be 4 of 176, for nothing that
// shows.
//
// What bounds them: vector operations in the forward (a score costs an
// exponential, at a quarter of the rate, and four more), registers in the
// backward, where two to three waves a SIMD cover little of each other's
// latency.  Without masks, forward / dq / dk/dv in TFLOP/s (4, 6 and 8 D
// operations a pair): 32 x 512 tokens, 12 heads of 64, 540 / 630 / 675; 2 x
// 8192 825 / 985 / 951; 8 x 2048, 16 heads of 128, 820 / 980 / 811.
//
// Scores are held in base 2 (scale * log2 e folded in) and every statistic in
// fp32.  Probabilities and dz are rounded to the operands' type for the second
// products; the sums in the denominator are of the unrounded ones.
//
// The mask is summarised per 32 tokens (smallest and largest document, any
// padding).  A workgroup first lists the tiles that it has to visit, with a
// mark for every 32 x 32 pairs: none attended (the wave skips them), all (no
// test in the loop) or some; tiles between documents that do not meet cost
// nothing.  Rows of padding are staged as zeros and rows of padding are written
// as zeros, so that whatever a padded token holds reaches no result.
//
// The backward recomputes p from the saved row statistic, in two kernels
// without atomics (dq with D, then dk/dv): 7 products instead of the 5 of a
// single kernel whose dq would be summed by atomics in an order that changes
// from run to run.
#pragma once

#include <type_traits>

#include "elem.h"
#include "encoder_api.h"

namespace colearn {

namespace masked_attn {

constexpr int kTile = kAttnTile;   // streamed tokens a tile
constexpr int kList = 1024;        // tiles listed at a time
constexpr int kShort = kAttnShort;  // tokens summarised by the workgroup itself
constexpr unsigned kZeros = 1u << 16;  // a list entry's mark
constexpr float kLog2e = 1.4426950408889634f;

// What happens to a score before the exponential, besides its scale
enum Mode : int { kPlain = 0, kBias = 1, kCap = 2 };  // kCap: bias too, if any

typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;

template <typename T>
DEV_INLINE f32x16 mfma(s16x8 a, s16x8 b, f32x16 c);
template <>
DEV_INLINE f32x16 mfma<bf16>(s16x8 a, s16x8 b, f32x16 c) {
  typedef __attribute__((ext_vector_type(8))) __bf16 V;
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
}
template <>
DEV_INLINE f32x16 mfma<f16>(s16x8 a, s16x8 b, f32x16 c) {
  typedef __attribute__((ext_vector_type(8))) _Float16 V;
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(
      __builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
}

// registers 8k .. 8k+7 of a result, rounded to T
template <typename T>
DEV_INLINE s16x8 round8(const f32x16& x, int k) {
  typedef __attribute__((ext_vector_type(8))) typename Bits16<T>::hw V;
  f32x8 f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = x[8 * k + j];
  return __builtin_bit_cast(s16x8, __builtin_convertvector(f, V));
}

// log2 of what a probability is multiplied with before dv's product rounds it
template <typename T>
constexpr float kLift = std::is_same<T, f16>::value ? 15.f : 0.f;

// The power of two that an owned token's dz is rounded with, in its sum.  Only
// fp16 has one: bf16 reaches as far down as fp32.
template <typename T>
struct Lift {
  DEV_INLINE float log2() const { return 0.f; }
  template <int N>
  DEV_INLINE void fit(f32x16&, f32x16 (&)[N]) {}
  template <int N>
  DEV_INLINE void leave(f32x16 (&)[N]) const {}
};
template <>
struct Lift<f16> {
  static constexpr int kHigh = 14, kGood = 6;
  float k = 60.f;  // the first dz other than 0 lowers it

  DEV_INLINE float log2() const { return k; }
  // x: lifted, and in range after this
  template <int N>
  DEV_INLINE void fit(f32x16& x, f32x16 (&acc)[N]) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(x[r]));
    if (!__any(m > static_cast<float>(1 << kHigh))) return;
    m = fmaxf(m, swap32(m));  // both halves hold sums of the token
    if (!(m > static_cast<float>(1 << kHigh)) || m == INFINITY) return;
    const int drop = __builtin_amdgcn_frexp_expf(m) - kGood;
    const float f = __builtin_amdgcn_ldexpf(1.f, -drop);
    k -= static_cast<float>(drop);
    x *= f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= f;
  }
  template <int N>
  DEV_INLINE void leave(f32x16 (&acc)[N]) const {
    const float f = __builtin_amdgcn_ldexpf(1.f, static_cast<int>(-k));
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= f;
  }
};

DEV_INLINE float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh from one exponential and one reciprocal; off by about 1e-7 whatever x is
DEV_INLINE float fast_tanh(float x) {
  const float e = fast_exp2(x * (2.f * kLog2e));
  return 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
}
// tanh off by about 4e-7 of itself: below 1/4 its series, whose first term left
// out is 1e-8 of x there
DEV_INLINE float near_tanh(float x) {
  const float t = x * x;
  float s = __builtin_fmaf(t, 62.f / 2835.f, -17.f / 315.f);
  s = __builtin_fmaf(t, s, 2.f / 15.f);
  s = __builtin_fmaf(t, s, -1.f / 3.f);
  return fabsf(x) < 0.25f ? __builtin_fmaf(x * t, s, x) : fast_tanh(x);
}
// The cap multiplies the error of tanh: a probability is off by 1e-7 of the cap
// with fast_tanh, 6e-6 here, a hundredth of fp16's half step and the size of
// the error that a score of 50 has in fp32 itself.  Larger caps take near_tanh,
// with which scores far below the cap keep their digits.  2 x 1999 tokens, 16
// heads of size 128, forward / dq / dk/dv: 109 / 144 / 205 us with fast_tanh,
// 121 / 155 / 206 with near_tanh.
constexpr float kFastCap = 64.f;

// the other half's value (lane ^ 32)
DEV_INLINE float other_half(float x) { return swap32(x); }

// A tile of kTile rows of DP 16-bit values.  16-byte slots are permuted
// within a row so that neither read below hits a bank twice in 256 bytes: 16
// consecutive rows of one slot (row operand) lie over all of them, and so do
// four consecutive rows of four neighbouring slots (transposed operand, 32
// lanes).
template <int DP>
struct Tile {
  static constexpr int kSlots = DP / 8;
  static constexpr int kBytes = kTile * DP * 2;

  DEV_INLINE static int at(int row, int slot) {
    const int f = DP == 32   ? (row >> 2) & 3
                  : DP == 64 ? (((row & 3) << 1) | ((row >> 2) & 1)) ^
                                   (((row >> 3) & 1) << 1)
                             : ((row & 3) << 2) | ((row >> 2) & 3);
    return row * (DP * 2) + ((slot ^ f) << 4);
  }

  // left operand: rows 0..31 of `half` (32 rows), columns 16 kk + 0..15
  DEV_INLINE static s16x8 rows(const char* half, int kk) {
    const int lane = threadIdx.x % kWave;
    return *reinterpret_cast<const s16x8*>(
        half + at(lane & 31, kk * 2 + (lane >> 5)));
  }
  // transposed left operand: columns 32 db + 0..31 as rows, tokens 16 ks +
  // 0..15 of `half` in the order of the file's head
  DEV_INLINE static s16x8 cols(const char* half, int ks, int db) {
    const int lane = threadIdx.x % kWave;
    const int i = lane & 15;
    const int row = ((lane >> 5) << 2) + (i >> 2);
    const int slot = db * 4 + ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
    const char* p = half + (i & 1) * 8 + ks * (16 * DP * 2);
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(p + at(row, slot)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(p + at(row + 8, slot)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// One streamed operand [S, D] on its way into LDS, by W waves.  Each of a tile's
// kPer passes moves 16 bytes a thread.  A row's offset in a tile is 32 bits of
// bytes (the host sees to it), the tile's own 64.
template <int DP, int W = 4>
struct Stream {
  using L = Tile<DP>;
  static constexpr int kStep = W * kWave / L::kSlots;  // rows a pass
  static constexpr int kPer = kTile / kStep;           // passes
  const short* base;
  int64_t ss;

  DEV_INLINE Stream(const short* p, int64_t stride) : base(p), ss(stride) {}

  // A tile of which every row is there and none is padding, and D == DP:
  // straight from memory into LDS, no registers on the way.  A wave's 16 bytes
  // a lane land side by side, so the permutation of slots is in what a lane
  // fetches.  In assembly, which the compiler does not look into: it takes a
  // load into LDS for a write that every later read of LDS may depend on, and
  // would wait for the next tile in the middle of this one.  What has to wait
  // is `arrived`, before the barrier that hands the tile over.
  DEV_INLINE void send(char* lds, int t0) const {
    const int row = threadIdx.x / L::kSlots, slot = threadIdx.x % L::kSlots;
    const unsigned step = static_cast<unsigned>(2 * ss);
    // the permutation goes by the row's lowest four bits, which all passes
    // share: kStep is a multiple of 16
    const unsigned off = row * step + (L::at(row, slot) - row * (DP * 2));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const char* p = reinterpret_cast<const char*>(base + t0 * ss);
    const unsigned to = __builtin_amdgcn_readfirstlane(
        static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_void*)lds)) +
        wave * 1024);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      asm volatile(
          "s_mov_b32 m0, %0\n\t"
          "s_nop 0\n\t"
          "global_load_lds_dwordx4 %1, %2"
          :
          : "s"(to + i * (W * 1024)), "v"(off), "s"(p + i * kStep * step)
          : "memory", "m0");
  }
  // Any tile: rows that `live` has no bit of, and columns past D, as zeros.
  DEV_INLINE void copy(char* lds, int t0, int S, int D,
                       unsigned long long live) const {
    const int row0 = threadIdx.x / L::kSlots, slot = threadIdx.x % L::kSlots;
    const unsigned step = static_cast<unsigned>(2 * ss);
    const char* p = reinterpret_cast<const char*>(base + t0 * ss);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int row = row0 + i * kStep;
      s16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
      if (slot * 8 < D && ((live >> row) & 1))
        x = *reinterpret_cast<const s16x8*>(p + row * step + slot * 16);
      *reinterpret_cast<s16x8*>(lds + L::at(row, slot)) = x;
    }
  }
};

// Everything that this wave has sent is in LDS.
DEV_INLINE void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The streamed tokens' documents: every wave's lanes hold those of the tile's
// 64 tokens.
struct Docs {
  const int* doc;  // of this sequence, or null
  int tok = 0;

  DEV_INLINE Docs(const MaskedAttn& a, int n)
      : doc(a.doc != nullptr ? a.doc + static_cast<int64_t>(n) * a.S
                             : nullptr) {}
  DEV_INLINE void load(int t0, int S) {
    if (doc != nullptr)
      tok = doc[min(t0 + static_cast<int>(threadIdx.x) % kTile, S - 1)];
  }
  // -1 for padding and past the end, 0 without documents
  DEV_INLINE int own(int t0, int S) const {
    return t0 + static_cast<int>(threadIdx.x) % kTile < S ? max(tok, -1) : -1;
  }
  // a bit for every token of the tile that is neither
  DEV_INLINE unsigned long long live(int t0, int S) const {
    return __ballot(own(t0, S) >= 0);
  }
};

// right operand of an owned token's row: columns 16 kk + 8 h + 0..7.  The load
// does not wait to know whether the token is there or padding (`row` is one
// that can be read); `clear` makes zeros of those and of columns past D.
template <int DP>
DEV_INLINE void own_rows(const short* row, int D, s16x8 (&r)[DP / 16]) {
  const int h = (threadIdx.x % kWave) >> 5;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk)
    r[kk] =
        *reinterpret_cast<const s16x8*>(row + min(kk * 16 + h * 8, D - 8));
}
template <int DP>
DEV_INLINE void clear(bool live, int D, s16x8 (&r)[DP / 16]) {
  const int h = (threadIdx.x % kWave) >> 5;
  if (D == DP && __all(live)) return;
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const s16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    if (!live || kk * 16 + h * 8 >= D) r[kk] = zero;
  }
}

// The operand is in its registers from here on.  Before a loop: loads that may
// still be under way when it begins would be waited for, with everything sent
// since, in each of its rounds.
template <int N>
DEV_INLINE void settle(s16x8 (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(r[i]));
}

// A transposed result: this lane's token has columns 32 db + (r & 3) +
// 8 (r >> 2) + 4 h, times f, or zeros.
template <int DP>
DEV_INLINE void put_cols(float* row, const f32x16 (&acc)[DP / 32], float f,
                         bool live, int D) {
  const int h = (threadIdx.x % kWave) >> 5;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = db * 32 + g * 8 + h * 4;
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = live ? acc[db][g * 4 + j] * f : 0.f;
      if (col < D) elem_store4(row + col, x);
    }
}
// The same for a wave's 32 tokens from `first` on, rounded to T, by way of LDS:
// a lane's own stores would be 8 bytes each, a row apart; these are whole rows,
// 16 bytes a lane.  lds: 64 DP bytes that nobody but this wave touches.
template <typename T, int DP>
DEV_INLINE void store_cols(char* lds, T* base, int64_t ss, int first, int S,
                           const f32x16 (&acc)[DP / 32], float f, bool live,
                           int D) {
  using L = Tile<DP>;
  const int lane = threadIdx.x % kWave, h = lane >> 5;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = live ? acc[db][g * 4 + j] * f : 0.f;
      elem_store4(reinterpret_cast<T*>(lds + L::at(lane & 31, db * 4 + g) +
                                       h * 8),
                  x);
    }
  const int slot = lane % L::kSlots;
#pragma unroll
  for (int i = 0; i < L::kSlots / 2; ++i) {
    const int row = i * (kWave / L::kSlots) + lane / L::kSlots;
    const s16x8 x =
        *reinterpret_cast<const s16x8*>(lds + L::at(row, slot));
    if (first + row < S && slot * 8 < D)
      *reinterpret_cast<s16x8*>(reinterpret_cast<short*>(base) +
                                (first + row) * ss + slot * 8) = x;
  }
}

// What the pairs of tokens [q0, q1) x [k0, k1) are: 0 none attended, 1 some,
// 2 all.  Keys past S count as not attended; queries past S are never written,
// or have a statistic of +inf.
DEV_INLINE int meet(bool causal, int prefix, int S, int q0, int q1, int k0,
                    int k1, bool doc, int4 a, int4 b) {
  if (k0 >= S || q0 >= S) return 0;
  int c = k1 > S ? 1 : 2;
  const int qe = min(q1, S) - 1, ke = min(k1, S) - 1;
  if (causal) {
    if (k0 > qe && k0 >= prefix) return 0;
    if (!(ke <= q0 || ke < prefix)) c = 1;
  }
  if (doc) {
    if (a.x > b.y || b.x > a.y) return 0;
    if (a.x != a.y || b.x != b.y || a.z || b.z) c = 1;
  }
  return c;
}

// Summary of 32 tokens' documents (of the 32 lanes around this one): smallest,
// largest, whether there is padding; (INT_MAX, -1) if there is nothing else.
DEV_INLINE int4 summarise(int d, bool there) {
  const bool real = there && d >= 0;
  int lo = real ? d : 0x7fffffff, hi = real ? d : -1;
  int pad = there && d < 0;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    lo = min(lo, __shfl_xor(lo, off));
    hi = max(hi, __shfl_xor(hi, off));
    pad |= __shfl_xor(pad, off);
  }
  return make_int4(lo, hi, pad, 0);
}

// The summary of a sequence: made before (a.tiles), or here in LDS for up to
// kShort tokens, where a launch of its own would cost more.
DEV_INLINE const int4* summary_of(const MaskedAttn& a, int n, int4* lds) {
  if (a.doc == nullptr) return nullptr;
  const int groups = (a.S + 31) / 32;
  if (a.tiles != nullptr) return a.tiles + static_cast<int64_t>(n) * groups;
  const int* doc = a.doc + static_cast<int64_t>(n) * a.S;
  for (int t0 = 0; t0 < a.S; t0 += static_cast<int>(blockDim.x)) {
    const int t = t0 + threadIdx.x;
    const int4 s = summarise(doc[min(t, a.S - 1)], t < a.S);
    if (threadIdx.x % 32 == 0 && t < a.S) lds[t / 32] = s;
  }
  return lds;  // list_tiles begins with a barrier
}

// Lists the tiles of [base, base + kList) that meet the owned tokens from own0
// on, in order: (tile - base) << 17; kZeros if rows of the tile have to be
// staged as zeros (padding, or none there); and two bits (`meet`) for every
// 32 owned tokens g and either half of the tile: bits 4 g + 2 half.  Called by
// the whole workgroup.
template <bool OWN_Q, int GROUPS>
DEV_INLINE int list_tiles(const MaskedAttn& a, int n, int own0, int base,
                          const int4* sum, unsigned* list, int* count) {
  const int tiles = (a.S + kTile - 1) / kTile;
  __syncthreads();  // the summary is there, the previous list used up
  if (threadIdx.x < kWave) {
    const int lane = threadIdx.x;
    const int prefix = a.prefix != nullptr ? a.prefix[n] : 0;
    const int last = (a.S + 31) / 32 - 1;
    const bool docs = sum != nullptr;
    int4 mine[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
      mine[g] = docs ? sum[min(own0 / 32 + g, last)] : make_int4(0, 0, 0, 0);
    int found = 0;
    const int end = min(base + kList, tiles);
    for (int t0 = base; t0 < end; t0 += kWave) {
      const int t = t0 + lane;
      unsigned c = 0;
      int pad = 0;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int4 other =
            docs ? sum[min(t * 2 + hf, last)] : make_int4(0, 0, 0, 0);
        const int s0 = t * kTile + hf * 32;
        pad |= other.z;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const int o0 = own0 + g * 32;
          const int x =
              OWN_Q ? meet(a.causal, prefix, a.S, o0, o0 + 32, s0, s0 + 32,
                           docs, mine[g], other)
                    : meet(a.causal, prefix, a.S, s0, s0 + 32, o0, o0 + 32,
                           docs, mine[g], other);
          c |= x << (4 * g + 2 * hf);
        }
      }
      if (t >= end) c = 0;
      const unsigned long long hit = __ballot(c != 0);
      if (c != 0)
        list[found + __popcll(hit & ((1ull << lane) - 1))] =
            (static_cast<unsigned>(t - base) << 17) | c |
            (pad != 0 || (t + 1) * kTile > a.S ? kZeros : 0);
      found += __popcll(hit);
    }
    if (lane == 0) *count = found;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*count);
}

DEV_INLINE unsigned entry_of(const unsigned* list, int e, int count) {
  return __builtin_amdgcn_readfirstlane(list[min(e, count - 1)]);
}
DEV_INLINE int first_of(unsigned entry, int base) {
  return (base + static_cast<int>(entry >> 17)) * kTile;
}

// document of an owned token: -1 for padding and past the end, 0 without
// documents
DEV_INLINE int doc_of(const MaskedAttn& a, int n, int tok) {
  if (tok >= a.S) return -1;
  if (a.doc == nullptr) return 0;
  return max(a.doc[static_cast<int64_t>(n) * a.S + tok], -1);
}

DEV_INLINE const short* row_of(const HeadView& v, int n, int h) {
  return static_cast<const short*>(v.p) + n * v.sn + h * v.sh;
}

// block -> (sequence, head, owned tokens): one head's blocks stay on one XCD,
// whose L2 then holds what they stream
template <int OWN>
DEV_INLINE void locate(const MaskedAttn& a, int heads, bool last_first,
                       int* n, int* h, int* own0) {
  const int blocks = (a.S + OWN - 1) / OWN;
  const int total = gridDim.x;
  const int q = total / kNumXCD, r = total % kNumXCD;
  const int xcd = blockIdx.x % kNumXCD, idx = blockIdx.x / kNumXCD;
  const int id =
      (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  const int nh = id / blocks;
  int b = id % blocks;
  if (last_first) b = blocks - 1 - b;  // causal: the longest rows first
  *n = nh / heads;
  *h = nh % heads;
  *own0 = b * OWN;
}

// From q.k to what the exponential takes: p = exp2(c z - statistic), with z
// -inf where the pair is masked.
template <Mode M>
struct Score {
  float c;       // scale * log2 e, or cap * log2 e
  float cap_in;  // scale / cap
  float slope;   // slope * log2 e / c
  bool fast;     // fast_tanh will do

  DEV_INLINE Score(const MaskedAttn& a, int h) {
    c = a.scale * kLog2e;
    cap_in = 0.f;
    fast = a.softcap <= kFastCap;
    if (M == kCap) {
      cap_in = a.scale / a.softcap;
      c = a.softcap * kLog2e;
    }
    slope = M != kPlain && a.slopes != nullptr ? a.slopes[h] * kLog2e / c
                                               : 0.f;
  }

  // the cap, in units of it
  DEV_INLINE void bend(f32x16& z) const {
    if constexpr (M == kCap) {
      if (fast) {
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = fast_tanh(z[r] * cap_in);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = near_tanh(z[r] * cap_in);
      }
    }
  }
  // The bias, after the cap.  dist: owned token minus the streamed token of
  // register 0
  DEV_INLINE void lean(f32x16& z, float dist) const {
    if constexpr (M != kPlain) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        z[r] -= slope * fabsf(dist - ((r & 3) + 8 * (r >> 2)));
    }
  }
  // The same but for a part that all of the lane's scores share, which is
  // returned.  rel: the wave's first owned token minus the first streamed one.
  // Where one side's tokens all precede the other's, the distance is a sum of
  // the lane's part and the register's, one operation a score.
  DEV_INLINE float lean(f32x16& z, float dist, int rel) const {
    if constexpr (M == kPlain) return 0.f;
    if (rel > -31 && rel < 31) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        z[r] -= slope * fabsf(dist - ((r & 3) + 8 * (r >> 2)));
      return 0.f;
    }
    const float s = rel > 0 ? slope : -slope;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      z[r] = __builtin_fmaf(static_cast<float>((r & 3) + 8 * (r >> 2)), s,
                            z[r]);
    return -s * dist;
  }
};

// -inf where this lane's token and the streamed ones are not a pair.  doc: the
// streamed tokens' documents from register 0's on; own_doc: -2 for a token
// without any.  OWN_Q: the streamed token has to be at most `lim`, else at
// least.  One test covers the causal mask and the prefix (pair_limit).
template <bool OWN_Q>
DEV_INLINE void mask(f32x16& z, int own_doc, int lim, int other0,
                     const int* doc) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int4 d = *reinterpret_cast<const int4*>(doc + g * 8);
    const int dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int tok = other0 + g * 8 + j;
      const bool ok = (dd[j] == own_doc) & (OWN_Q ? tok <= lim : tok >= lim);
      z[g * 4 + j] = ok ? z[g * 4 + j] : -INFINITY;
    }
  }
}

// OWN_Q: the last key that query `own` may attend to; else the first query
// that may attend to key `own`
template <bool OWN_Q>
DEV_INLINE int pair_limit(const MaskedAttn& a, int n, int own) {
  if (!a.causal) return OWN_Q ? 0x7fffffff : 0;
  const int prefix = a.prefix != nullptr ? a.prefix[n] : 0;
  if (OWN_Q) return max(own, max(prefix, 0) - 1);
  return own < prefix ? 0 : own;
}

template <int DP, bool OWN = false>
struct Smem {
  char tile[2][2][Tile<DP>::kBytes];  // buffer, operand
  char own[OWN ? 2 : 0][2][Tile<DP>::kBytes];  // operand, 64 tokens
  int doc[2][kTile];
  float lse[2][kTile];    // dk/dv only
  float delta[2][kTile];  // dk/dv only
  unsigned list[kList];
  int4 sum[kShort / 32];
  int count;
};

// The two waves of 32 owned tokens (KS = 2) meet in the tile buffers: the
// second leaves its registers, the first picks them up.
template <int N>
DEV_INLINE void leave(float* at, const f32x16 (&x)[N]) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) at[(i * 16 + r) * kWave + lane] = x[i][r];
}
template <int N>
DEV_INLINE void pick_up(const float* at, f32x16 (&x)[N]) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) x[i][r] = at[(i * 16 + r) * kWave + lane];
}

inline Mode mode_of(const MaskedAttn& a) {
  return a.softcap > 0.f ? kCap : a.slopes != nullptr ? kBias : kPlain;
}

// calls f.template run<T, DP, M>()
template <typename F, typename T, int DP>
void with_mode(const F& f, const MaskedAttn& a) {
  switch (mode_of(a)) {
    case kPlain:
      return f.template run<T, DP, kPlain>();
    case kBias:
      return f.template run<T, DP, kBias>();
    case kCap:
      return f.template run<T, DP, kCap>();
  }
}
template <typename F, typename T>
void with_size(const F& f, const MaskedAttn& a) {
  if (a.D <= 32)
    with_mode<F, T, 32>(f, a);
  else if (a.D <= 64)
    with_mode<F, T, 64>(f, a);
  else
    with_mode<F, T, 128>(f, a);
}
template <typename F>
void with_type(const F& f, const MaskedAttn& a, Elem type) {
  if (type == Elem::kBF16)
    with_size<F, bf16>(f, a);
  else
    with_size<F, f16>(f, a);
}

}  // namespace masked_attn

}  // namespace colearn
