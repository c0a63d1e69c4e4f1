// AdamW over many tensors: one launch takes up to 48 tensors, whose addresses
// travel in the kernel's arguments (no table in memory to keep in step with
// gradients that move).
//
//   g' = g + mu (w - ref)                      (FedProx, optional)
//   m  = b1 m + (1 - b1) g'
//   v  = b2 v + (1 - b2) g'^2
//   w  = (1 - lr wd) w - (lr / bc1) m / (sqrt(v / bc2) + eps)
//
// States in 32 bits, or in 8: blocks of 256 consecutive elements of a tensor
// share an fp32 scale and hold e4m3(x / scale).  The second moment is held as
// its root, whose range is half as wide in the exponent, and a positive root
// never rounds to 0: the next step divides by it, and a first moment over a
// lost root would be a step without bound.  The step itself uses the moments
// before they are rounded.
//
// Every operation is rounded by itself, to nearest (no contraction; hipcc's
// division and square root are correctly rounded by default): a code next to a
// rounding border depends on the last bit, and one code off is a parameter off
// by a sixteenth of its step, so the operations are part of the format:
//   scale = max|x| * fl(1 / 448),   code = e4m3(x * fl(448 * fl(1 / max|x|)))
// Products, not divisions: torch divides a GPU tensor by a number, and a number
// by a tensor, in just these steps, so its GPU operations, its CPU ones and
// this kernel give the same bits.  (With true divisions here, half of all
// scales and about 40 of BERT-base's 220 M codes differ from torch's on the GPU
// after one step, and parameters from the second on.)
//
// Bound by memory: 28 bytes an element with fp32 states, 16 with 8-bit ones.
// A wave owns a block (four elements a lane), so a block's maximum is a wave
// reduction and nothing goes through LDS.  One block a wave and nothing left to
// wait for: BERT-base's 153 tensors, 110 M parameters, take 578 us with fp32
// states (5.3 TB/s) and 317 us with 8-bit ones (5.5 TB/s) in four launches; two
// blocks a wave, one after another, take 594 and 350 us.

#include "elem.h"
#include "encoder_api.h"

namespace colearn {

namespace {

constexpr float kE4M3Max = 448.f;
constexpr float kE4M3Min = 0.001953125f;  // 2^-9
constexpr float kTiny = 1e-30f;  // blocks below this are held as 0: 448 / top
                                 // stays finite

DEV_INLINE void codes_to_f(unsigned c, float (&x)[4]) {
  x[0] = __builtin_amdgcn_cvt_f32_fp8(c, 0);
  x[1] = __builtin_amdgcn_cvt_f32_fp8(c, 1);
  x[2] = __builtin_amdgcn_cvt_f32_fp8(c, 2);
  x[3] = __builtin_amdgcn_cvt_f32_fp8(c, 3);
}
DEV_INLINE unsigned f_to_codes(const float (&x)[4]) {
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], c, true);
}

template <typename P, typename G, bool EIGHT, bool PROX>
__global__ __launch_bounds__(256) void adamw_kernel(AdamwTable tab,
                                                    AdamwScalars sc) {
#pragma clang fp contract(off)
  // this workgroup's tensor: the last one that starts at or before it
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= static_cast<int>(blockIdx.x))
      lo = mid;
    else
      hi = mid - 1;
  }
  const AdamwTensor t = tab.t[lo];
  const float keep = tab.keep[lo];
  const bool vec = (tab.aligned >> lo) & 1;
  float step = sc.step, inv_bc2 = sc.inv_bc2;
  if (sc.live != nullptr) {
    step = sc.live[0];
    inv_bc2 = sc.live[1];
  }
  P* const p = static_cast<P*>(t.p);
  const G* const g = static_cast<const G*>(t.g);
  static_assert(kAdamwChunk == 4 * kAdamwBlock, "a block a wave");
  const int64_t base =
      static_cast<int64_t>(blockIdx.x - tab.first[lo]) * kAdamwChunk +
      wave * kAdamwBlock;
  if (base >= t.n) return;  // whole waves leave: no barrier follows
  const bool whole = vec && base + kAdamwBlock <= t.n;
  float w[4], gr[4], m[4], v[4], rf[4];
  float s_m = 1.f, s_v = 1.f;
  const int64_t blk = base / kAdamwBlock;
  if constexpr (EIGHT) {
    s_m = t.ms[blk];
    s_v = t.vs[blk];
  }
  if (whole) {
    const int64_t i = base + lane * 4;
    elem_load4(p + i, w);
    elem_load4(g + i, gr);
    if constexpr (EIGHT) {
      codes_to_f(*reinterpret_cast<const unsigned*>(
                     static_cast<const unsigned char*>(t.m) + i), m);
      codes_to_f(*reinterpret_cast<const unsigned*>(
                     static_cast<const unsigned char*>(t.v) + i), v);
    } else {
      elem_load4(static_cast<const float*>(t.m) + i, m);
      elem_load4(static_cast<const float*>(t.v) + i, v);
    }
    if constexpr (PROX) elem_load4(t.ref + i, rf);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = base + j * kWave + lane;
      w[j] = gr[j] = m[j] = v[j] = rf[j] = 0.f;
      if (i < t.n) {
        w[j] = elem_load(p + i);
        gr[j] = elem_load(g + i);
        if constexpr (EIGHT) {
          m[j] = __builtin_amdgcn_cvt_f32_fp8(
              static_cast<const unsigned char*>(t.m)[i], 0);
          v[j] = __builtin_amdgcn_cvt_f32_fp8(
              static_cast<const unsigned char*>(t.v)[i], 0);
        } else {
          m[j] = static_cast<const float*>(t.m)[i];
          v[j] = static_cast<const float*>(t.v)[i];
        }
        if constexpr (PROX) rf[j] = t.ref[i];
      }
    }
  }
  float top_m = 0.f, top_v = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (EIGHT) {
      m[j] = m[j] * s_m;
      v[j] = v[j] * s_v;
      v[j] = v[j] * v[j];
    }
    float gk = gr[j];
    if constexpr (PROX) gk = gk + sc.mu * (w[j] - rf[j]);
    m[j] = m[j] * sc.b1 + gk * sc.omb1;
    v[j] = v[j] * sc.b2 + (gk * gk) * sc.omb2;
    w[j] = w[j] * keep -
           (m[j] / (sqrtf(v[j] * inv_bc2) + sc.eps)) * step;
    if constexpr (EIGHT) {
      v[j] = sqrtf(v[j]);
      top_m = fmaxf(top_m, fabsf(m[j]));
      top_v = fmaxf(top_v, v[j]);
    }
  }
  if constexpr (EIGHT) {
    top_m = lanes_max(top_m);
    top_v = lanes_max(top_v);
    const float inv_m = top_m > kTiny ? (1.f / top_m) * kE4M3Max : 0.f;
    const float inv_v = top_v > kTiny ? (1.f / top_v) * kE4M3Max : 0.f;
    if (lane == 0) {
      t.ms[blk] = top_m > kTiny ? top_m * (1.f / kE4M3Max) : 0.f;
      t.vs[blk] = top_v > kTiny ? top_v * (1.f / kE4M3Max) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = m[j] * inv_m;
      v[j] = v[j] * inv_v;
      if (v[j] > 0.f) v[j] = fmaxf(v[j], kE4M3Min);
    }
  }
  if (whole) {
    const int64_t i = base + lane * 4;
    elem_store4(p + i, w);
    if constexpr (EIGHT) {
      *reinterpret_cast<unsigned*>(static_cast<unsigned char*>(t.m) + i) =
          f_to_codes(m);
      *reinterpret_cast<unsigned*>(static_cast<unsigned char*>(t.v) + i) =
          f_to_codes(v);
    } else {
      elem_store4(static_cast<float*>(t.m) + i, m);
      elem_store4(static_cast<float*>(t.v) + i, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = base + j * kWave + lane;
      if (i < t.n) {
        elem_store(p + i, w[j]);
        if constexpr (EIGHT) {
          static_cast<unsigned char*>(t.m)[i] =
              __builtin_amdgcn_cvt_pk_fp8_f32(m[j], m[j], 0, false) & 0xff;
          static_cast<unsigned char*>(t.v)[i] =
              __builtin_amdgcn_cvt_pk_fp8_f32(v[j], v[j], 0, false) & 0xff;
        } else {
          static_cast<float*>(t.m)[i] = m[j];
          static_cast<float*>(t.v)[i] = v[j];
        }
      }
    }
  }
}

template <typename P, typename G, bool EIGHT>
void pick_prox(const AdamwTable& t, const AdamwScalars& s, bool prox,
               hipStream_t stream) {
  const int grid = t.first[t.count];
  if (prox)
    adamw_kernel<P, G, EIGHT, true><<<grid, 256, 0, stream>>>(t, s);
  else
    adamw_kernel<P, G, EIGHT, false><<<grid, 256, 0, stream>>>(t, s);
}

template <typename P, typename G>
void pick_bits(const AdamwTable& t, const AdamwScalars& s, bool eight,
               bool prox, hipStream_t stream) {
  if (eight)
    pick_prox<P, G, true>(t, s, prox, stream);
  else
    pick_prox<P, G, false>(t, s, prox, stream);
}

}  // namespace

void launch_adamw(const AdamwTable& t, const AdamwScalars& s, bool p_bf16,
                  bool g_bf16, bool eight, bool prox, hipStream_t stream) {
  static_assert(sizeof(AdamwTable) + sizeof(AdamwScalars) <= 4096,
                "the table has to fit the kernel's arguments");
  if (p_bf16 && g_bf16)
    pick_bits<bf16, bf16>(t, s, eight, prox, stream);
  else if (p_bf16)
    pick_bits<bf16, float>(t, s, eight, prox, stream);
  else if (g_bf16)
    pick_bits<float, bf16>(t, s, eight, prox, stream);
  else
    pick_bits<float, float>(t, s, eight, prox, stream);
}

}  // namespace colearn
