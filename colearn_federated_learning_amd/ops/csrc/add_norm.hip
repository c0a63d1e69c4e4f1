// Residual add + layer norm, forward and backward, in fp32, bf16 or fp16.
//
//   s = round(x + r)            (a tensor of the model's type: what is
//                                normalised, and what the backward reads)
//   y = (s - mean) * inv * w + b,   inv = 1 / sqrt(var + eps)
//   gx = inv * (gw' - mean(gw') - xh * mean(gw' * xh)) [+ gs],  gw' = gy * w
//   dw = sum over rows gy * xh,     db = sum over rows gy
//
// Rows are client-major in groups of rpg rows, each group with its own w and b
// (the stacked engine; one group otherwise).  Statistics are fp32, and the
// variance is the mean of squared distances from the mean: the row stays in
// registers, so the second pass over it costs no memory.
//
// Bound by memory: 65536 x 768 in bf16, forward 74 us (5.4 TB/s), backward 58
// to 62 and the join 4 (4.5 to 4.9 TB/s); 4096 x 768, where a launch begins to
// show, 7 and 8 + 3; 16384 x 1024 in fp32 54 and 33 + 4 (5.0, 5.4 TB/s).  A
// row's elements lie over W waves, at most 16 a lane (W = 1 up to 1024 columns,
// 4 up to 4096, 16 up to 16384), so the backward can hold both weight sums of
// its columns in registers over all its rows and read everything once: each
// workgroup leaves one row of partial sums, which a second launch adds up in a
// fixed order.

#include "elem.h"
#include "encoder_api.h"

namespace colearn {

namespace {

// sums over the W waves of a row; every lane gets them
template <int W, int N>
DEV_INLINE void row_sum(float (&v)[N], float (*red)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum(v[i]);
  if constexpr (W > 1) {
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) t += red[k][i];
      v[i] = t;
    }
    __syncthreads();  // red is free again
  }
}

// element index of this lane's k-th vector
template <int VEC, int W>
DEV_INLINE int col_of(int k) {
  const int wave = W > 1 ? threadIdx.x / kWave : 0;
  return ((k * W + wave) * kWave + threadIdx.x % kWave) * VEC;
}

// a vector as it lies in memory, and its values
template <typename T, int VEC>
struct Raw {
  T x[VEC];
};
template <typename T>
struct alignas(4 * sizeof(T)) Raw<T, 4> {
  T x[4];
};
template <int VEC, typename T>
DEV_INLINE Raw<T, VEC> load_raw(const T* p) {
  return *reinterpret_cast<const Raw<T, VEC>*>(p);
}
template <int VEC, typename T>
DEV_INLINE void widen(const Raw<T, VEC>& r, float* x) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) x[j] = elem_load(&r.x[j]);
}

template <int VEC, typename T>
DEV_INLINE void load_vec(const T* p, float* x) {
  if constexpr (VEC == 4)
    elem_load4(p, x);
  else
    x[0] = elem_load(p);
}
template <int VEC, typename T>
DEV_INLINE void store_vec(T* p, const float* x) {
  if constexpr (VEC == 4)
    elem_store4(p, x);
  else
    elem_store(p, x[0]);
}

template <typename T, int VEC, int NV, int W>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void add_norm_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ r,
    const float* __restrict__ wg, const float* __restrict__ bg,
    T* __restrict__ s, T* __restrict__ y, float* __restrict__ mean,
    float* __restrict__ inv, int64_t rows, int64_t rpg, int H, float eps) {
  constexpr int kRows = W == 1 ? 4 : 1;
  __shared__ float red[W][1];
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * kRows +
      (W == 1 ? threadIdx.x / kWave : 0);
  if (row >= rows) return;  // W > 1: the whole workgroup
  const float* w = wg + (row / rpg) * H;
  const float* b = bg + (row / rpg) * H;
  float v[NV * VEC];
  float sum[1] = {0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = col_of<VEC, W>(k);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[k * VEC + j] = 0.f;
    if (c < H) {
      load_vec<VEC>(x + row * H + c, v + k * VEC);
      if (r != nullptr) {
        float u[VEC];
        load_vec<VEC>(r + row * H + c, u);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          v[k * VEC + j] = elem_round(v[k * VEC + j] + u[j], x);
        store_vec<VEC>(s + row * H + c, v + k * VEC);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[0] += v[k * VEC + j];
    }
  }
  row_sum<W>(sum, red);
  const float mu = sum[0] / H;
  sum[0] = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (col_of<VEC, W>(k) < H) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = v[k * VEC + j] - mu;
        sum[0] += d * d;
      }
    }
  row_sum<W>(sum, red);
  const float is = 1.f / sqrtf(sum[0] / H + eps);
  if (W == 1 ? threadIdx.x % kWave == 0 : threadIdx.x == 0) {
    mean[row] = mu;
    inv[row] = is;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = col_of<VEC, W>(k);
    if (c < H) {
      float wv[VEC], bv[VEC], o[VEC];
      load_vec<VEC>(w + c, wv);
      load_vec<VEC>(b + c, bv);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        o[j] = (v[k * VEC + j] - mu) * is * wv[j] + bv[j];
      store_vec<VEC>(y + row * H + c, o);
    }
  }
}

// grid (workgroups a group, groups); partials [groups][gridDim.x][2][H]
template <typename T, int VEC, int NV, int W>
__global__ __launch_bounds__(W == 16 ? 1024 : 256) void add_norm_bwd_kernel(
    const T* __restrict__ gy, const T* __restrict__ gs,
    const T* __restrict__ s, const float* __restrict__ wg,
    const float* __restrict__ mean, const float* __restrict__ inv,
    T* __restrict__ gx, float* __restrict__ partials, int64_t rpg, int H) {
  constexpr int kRows = W == 1 ? 4 : 1;
  constexpr int EL = NV * VEC;
  __shared__ float red[W][2];
  const float* w = wg + static_cast<int64_t>(blockIdx.y) * H;
  float wv[EL], aw[EL], ab[EL];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = col_of<VEC, W>(k);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      wv[k * VEC + j] = aw[k * VEC + j] = ab[k * VEC + j] = 0.f;
    if (c < H) load_vec<VEC>(w + c, wv + k * VEC);
  }
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * rpg;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t q = static_cast<int64_t>(blockIdx.x) * kRows +
              (W == 1 ? threadIdx.x / kWave : 0);
  // The next rows' loads are under way while a row is reduced and written: two
  // rows of 16-bit elements (65536 x 768 in 8 groups 58 us, one row 63; 8192 x
  // 4096 37 and 41), one of 32-bit ones (4099 x 1023, both gradients, 25.0, two
  // 25.4; without the sum's 13.3, 13.8), none where 16 waves leave no registers
  // for them.
  constexpr int kAhead = W == 16 ? 0 : sizeof(T) == 2 ? 2 : 1;
  struct Row {
    Raw<T, VEC> g[NV], s[NV];
    float mu, is;
  } rows[kAhead > 0 ? kAhead : 1];
  auto fetch = [&](Row& to, int64_t row) {
    to.mu = mean[row];
    to.is = inv[row];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = min(col_of<VEC, W>(k), H - VEC);
      to.g[k] = load_raw<VEC>(gy + row * H + c);
      to.s[k] = load_raw<VEC>(s + row * H + c);
    }
  };
  auto work = [&](Row& in) {
    const int64_t row = row0 + q;
    if (kAhead == 0) fetch(in, row);
    float g[EL], xh[EL];
    float sum[2] = {0.f, 0.f};
    const float m = in.mu, rs = in.is;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      widen<VEC>(in.g[k], g + k * VEC);
      widen<VEC>(in.s[k], xh + k * VEC);
    }
    if (kAhead > 0 && q + kAhead * stride < rpg)
      fetch(in, row + kAhead * stride);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (col_of<VEC, W>(k) < H) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = k * VEC + j;
          xh[e] = (xh[e] - m) * rs;
          ab[e] += g[e];
          aw[e] += g[e] * xh[e];
          g[e] *= wv[e];
          sum[0] += g[e];
          sum[1] += g[e] * xh[e];
        }
      }
    }
    row_sum<W>(sum, red);
    sum[0] /= H;
    sum[1] /= H;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = col_of<VEC, W>(k);
      if (c < H) {
        float o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const int e = k * VEC + j;
          o[j] = rs * (g[e] - sum[0] - xh[e] * sum[1]);
        }
        if (gs != nullptr) {
          float u[VEC];
          load_vec<VEC>(gs + row * H + c, u);
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] += u[j];
        }
        store_vec<VEC>(gx + row * H + c, o);
      }
    }
    q += stride;
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (q + i * stride < rpg) fetch(rows[i], row0 + q + i * stride);
  while (q < rpg) {
    work(rows[0]);
    if (kAhead > 1 && q < rpg) work(rows[kAhead - 1]);
  }
  float* out = partials + (static_cast<int64_t>(blockIdx.y) * gridDim.x +
                           blockIdx.x) * 2 * H;
  if constexpr (W == 1) {
    // the workgroup's four waves hold the same columns: joined in LDS, wave
    // by wave in order
    __shared__ float join[2 * kWave * EL];
    const int wave = threadIdx.x / kWave;
    for (int step = 0; step < 4; ++step) {
      if (wave == step) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int e = k * VEC + j, c = col_of<VEC, W>(k) + j;
            float* a = join + c;
            float* d = join + kWave * EL + c;
            *a = step == 0 ? aw[e] : *a + aw[e];
            *d = step == 0 ? ab[e] : *d + ab[e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < H; c += 256) {
      out[c] = join[c];
      out[H + c] = join[kWave * EL + c];
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = col_of<VEC, W>(k);
      if (c < H) {
        store_vec<VEC>(out + c, aw + k * VEC);
        store_vec<VEC>(out + H + c, ab + k * VEC);
      }
    }
  }
}

// grid (columns / 64, groups), 16 waves: lane = column, wave = every 16th
// partial row
__global__ __launch_bounds__(1024) void add_norm_join_kernel(
    const float* __restrict__ partials, float* __restrict__ dw,
    float* __restrict__ db, int n, int H) {
  __shared__ float red[16][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int c = blockIdx.x * kWave + lane;  // of 2 H
  const float* p = partials + static_cast<int64_t>(blockIdx.y) * n * 2 * H;
  float t = 0.f;
  if (c < 2 * H) {
#pragma unroll 8
    for (int i = wave; i < n; i += 16)
      t += p[static_cast<int64_t>(i) * 2 * H + c];
  }
  red[wave][lane] = t;
  __syncthreads();
  if (wave == 0 && c < 2 * H) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[k][lane];
    float* out = c < H ? dw : db;
    out[static_cast<int64_t>(blockIdx.y) * H + (c < H ? c : c - H)] = t;
  }
}

struct NormArgs {
  const AddNormFwd* f;
  const AddNormBwd* b;
  hipStream_t stream;
};

template <typename T, int VEC, int NV, int W>
void run(const NormArgs& a) {
  constexpr int kThreads = W == 16 ? 1024 : 256;
  constexpr int kRows = W == 1 ? 4 : 1;
  if (a.f != nullptr) {
    const AddNormFwd& f = *a.f;
    const int64_t grid = (f.rows + kRows - 1) / kRows;
    add_norm_fwd_kernel<T, VEC, NV, W>
        <<<static_cast<unsigned>(grid), kThreads, 0, a.stream>>>(
            static_cast<const T*>(f.x), static_cast<const T*>(f.r), f.w, f.b,
            static_cast<T*>(f.s), static_cast<T*>(f.y), f.mean, f.inv, f.rows,
            f.rows / f.groups, f.H, f.eps);
  } else {
    const AddNormBwd& b = *a.b;
    add_norm_bwd_kernel<T, VEC, NV, W>
        <<<dim3(b.parts, b.groups), kThreads, 0, a.stream>>>(
            static_cast<const T*>(b.gy), static_cast<const T*>(b.gs),
            static_cast<const T*>(b.s), b.w, b.mean, b.inv,
            static_cast<T*>(b.gx), b.partials, b.rows / b.groups, b.H);
    add_norm_join_kernel<<<dim3((2 * b.H + kWave - 1) / kWave, b.groups),
                           1024, 0, a.stream>>>(b.partials, b.dw, b.db,
                                                b.parts, b.H);
  }
}

template <typename T, int VEC, int W>
void pick_nv(const NormArgs& a, int H) {
  const int q = (H + kWave * W * 4 - 1) / (kWave * W * 4);  // quads a lane
  constexpr int U = 4 / VEC;
  if (q <= 1)
    run<T, VEC, U, W>(a);
  else if (q == 2)
    run<T, VEC, 2 * U, W>(a);
  else if (q == 3)
    run<T, VEC, 3 * U, W>(a);
  else
    run<T, VEC, 4 * U, W>(a);
}

template <typename T, int VEC>
void pick_w(const NormArgs& a, int H) {
  if (H <= 16 * kWave)
    pick_nv<T, VEC, 1>(a, H);
  else if (H <= 16 * kWave * 4)
    pick_nv<T, VEC, 4>(a, H);
  else
    pick_nv<T, VEC, 16>(a, H);
}

void pick(const NormArgs& a, Elem type, bool vec, int H) {
  switch (type) {
    case Elem::kF32:
      return vec ? pick_w<float, 4>(a, H) : pick_w<float, 1>(a, H);
    case Elem::kBF16:
      return vec ? pick_w<bf16, 4>(a, H) : pick_w<bf16, 1>(a, H);
    case Elem::kF16:
      return vec ? pick_w<f16, 4>(a, H) : pick_w<f16, 1>(a, H);
  }
}

}  // namespace

int add_norm_parts(int64_t rows, int groups, int H) {
  // A row of partial sums costs as much as two thirds of a 16-bit data row:
  // at least two rows a wave, and two workgroups a CU over all groups.  Rows
  // of 768 in bf16, us with the join at 1 / 2 / 4 / 8 rows a wave: 4096 rows
  // 14.2 / 11.7 / 12.6 / 15.5; 65536 rows at 2 / 4 / 8 workgroups a CU: 66 /
  // 68 / 69.
  const int64_t rpg = rows / groups;
  const int64_t per = H <= 16 * kWave ? 8 : 2;
  const int64_t most = (2 * kNumCU + groups - 1) / groups;
  int64_t n = (rpg + per - 1) / per;
  n = n < most ? n : most;
  return static_cast<int>(n > 0 ? n : 1);
}

void launch_add_norm_fwd(const AddNormFwd& f, Elem type, bool vec,
                         hipStream_t stream) {
  pick({&f, nullptr, stream}, type, vec, f.H);
}

void launch_add_norm_bwd(const AddNormBwd& b, Elem type, bool vec,
                         hipStream_t stream) {
  pick({nullptr, &b, stream}, type, vec, b.H);
}

}  // namespace colearn
