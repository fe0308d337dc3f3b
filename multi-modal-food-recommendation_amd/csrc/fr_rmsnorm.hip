// Root-mean-square norm with the residual's addition, forward (also with an 8-bit output) and backward.
//
//   h = x + residual        (rounded to the storage type where it is stored)
//   y = w h rstd,  rstd = 1 / sqrt(mean(h^2) + eps), from the unrounded h
//   8 bits: q = e4m3(y / s),  s = max |y| / 448 per row (1 for a row of zeros)
//   dx = dresidual = rstd (w dy - xh mean(w dy xh)) + dh,   dw = sum over rows of dy xh,   xh = h rstd
//
// One pass: a group of G threads keeps its whole row in registers as fp32 (K vectors of VN elements
// per thread), so x and the residual are read once and y and h written once; the backward reads dy,
// dh and h once.  A stored h of bf16 is rounded, which dw would show (each of its terms off by 2^-9, as
// much as dw's own rounding): the backward then takes x and the residual and adds them again, one
// read more.  The kernels are bound by HBM: 16,384 x 2,048 bf16 forward 44 us (6.1 TB/s), backward 65 us
// (5.2 TB/s) and 5 us for dw's sum; 20,480 x 64 fp32 5 + 5 + 4 us.
//
// The backward's dw: a thread owns the same columns for every row that its group takes (rows in a
// grid-stride order), adds them up in registers, groups and waves of a block are joined in a fixed
// order, and a second kernel adds the blocks' partials in block order: deterministic, no atomics.
#include "fr_vec.h"

#include <algorithm>

namespace {

using fr::bf16_t;

// upper limit of the backward's blocks = partial rows of dw: three per compute unit are resident with wide rows
// (16,384 x 2,048 bf16 with a residual: 65 us, 73 us with 1,024, whose last third waits)
constexpr int kBwdBlocks = 768;

template <int G>
__device__ __forceinline__ float gsum(float v, float* red) {
  if constexpr (G <= 64) {
    return group_sum<G>(v);
  } else {
    v = group_sum<64>(v);
    __syncthreads();  // the previous row's (or sum's) readers are done with red
    if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int i = 1; i < G / 64; ++i) s += red[i];
    return s;
  }
}

// maximum of non-negative floats as integers: a NaN is larger than every number, so it is kept
template <int G>
__device__ __forceinline__ uint32_t gmax(uint32_t v, float* red) {
#pragma unroll
  for (int off = (G < 64 ? G : 64) / 2; off > 0; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
  if constexpr (G > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = __uint_as_float(v);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G / 64; ++i) v = max(v, __float_as_uint(red[i]));
  }
  return v;
}

// s of a row whose largest |y| has the bits `top`: never 0, and of the two subnormal numbers around a quotient the
// one that keeps |y| / s within 8 bits' range
__device__ __forceinline__ float quant_scale(uint32_t top) {
  if (!top) return 1.f;
  const float y = __uint_as_float(top), s = y / 448.f;
  return s < 1.17549435e-38f && s * 448.f < y ? __uint_as_float(__float_as_uint(s) + 1u) : s;
}

struct FwdArgs {
  const void *x, *r, *w;
  void *y, *h;
  float *rstd, *scale;
  int64_t ldx, ldr, rows;
  int d, w_f32;
  float eps, inv_d;
};

template <typename T, int VN>
__device__ __forceinline__ void load_w(const void* w, int w_f32, int c, float* o) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < VN; ++i) o[i] = 1.f;
  } else if (w_f32) {
    // VN floats: fp32 vectors where the rows are vectors (the host has checked w's alignment)
    constexpr int FN = VN >= 4 ? 4 : 1;
#pragma unroll
    for (int i = 0; i < VN; i += FN) fr::Vec<float, FN>::load(static_cast<const float*>(w) + c + i, o + i);
  } else {
    fr::Vec<T, VN>::load(static_cast<const T*>(w) + c, o);
  }
}

template <typename T, int VN, int G, int K, bool QUANT>
__global__ __launch_bounds__(256) void rms_fwd_kernel(FwdArgs a) {
  __shared__ float red[4];
  constexpr int GPB = 256 / G;
  const int t = threadIdx.x % G;
  const int64_t row = fr::block_number() * GPB + threadIdx.x / G;
  const bool live = row < a.rows;  // a group past the end still takes part in the barriers and shuffles
  const T* X = static_cast<const T*>(a.x) + (live ? row : 0) * a.ldx;
  const T* R = a.r ? static_cast<const T*>(a.r) + (live ? row : 0) * a.ldr : nullptr;
  float v[K][VN];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * G + t) * VN;
#pragma unroll
    for (int i = 0; i < VN; ++i) v[k][i] = 0.f;
    if (live && c < a.d) {
      fr::Vec<T, VN>::load(X + c, v[k]);
      if (R) {
        float r[VN];
        fr::Vec<T, VN>::load(R + c, r);
#pragma unroll
        for (int i = 0; i < VN; ++i) v[k][i] += r[i];
        if (a.h) fr::Vec<T, VN>::store(static_cast<T*>(a.h) + row * a.d + c, v[k]);
      }
    }
#pragma unroll
    for (int i = 0; i < VN; ++i) ss = fmaf(v[k][i], v[k][i], ss);
  }
  const float rstd = 1.f / sqrtf(gsum<G>(ss, red) * a.inv_d + a.eps);
  if (live && t == 0 && a.rstd) a.rstd[row] = rstd;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * G + t) * VN;
    if (live && c < a.d) {
      float w[VN];
      load_w<T, VN>(a.w, a.w_f32, c, w);
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        v[k][i] = v[k][i] * rstd * w[i];
        if constexpr (QUANT) top = max(top, __float_as_uint(v[k][i]) & 0x7fffffffu);
      }
      if constexpr (!QUANT) fr::Vec<T, VN>::store(static_cast<T*>(a.y) + row * a.d + c, v[k]);
    }
  }
  if constexpr (QUANT) {
    top = gmax<G>(top, red);
    const float s = quant_scale(top);
    if (live && t == 0) a.scale[row] = s;
    uint8_t* Q = static_cast<uint8_t*>(a.y) + row * a.d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * G + t) * VN;
      if (!live || c >= a.d) continue;
      if constexpr (VN == 1) {
        Q[c] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[k][0] / s, 0.f, 0, false);
      } else {
        uint32_t p[VN / 4];
#pragma unroll
        for (int i = 0; i < VN; i += 4) {
          int u = __builtin_amdgcn_cvt_pk_fp8_f32(v[k][i] / s, v[k][i + 1] / s, 0, false);
          u = __builtin_amdgcn_cvt_pk_fp8_f32(v[k][i + 2] / s, v[k][i + 3] / s, u, true);
          p[i / 4] = (uint32_t)u;
        }
        if constexpr (VN == 4) *reinterpret_cast<uint32_t*>(Q + c) = p[0];
        else *reinterpret_cast<uint2*>(Q + c) = make_uint2(p[0], p[1]);
      }
    }
  }
}

template <typename T, int VN>
__device__ __forceinline__ void add_floats(const typename fr::Vec<T, VN>::Raw& v, float* x) {
  float f[VN];
  fr::Vec<T, VN>::floats(v, f);
#pragma unroll
  for (int i = 0; i < VN; ++i) x[i] += f[i];
}

struct BwdArgs {
  const void *dy, *dh, *h, *r, *w;  // the normed rows are h, or h + r
  const float* rstd;
  void* dx;
  float* part;  // [gridDim.x][d] or null
  int64_t lddy, lddh, ldh, ldr, rows;
  int d, w_f32;
  float inv_d;
};

template <typename T, int VN, int G, int K>
__global__ __launch_bounds__(256) void rms_bwd_kernel(BwdArgs a) {
  constexpr int GPB = 256 / G, GPW = G < 64 ? 64 / G : 1;
  __shared__ float red[4];
  __shared__ float fold[G <= 64 ? 4 * G * K * VN : 1];
  const int t = threadIdx.x % G;
  using V = fr::Vec<T, VN>;
  float dw[K][VN];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < VN; ++i) dw[k][i] = 0.f;
  // the trip count is the block's, so that every thread meets the barriers and shuffles
  for (int64_t r0 = (int64_t)blockIdx.x * GPB; r0 < a.rows; r0 += (int64_t)gridDim.x * GPB) {
    const int64_t row = r0 + threadIdx.x / G;
    const bool live = row < a.rows;
    const float rstd = live ? a.rstd[row] : 0.f;
    // all of the row's loads first, kept as they lie in memory: half the registers of their floats in bf16
    typename V::Raw dy[K], h[K], r[K], dh[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * G + t) * VN;
      dy[k] = h[k] = r[k] = dh[k] = typename V::Raw{};
      if (live && c < a.d) {
        dy[k] = V::raw(static_cast<const T*>(a.dy) + row * a.lddy + c);
        h[k] = V::raw(static_cast<const T*>(a.h) + row * a.ldh + c);
        if (a.r) r[k] = V::raw(static_cast<const T*>(a.r) + row * a.ldr + c);
        if (a.dh) dh[k] = V::raw(static_cast<const T*>(a.dh) + row * a.lddh + c);
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * G + t) * VN;
      if (c < a.d) {
        float g[VN], x[VN], w[VN];
        load_w<T, VN>(a.w, a.w_f32, c, w);
        V::floats(dy[k], g);
        V::floats(h[k], x);
        if (a.r) add_floats<T, VN>(r[k], x);
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const float gx = g[i] * (x[i] * rstd);
          dw[k][i] += gx;
          dot = fmaf(gx, w[i], dot);
        }
      }
    }
    const float m = gsum<G>(dot, red) * a.inv_d;
    if (!a.dx) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * G + t) * VN;
      if (live && c < a.d) {
        float g[VN], x[VN], e[VN], w[VN];
        load_w<T, VN>(a.w, a.w_f32, c, w);
        V::floats(dy[k], g);
        V::floats(h[k], x);
        if (a.r) add_floats<T, VN>(r[k], x);
        V::floats(dh[k], e);
#pragma unroll
        for (int i = 0; i < VN; ++i) e[i] = fmaf(rstd, fmaf(-(x[i] * rstd), m, g[i] * w[i]), e[i]);
        V::store(static_cast<T*>(a.dx) + row * a.d + c, e);
      }
    }
  }
  if (!a.part) return;
  float* P = a.part + (int64_t)blockIdx.x * a.d;
  if constexpr (G > 64) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VN; ++i)
        if ((k * G + t) * VN + i < a.d) P[(k * G + t) * VN + i] = dw[k][i];
  } else {
    // the wave's groups by exchanges, then the four waves in order through LDS
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < VN; ++i) {
#pragma unroll
        for (int off = G; off < 64; off <<= 1) dw[k][i] += __shfl_xor(dw[k][i], off, 64);
        if ((threadIdx.x & 63) / G == 0 || GPW == 1)
          fold[(threadIdx.x / 64 * G * K + k * G + t) * VN + i] = dw[k][i];
      }
    __syncthreads();
    constexpr int W = G * K * VN;
    for (int c = threadIdx.x; c < a.d; c += 256) P[c] = ((fold[c] + fold[W + c]) + fold[2 * W + c]) + fold[3 * W + c];
  }
}

// dw[c] = sum over the blocks' partials: 16 columns per block, 16 threads per column each adding every
// 16th partial, joined in a fixed order
template <typename T>
__global__ __launch_bounds__(256) void rms_dw_kernel(const float* __restrict__ part, int nblocks, int d,
                                                     T* __restrict__ dw) {
  __shared__ float red[16][17];
  const int cl = threadIdx.x % 16, g = threadIdx.x / 16;
  const int c = blockIdx.x * 16 + cl;
  float s = 0.f;
  if (c < d) {
    int b = g;
    for (; b + 112 < nblocks; b += 128) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(int64_t)(b + 16 * k) * d + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; b < nblocks; b += 16) s += part[(int64_t)b * d + c];
  }
  red[g][cl] = s;
  __syncthreads();
  if (g == 0 && c < d) {
    float r = red[0][cl];
#pragma unroll
    for (int k = 1; k < 16; ++k) r += red[k][cl];
    dw[c] = fr::from_f32<T>(r);
  }
}

// G threads and K vectors per thread for `nv` vectors per row: up to a wave with 1 to 4 vectors each, a whole block
// with 2 to 8, and with 32 single elements for rows of more than 2,048 that are not whole 16-byte words (a row of
// 2,049 keeps 32 slots per thread, too, three quarters of them empty)
template <typename F>
bool by_width(int64_t nv, F&& f) {
  if (nv <= 8) f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
  else if (nv <= 16) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  else if (nv <= 32) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
  else if (nv <= 64) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  else if (nv <= 128) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  else if (nv <= 256) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
  else if (nv <= 512) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 2>{});
  else if (nv <= 1024) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
  else if (nv <= 2048) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
  else if (nv <= 8192) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 32>{});
  else return false;
  return true;
}

constexpr int kMaxD = 8192;

template <typename T, bool QUANT>
hipError_t launch_fwd(const FwdArgs& a, bool vec, hipStream_t s) {
  auto go = [&](auto vn, auto g, auto k) {
    constexpr int VN = decltype(vn)::value, G = decltype(g)::value, K = decltype(k)::value;
    if constexpr (VN * K <= 32)
      hipLaunchKernelGGL((rms_fwd_kernel<T, VN, G, K, QUANT>), fr::many_blocks(fr::ceil_div(a.rows, 256 / G)), dim3(256),
                         0, s, a);
  };
  if (vec) by_width(a.d / fr::kVec<T>, [&](auto g, auto k) { go(std::integral_constant<int, fr::kVec<T>>{}, g, k); });
  else by_width(a.d, [&](auto g, auto k) { go(std::integral_constant<int, 1>{}, g, k); });
  return hipGetLastError();
}

template <typename T>
hipError_t launch_bwd(BwdArgs a, bool vec, float* part, void* dw, hipStream_t s) {
  int nblocks = 0;
  auto go = [&](auto vn, auto g, auto k) {
    constexpr int VN = decltype(vn)::value, G = decltype(g)::value, K = decltype(k)::value;
    if constexpr (VN * K <= 32) {
      nblocks = (int)std::min<int64_t>(fr::ceil_div(a.rows, 256 / G), kBwdBlocks);
      a.part = part;
      hipLaunchKernelGGL((rms_bwd_kernel<T, VN, G, K>), dim3((unsigned)nblocks), dim3(256), 0, s, a);
    }
  };
  if (vec) by_width(a.d / fr::kVec<T>, [&](auto g, auto k) { go(std::integral_constant<int, fr::kVec<T>>{}, g, k); });
  else by_width(a.d, [&](auto g, auto k) { go(std::integral_constant<int, 1>{}, g, k); });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !dw) return e;
  const dim3 grid((unsigned)fr::ceil_div(a.d, 16));
  if (a.w_f32 || sizeof(T) == 4)
    hipLaunchKernelGGL(rms_dw_kernel<float>, grid, dim3(256), 0, s, part, nblocks, a.d, static_cast<float*>(dw));
  else
    hipLaunchKernelGGL(rms_dw_kernel<bf16_t>, grid, dim3(256), 0, s, part, nblocks, a.d, static_cast<bf16_t*>(dw));
  return hipGetLastError();
}

// rows of 16-byte vectors: the pointer aligned and the stride a whole number of vectors
bool vec_ok(const void* p, int64_t ld, int vn) { return !p || (fr::aligned16(p) && ld % vn == 0); }

}  // namespace

extern "C" int fr_rms_norm_fwd(const void* d_x, int64_t ldx, const void* d_residual, int64_t ldr, int64_t rows, int d,
                               int dtype, const void* d_w, int w_dtype, float eps, void* d_y, int quant,
                               float* d_scale, void* d_h, float* d_rstd, void* stream) {
  FR_REQUIRE(dtype == FR_F32 || dtype == FR_BF16, "dtype must be FR_F32 or FR_BF16");
  FR_REQUIRE(w_dtype == FR_F32 || w_dtype == dtype, "the weight is fp32 or of the rows' type");
  FR_REQUIRE(d >= 1 && d <= kMaxD, "d must be in [1, 8192]");
  FR_REQUIRE(rows >= 0 && rows < ((int64_t)1 << 31) && ldx >= d && (!d_residual || ldr >= d), "bad shape");
  FR_REQUIRE(!d_h || d_residual, "h is x itself without a residual");
  FR_REQUIRE(eps >= 0.f && eps < INFINITY, "eps must be a number >= 0");
  if (rows == 0) return FR_OK;
  FR_REQUIRE(d_x && d_y && (!quant || d_scale), "null pointer");
  const int vn = dtype == FR_F32 ? 4 : 8;
  const bool vec = d % vn == 0 && vec_ok(d_x, ldx, vn) && vec_ok(d_residual, ldr, vn) && vec_ok(d_w, 0, vn) &&
                   vec_ok(d_y, 0, vn) && vec_ok(d_h, 0, vn);
  FwdArgs a{d_x, d_residual, d_w, d_y, d_h, d_rstd, d_scale, ldx, ldr, rows, d, w_dtype == FR_F32, eps, 1.f / (float)d};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == FR_F32) FR_HIP_CHECK((quant ? launch_fwd<float, true>(a, vec, s) : launch_fwd<float, false>(a, vec, s)));
  else FR_HIP_CHECK((quant ? launch_fwd<bf16_t, true>(a, vec, s) : launch_fwd<bf16_t, false>(a, vec, s)));
  return FR_OK;
}

extern "C" int64_t fr_rms_norm_bwd_workspace(int64_t rows, int d) {
  return d < 1 || rows < 1 ? 256 : std::min<int64_t>(rows, kBwdBlocks) * d * 4 + 256;
}

extern "C" int fr_rms_norm_bwd(const void* d_dy, int64_t lddy, const void* d_dh, int64_t lddh, const void* d_h,
                               int64_t ldh, const void* d_residual, int64_t ldr, int64_t rows, int d, int dtype,
                               const void* d_w, int w_dtype, const float* d_rstd, void* d_dx, void* d_dw,
                               void* d_workspace, int64_t workspace_bytes, void* stream) {
  FR_REQUIRE(dtype == FR_F32 || dtype == FR_BF16, "dtype must be FR_F32 or FR_BF16");
  FR_REQUIRE(w_dtype == FR_F32 || w_dtype == dtype, "the weight is fp32 or of the rows' type");
  FR_REQUIRE(d >= 1 && d <= kMaxD, "d must be in [1, 8192]");
  FR_REQUIRE(rows >= 1 && rows < ((int64_t)1 << 31) && lddy >= d && ldh >= d && (!d_dh || lddh >= d) &&
                 (!d_residual || ldr >= d), "bad shape");
  FR_REQUIRE(d_dy && d_h && d_rstd && (d_dx || d_dw), "null pointer");
  FR_REQUIRE(!d_dw || (d_workspace && fr::aligned16(d_workspace) &&
                       workspace_bytes >= fr_rms_norm_bwd_workspace(rows, d)), "workspace too small");
  const int vn = dtype == FR_F32 ? 4 : 8;
  const bool vec = d % vn == 0 && vec_ok(d_dy, lddy, vn) && vec_ok(d_dh, lddh, vn) && vec_ok(d_h, ldh, vn) &&
                   vec_ok(d_residual, ldr, vn) && vec_ok(d_w, 0, vn) && vec_ok(d_dx, 0, vn);
  BwdArgs a{d_dy, d_dh, d_h, d_residual, d_w, d_rstd, d_dx, nullptr, lddy, lddh, ldh, ldr, rows, d,
            w_dtype == FR_F32, 1.f / (float)d};
  float* part = d_dw ? static_cast<float*>(d_workspace) : nullptr;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  FR_HIP_CHECK(dtype == FR_F32 ? launch_bwd<float>(a, vec, part, d_dw, s) : launch_bwd<bf16_t>(a, vec, part, d_dw, s));
  return FR_OK;
}
