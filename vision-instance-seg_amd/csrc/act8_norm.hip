// LayerNorm over the last dim of [M, C] rows that keeps its input in 8 bits (act8.h): forward
// y = (x - mean) rstd w + b (of x, or of s = x + r rounded to the storage type and written out),
// backward from the checkpoint of the input, mean and rstd:
//     xh = (h - mean) rstd (h: what the checkpoint stands for),  g = dy w
//     dx = rstd (g - <g>_C - xh <g xh>_C) (+ ds),  dw = sum_rows dy xh,  db = sum_rows dy
// (mean and rstd are the uncompressed row's, so the checkpoint's error enters through xh alone).
//
// Bound by memory: one read and one write an element.  A row belongs to a GROUP of G lanes and
// every lane owns K chunks of it (chunk = lane + k G: an aligned quad of lanes holds a block of
// the checkpoint), so that a wave carries 64 / G rows, the row stays in registers between the
// statistics and the result, and the sums over a row are exchanges inside the group.  Rows of
// more than 2048 features take the whole workgroup (G = 256, one exchange through LDS).
// Statistics are f32, the variance in a second pass over the registers.
//
// Measured: 589824 x 192 bf16 with the residual, forward 197 us (5.2 TB/s), backward 166 (4.8) + 5 for
// the sum, in the window layout the same;  65536 x 768 bf16, 49 (5.2) and 49 + 4 (5.2);  4099 x 1003
// f32, 14 (2.7) and 18 + 4 (2.1: four waves a CU ask for a row, wait for it and store before they ask for
// the next), with the residual 17 (4.1) and 16.5 + 4 (3.2).
//
// dw / db: summed by every lane over the rows it sweeps, over the workgroup's groups in LDS,
// written as one f32 row a workgroup and added up by a second kernel: a fixed order, no atomics.
#include <type_traits>

#include "act8.h"

namespace vs {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxFeatures = 8192;
constexpr int kMaxParts = 1024;                  // workgroups of a backward sweep
constexpr int kCus = 256;

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// sum over the G lanes of a group, in all of them
template <int G>
__device__ __forceinline__ float group_sum(float x, float* lds) {
  x = dpp_add<0xB1>(x);                          // the quad
  x = dpp_add<0x4E>(x);
  if constexpr (G >= 8) x = dpp_add<0x141>(x);   // the row's halves mirrored: 8 lanes
  if constexpr (G >= 16) x = dpp_add<0x140>(x);  // the row mirrored: 16 lanes
  if constexpr (G >= 32) x += __shfl_xor(x, 16);
  if constexpr (G >= 64) x += __shfl_xor(x, 32);
  if constexpr (G == 256) {                      // four waves; every thread of the workgroup gets here
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
  return x;
}

template <typename T, int G, int K, bool RES>
__global__ void __launch_bounds__(kThreads) act8_ln_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ r, const T* __restrict__ w, const T* __restrict__ b,
    T* __restrict__ s_out, T* __restrict__ y, unsigned char* __restrict__ q, unsigned char* __restrict__ scale,
    float* __restrict__ mean, float* __restrict__ rstd, long long M, int C, float eps,
    const int* __restrict__ yrows, long long ycount) {
  __shared__ float lds[4];
  constexpr int R = kThreads / G;                // rows of a workgroup at a time
  const int lane = threadIdx.x & (G - 1), cpr = padded32(C) >> 3;
  const float inv_c = 1.f / (float)C;
  float wv[K][8], bv[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Chunk<T> c;
    load_row_chunk(c, w, lane + k * G, C);
    c.unpack(wv[k]);
    load_row_chunk(c, b, lane + k * G, C);
    c.unpack(bv[k]);
  }
  // whole groups enter and leave the loop together (a workgroup of G = 256 as one)
  for (long long row = (long long)blockIdx.x * R + threadIdx.x / G; row < M; row += (long long)gridDim.x * R) {
    Chunk<T> xc[K];
    float v[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) load_row_chunk(xc[k], x + row * C, lane + k * G, C);
    if constexpr (RES) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        Chunk<T> rc;
        float a[8], c[8];
        load_row_chunk(rc, r + row * C, lane + k * G, C);
        xc[k].unpack(a);
        rc.unpack(c);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] += c[i];
        xc[k].pack(a);
        store_row_chunk(xc[k], s_out + row * C, lane + k * G, C);
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      xc[k].unpack(v[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[k][i];
    }
    const float mu = group_sum<G>(sum, lds) * inv_c;
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int n = C - 8 * (lane + k * G);      // features of this chunk inside the row
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = v[k][i] - mu;
        sq += i < n ? d * d : 0.f;
      }
    }
    const float rs = 1.f / sqrtf(group_sum<G>(sq, lds) * inv_c + eps);
    const long long yr = yrows ? (long long)yrows[row] : row;
    const bool yin = yr >= 0 && yr < ycount;     // a row map that points outside y writes nothing
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = lane + k * G;
      if (q) {
        uint32_t sb;
        const uint2 c = pack_chunk(v[k], sb);
        if (j < cpr) {
          *reinterpret_cast<uint2*>(q + (row * cpr + j) * 8) = c;
          if ((lane & 3) == 0) scale[(row * cpr + j) >> 2] = (unsigned char)sb;
        }
      }
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf((v[k][i] - mu) * rs, wv[k][i], bv[k][i]);
      Chunk<T> c;
      c.pack(o);
      if (yin) store_row_chunk(c, y + yr * C, j, C);
    }
    if (lane == 0) {
      mean[row] = mu;
      rstd[row] = rs;
    }
  }
}

// part [gridDim.x][2][C]: the workgroup's dw, db
template <typename T, int G, int K, bool RES>
__global__ void __launch_bounds__(kThreads) act8_ln_bwd_kernel(
    const T* __restrict__ gy, const T* __restrict__ gs, const unsigned char* __restrict__ q,
    const unsigned char* __restrict__ scale, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* __restrict__ gx, float* __restrict__ part, long long M, int C,
    const int* __restrict__ grows, long long gcount) {
  constexpr int R = kThreads / G;
  // the groups' sums, eight features of one chunk slot at a time: [R][2][G][8]
  __shared__ float lds[R * 2 * G * 8];
  const int lane = threadIdx.x & (G - 1), grp = threadIdx.x / G, cpr = padded32(C) >> 3;
  const float inv_c = 1.f / (float)C;
  float wv[K][8], aw[K][8], ab[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Chunk<T> c;
    load_row_chunk(c, w, lane + k * G, C);
    c.unpack(wv[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) aw[k][i] = ab[k][i] = 0.f;
  }
  for (long long row = (long long)blockIdx.x * R + grp; row < M; row += (long long)gridDim.x * R) {
    const long long gr = grows ? (long long)grows[row] : row;
    const bool gin = gr >= 0 && gr < gcount;     // a row map that points outside gy reads zeros
    const float mu = mean[row], rs = rstd[row];
    Chunk<T> gc[K], sc[RES ? K : 1];
    uint2 b[K];
    uint32_t sb[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int j = lane + k * G;
      if (gin)
        load_row_chunk(gc[k], gy + gr * C, j, C);
      else
        gc[k].zero();
      if constexpr (RES) load_row_chunk(sc[k], gs + row * C, j, C);
      b[k] = make_uint2(0u, 0u);
      sb[k] = 1u;
      if (j < cpr) {
        b[k] = *reinterpret_cast<const uint2*>(q + (row * cpr + j) * 8);
        sb[k] = scale[(row * cpr + j) >> 2];
      }
    }
    // behind the row gy and w are 0, so that nothing there reaches a sum
    float c1 = 0.f, c2 = 0.f;
    float xh[K][8], g[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      unpack_chunk(b[k], sb[k], xh[k]);
      gc[k].unpack(g[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        xh[k][i] = (xh[k][i] - mu) * rs;
        aw[k][i] = fmaf(g[k][i], xh[k][i], aw[k][i]);
        ab[k][i] += g[k][i];
        g[k][i] *= wv[k][i];
        c1 += g[k][i];
        c2 = fmaf(g[k][i], xh[k][i], c2);
      }
    }
    c1 = group_sum<G>(c1, lds) * inv_c;
    c2 = group_sum<G>(c2, lds) * inv_c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float o[8], d[8];
      if constexpr (RES) sc[k].unpack(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[i] = rs * (g[k][i] - c1 - xh[k][i] * c2);
        if constexpr (RES) o[i] += d[i];
      }
      Chunk<T> c;
      c.pack(o);
      store_row_chunk(c, gx + row * C, lane + k * G, C);
    }
  }
  // the workgroup's row of partials: its R groups in order
#pragma unroll
  for (int k = 0; k < K; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lds[((grp * 2 + 0) * G + lane) * 8 + i] = aw[k][i];
      lds[((grp * 2 + 1) * G + lane) * 8 + i] = ab[k][i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * G * 8; e += kThreads) {
      const int which = e / (G * 8), c = k * G * 8 + (e & (G * 8 - 1));
      if (c >= C) continue;
      float s = 0.f;
#pragma unroll 4
      for (int p = 0; p < R; ++p) s += lds[(p * 2 + which) * G * 8 + (e & (G * 8 - 1))];
      part[((long long)blockIdx.x * 2 + which) * C + c] = s;
    }
  }
}

// dw / db [C] = the column sums of part [P][2 C]: 32 columns x 32 interleaved slices of the rows
// a workgroup, the slices added in order
template <typename T>
__global__ void __launch_bounds__(1024) act8_ln_sum_kernel(const float* __restrict__ part, T* __restrict__ dw,
                                                           T* __restrict__ db, int P, int C) {
  __shared__ float lds[32][33];
  const int cx = threadIdx.x & 31, sl = threadIdx.x >> 5;
  const long long col = (long long)blockIdx.x * 32 + cx, n = 2ll * C;
  float s = 0.f;
  if (col < n)
#pragma unroll 8
    for (int p = sl; p < P; p += 32) s += part[p * n + col];
  lds[sl][cx] = s;
  __syncthreads();
  if (sl == 0 && col < n) {
    float t = 0.f;
#pragma unroll
    for (int p = 0; p < 32; ++p) t += lds[p][cx];
    if (col < C)
      dw[col] = from_f32<T>(t);
    else
      db[col - C] = from_f32<T>(t);
  }
}

// calls go(G, K) (integral constants) for the lanes a row and chunks a lane of C features: the
// fewest lanes (4, 8, ... 64) that hold the row in at most three chunks each -- 96, 192, 384, ...
// features then fill every lane -- else up to four, else the workgroup.  (Forward / backward us with
// at most three, two, one chunk a lane: 589824 x 192 with the residual 203 / 158, 208 / 179, 229 /
// 156;  65536 x 768 41 / 51, 43 / 51, 90 / 84.)
template <typename F>
void with_shape(int C, F&& go) {
  using std::integral_constant;
  const int n = padded32(C) / 8;
#define VS_G(g)                                                                                   \
  if (n <= 3 * g) {                                                                               \
    if (n <= g) return go(integral_constant<int, g>{}, integral_constant<int, 1>{});              \
    if (n <= 2 * g) return go(integral_constant<int, g>{}, integral_constant<int, 2>{});          \
    return go(integral_constant<int, g>{}, integral_constant<int, 3>{});                          \
  }
  VS_G(4) VS_G(8) VS_G(16) VS_G(32) VS_G(64)
#undef VS_G
  if (n <= 4 * 64) return go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  if (n <= 2 * 256) return go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  return go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
}

int rows_at_a_time(int C) {
  int r = 1;
  with_shape(C, [&](auto g, auto) { r = kThreads / decltype(g)::value; });
  return r;
}

// workgroups of the backward sweep: one a CU before any sweeps twice, then at least four sweeps each
// (a workgroup's partial row costs as much traffic as two rows of f32: at 4099 x 1003 f32, 1024
// workgroups took 14.9 + 12.0 us, sweep and sum, 257 take 14.2 + 4.6)
int parts_of(long long M, int C) {
  const long long g = (M + rows_at_a_time(C) - 1) / rows_at_a_time(C);
  if (g <= kCus) return (int)(g < 1 ? 1 : g);
  return (int)(g / 4 < kCus ? kCus : g / 4 > kMaxParts ? kMaxParts : g / 4);
}

}  // namespace
}  // namespace vs

using namespace vs;

#define ACT8_NORM_CHECKS()                                                                       \
  VS_CHECK(dtype == VS_F32 || dtype == VS_BF16, "dtype must be VS_F32 or VS_BF16");              \
  VS_CHECK(rows >= 0 && rows < (1ll << 31), "0 <= rows < 2^31");                                 \
  VS_CHECK(features > 0 && features <= kMaxFeatures, "0 < features <= 8192")

extern "C" int vs_act8_layer_norm_forward(int dtype, const void* x, const void* r, const void* w, const void* b,
                                          void* s, void* y, void* q, void* scale, float* mean, float* rstd,
                                          long long rows, int features, float eps, const int* y_rows,
                                          long long y_count, void* stream) {
  ACT8_NORM_CHECKS();
  if (rows == 0) return VS_OK;
  VS_CHECK(x && w && b && y && mean && rstd && (!r == !s) && (!q == !scale),
           "null pointer (r and s, q and scale: both or neither)");
  VS_CHECK(((uintptr_t)q & 7) == 0, "q must be 8-B aligned");
  hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto tag, auto res) {
    using T = decltype(tag);
    constexpr bool RES = decltype(res)::value;
    with_shape(features, [&](auto g, auto k) {
      constexpr int G = decltype(g)::value, K = decltype(k)::value, R = kThreads / G;
      const int grid = grid_for(rows, R, 256 * 8);
      hipLaunchKernelGGL((act8_ln_fwd_kernel<T, G, K, RES>), dim3(grid), dim3(kThreads), 0, st, (const T*)x,
                         (const T*)r, (const T*)w, (const T*)b, (T*)s, (T*)y, (unsigned char*)q,
                         (unsigned char*)scale, mean, rstd, rows, features, eps, y_rows,
                         y_rows ? y_count : rows);
    });
  };
  if (dtype == VS_BF16)
    r ? launch(bf16{}, std::true_type{}) : launch(bf16{}, std::false_type{});
  else
    r ? launch(0.f, std::true_type{}) : launch(0.f, std::false_type{});
  VS_LAUNCH_CHECK();
  return VS_OK;
}

extern "C" long long vs_act8_layer_norm_backward_workspace_bytes(long long rows, int features) {
  if (rows < 0 || features <= 0 || features > kMaxFeatures) return 0;
  return (long long)parts_of(rows, features) * 2 * features * 4;
}

extern "C" int vs_act8_layer_norm_backward(int dtype, const void* gy, const void* gs, const void* q,
                                           const void* scale, const void* w, const float* mean, const float* rstd,
                                           void* gx, void* gw, void* gb, void* workspace, long long rows,
                                           int features, const int* gy_rows, long long gy_count, void* stream) {
  ACT8_NORM_CHECKS();
  VS_CHECK(w && gw && gb && workspace && (rows == 0 || (gy && q && scale && mean && rstd && gx)), "null pointer");
  VS_CHECK(((uintptr_t)q & 7) == 0, "q must be 8-B aligned");
  VS_CHECK(((uintptr_t)workspace & 3) == 0, "workspace must be 4-B aligned");
  hipStream_t st = (hipStream_t)stream;
  const int parts = parts_of(rows, features);
  float* part = (float*)workspace;
  auto launch = [&](auto tag, auto res) {
    using T = decltype(tag);
    constexpr bool RES = decltype(res)::value;
    with_shape(features, [&](auto g, auto k) {
      constexpr int G = decltype(g)::value, K = decltype(k)::value;
      hipLaunchKernelGGL((act8_ln_bwd_kernel<T, G, K, RES>), dim3(parts), dim3(kThreads), 0, st, (const T*)gy,
                         (const T*)gs, (const unsigned char*)q, (const unsigned char*)scale, (const T*)w, mean, rstd,
                         (T*)gx, part, rows, features, gy_rows, gy_rows ? gy_count : rows);
    });
    hipLaunchKernelGGL((act8_ln_sum_kernel<T>), dim3((2 * features + 31) / 32), dim3(1024), 0, st,
                       (const float*)part, (T*)gw, (T*)gb, parts, features);
  };
  if (dtype == VS_BF16)
    gs ? launch(bf16{}, std::true_type{}) : launch(bf16{}, std::false_type{});
  else
    gs ? launch(0.f, std::true_type{}) : launch(0.f, std::false_type{});
  VS_LAUNCH_CHECK();
  return VS_OK;
}
