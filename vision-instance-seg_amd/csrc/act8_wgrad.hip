// Weight and bias gradient of a Linear whose input was kept as an 8-bit checkpoint (act8.h):
//     dW[o, i] = sum_t gY[t, o] h[t, i],   db[o] = sum_t gY[t, o],   h[t, i] = q[t, i] 2^e[t, i / 32]
//
// The reduction runs over tokens, the strided dimension of both operands: 64-token chunks are
// staged in LDS in their natural [token][feature] order (images of 128 columns, lds_dma.h) and
// read as MFMA operands with the transposing LDS read.  The checkpoint is widened to bf16 on its
// way into LDS, once a workgroup, exactly (act8.h).  f32 gradients are cut into three bf16 parts
// by truncation, gY = hi + mid + lo: 8 bits of significand each, so the sum is exact, and three
// matrix products give what an f32 product of exact terms would; a non-finite value is its hi
// part alone.  Accumulation is f32 in the matrix units.  db comes from one more MFMA an operand
// tile, with a first operand of ones, in the workgroups of the first input columns.
//
// A workgroup owns 128 output rows x 128 input columns of dW for one split of the tokens.  The
// next chunk is in flight in registers while one is multiplied; LDS holds two chunks.  Splits
// write f32 partials that a second kernel adds up in a fixed order (no atomics).
#include <type_traits>

#include "act8.h"
#include "lds_dma.h"

namespace vs {
namespace {

constexpr int kTK = 64;                          // tokens of a chunk
constexpr int kThreads = 256;
constexpr int kImg = kTK * 256;                  // bytes of an image: 64 tokens x 128 bf16

struct Wgrad8 {
  const void* gy;
  const unsigned char* q;
  const unsigned char* scale;
  void* dw;
  void* db;
  float* part;                                   // [S][tiles][128 * 128] in fragment order (S > 1)
  float* pbias;                                  // [S][N]
  long long ldg, T;
  int N, K, P;                                   // P: the checkpoint's pitch
  int S, tiles_i, tiles;
  int f32_out;
};

__device__ __forceinline__ void store_out(void* p, size_t i, bool f32, float v) {
  if (f32)
    reinterpret_cast<float*>(p)[i] = v;
  else
    reinterpret_cast<bf16*>(p)[i] = __float2bfloat16(v);
}

// the bf16 parts of 8 f32 values (truncation; see the head of the file)
__device__ __forceinline__ void split3(const float* v, uint4& hi, uint4& mid, uint4& lo) {
  uint32_t h[8], m[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(v[i]);
    const bool fin = (u & 0x7f800000u) != 0x7f800000u;
    h[i] = u & 0xffff0000u;
    const float r1 = fin ? v[i] - __uint_as_float(h[i]) : 0.f;
    m[i] = __float_as_uint(r1) & 0xffff0000u;
    l[i] = __float_as_uint(r1 - __uint_as_float(m[i]));
    if (!fin && (u & 0x7fffffu)) h[i] = 0x7fc00000u;          // a NaN whose payload is in the low bits
  }
  auto two = [](const uint32_t* w, int i) { return (w[i + 1] & 0xffff0000u) | (w[i] >> 16); };
  hi = make_uint4(two(h, 0), two(h, 2), two(h, 4), two(h, 6));
  mid = make_uint4(two(m, 0), two(m, 2), two(m, 4), two(m, 6));
  lo = make_uint4(two(l, 0), two(l, 2), two(l, 4), two(l, 6));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) act8_wgrad_kernel(const Wgrad8 a) {
  constexpr int NP = std::is_same<T, float>::value ? 3 : 1;   // parts of a gradient
  constexpr int kStage = (NP + 1) * kImg;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];       // two stages
  const int wg = xcd_swizzle(blockIdx.x, gridDim.x);
  const int s = wg / a.tiles, tile = wg - s * a.tiles;
  const int ob = tile / a.tiles_i, ib = tile - ob * a.tiles_i;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63, r = l & 31, hh = l >> 5;
  const int wo = (w & 1) * 64, wi = (w >> 1) * 64;            // this wave's 64 x 64
  const long long nchunk = (a.T + kTK - 1) / kTK;
  const long long cb = nchunk * s / a.S, ce = nchunk * (s + 1) / a.S;
  const bool do_bias = a.db != nullptr && ib == 0 && (w >> 1) == 0;
  const T* gy = reinterpret_cast<const T*>(a.gy);

  // a chunk's pieces of this thread: 4 x 8 gradients (row = piece * 16 + tid / 16, columns 8 (tid
  // & 15)..), 2 x 16 bytes of the checkpoint (row = piece * 32 + tid / 8, columns 16 (tid & 7)..)
  const int gc = 8 * (threadIdx.x & 15), gr = threadIdx.x >> 4;
  const int xc = 16 * (threadIdx.x & 7), xr = threadIdx.x >> 3;
  const int gcol = ob * 128 + gc, xcol = ib * 128 + xc;
  const bool xin = xcol < a.P;
  Chunk<T> g[4];
  uint4 xq[2];
  uint32_t xs[2];
  auto fetch = [&](long long c) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const long long t = c * kTK + p * 16 + gr;
      if (t < a.T)
        load_row_chunk(g[p], gy + t * a.ldg, gcol >> 3, a.N);
      else
        g[p].zero();
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const long long t = c * kTK + p * 32 + xr;
      xq[p] = make_uint4(0u, 0u, 0u, 0u);
      xs[p] = 1u;
      if (t < a.T && xin) {
        xq[p] = *reinterpret_cast<const uint4*>(a.q + t * a.P + xcol);
        xs[p] = a.scale[t * (a.P >> 5) + (xcol >> 5)];
      }
    }
  };
  auto put = [&](int st) {
    unsigned char* base = smem + st * kStage;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int at = woff(p * 16 + gr, gc >> 3);
      if constexpr (NP == 1) {
        *reinterpret_cast<uint4*>(base + at) = g[p].a;
      } else {
        float v[8];
        uint4 hi, mid, lo;
        g[p].unpack(v);
        split3(v, hi, mid, lo);
        *reinterpret_cast<uint4*>(base + at) = hi;
        *reinterpret_cast<uint4*>(base + kImg + at) = mid;
        *reinterpret_cast<uint4*>(base + 2 * kImg + at) = lo;
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint2 half[2] = {make_uint2(xq[p].x, xq[p].y), make_uint2(xq[p].z, xq[p].w)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        unpack_chunk(half[h], xs[p], v);
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)              // exact in bf16: the upper halves
          o[i] = __builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);
        *reinterpret_cast<uint4*>(base + NP * kImg + woff(p * 32 + xr, (xc >> 3) + h)) =
            make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  };

  f32x16_t acc[2][2], accb[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    zero16(accb[x]);
    zero16(acc[x][0]);
    zero16(acc[x][1]);
  }
  const short one = (short)0x3f80;               // bf16 1.0
  const bf16x8_t ones = {one, one, one, one, one, one, one, one};
  if (cb < ce) fetch(cb);
  for (long long c = cb; c < ce; ++c) {
    const int st = (int)(c - cb) & 1;
    put(st);
    __syncthreads();                             // stage st is whole; stage st ^ 1 was read before it
    if (c + 1 < ce) fetch(c + 1);
    const unsigned char* sg = smem + st * kStage;
    const unsigned char* sx = sg + NP * kImg;
#pragma unroll
    for (int k = 0; k < kTK / 16; ++k) {
      bf16x8_t xa[2];
#pragma unroll
      for (int ti = 0; ti < 2; ++ti) xa[ti] = tr_frag(sx, 16 * k, wi + 32 * ti, l);
#pragma unroll
      for (int to = 0; to < 2; ++to)
#pragma unroll
        for (int p = NP - 1; p >= 0; --p) {      // the smallest part first
          const bf16x8_t gb = tr_frag(sg + p * kImg, 16 * k, wo + 32 * to, l);
#pragma unroll
          for (int ti = 0; ti < 2; ++ti) acc[to][ti] = mfma16(xa[ti], gb, acc[to][ti]);
          if (do_bias) accb[to] = mfma16(ones, gb, accb[to]);
        }
    }
  }

  // C tile: lane column = o, registers 4 g.. = 4 consecutive i
  if (a.S > 1) {
    float* pw = a.part + ((size_t)s * a.tiles + tile) * (128 * 128) + (size_t)w * 4096 + l * 4;
#pragma unroll
    for (int to = 0; to < 2; ++to)
#pragma unroll
      for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq)
          *reinterpret_cast<float4*>(pw + ((to * 2 + ti) * 4 + gq) * 256) = make_float4(
              acc[to][ti][4 * gq], acc[to][ti][4 * gq + 1], acc[to][ti][4 * gq + 2], acc[to][ti][4 * gq + 3]);
  }
#pragma unroll
  for (int to = 0; to < 2; ++to) {
    const int o = ob * 128 + wo + 32 * to + r;
    if (o >= a.N) continue;
    if (a.S == 1) {
#pragma unroll
      for (int ti = 0; ti < 2; ++ti)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int i = ib * 128 + wi + 32 * ti + crow(e, hh);
          if (i < a.K) store_out(a.dw, (size_t)o * a.K + i, a.f32_out, acc[to][ti][e]);
        }
    }
    if (do_bias && hh == 0) {
      if (a.S > 1)
        a.pbias[(size_t)s * a.N + o] = accb[to][0];
      else
        store_out(a.db, o, a.f32_out, accb[to][0]);
    }
  }
}

// dW[o][i] = the splits' partials added in order; db likewise
__global__ void __launch_bounds__(kThreads) act8_wgrad_sum_kernel(const Wgrad8 a) {
  const long long at = (long long)blockIdx.x * kThreads + threadIdx.x, n = (long long)a.N * a.K;
  if (at < n) {
    const int o = (int)(at / a.K), i = (int)(at - (long long)o * a.K);
    const int oo = o & 127, ii = i & 127, row = ii & 31;
    const int wv = (oo >> 6) | ((ii >> 6) << 1), to = (oo >> 5) & 1, ti = (ii >> 5) & 1;
    const int lane = (oo & 31) + 32 * ((row >> 2) & 1), e = (row & 3) + 4 * (row >> 3);
    const float* p = a.part + ((size_t)(o >> 7) * a.tiles_i + (i >> 7)) * (128 * 128) + (size_t)wv * 4096 +
                     ((to * 2 + ti) * 4 + (e >> 2)) * 256 + lane * 4 + (e & 3);
    float v = 0.f;
    for (int s = 0; s < a.S; ++s) v += p[(size_t)s * a.tiles * (128 * 128)];
    store_out(a.dw, at, a.f32_out, v);
  } else if (a.db && at - n < a.N) {
    float v = 0.f;
    for (int s = 0; s < a.S; ++s) v += a.pbias[(size_t)s * a.N + (at - n)];
    store_out(a.db, at - n, a.f32_out, v);
  }
}

// splits of the tokens: enough workgroups for the chip, at least 4 chunks each
int splits_of(long long T, int N, int K) {
  const long long tiles = (long long)((N + 127) / 128) * ((K + 127) / 128);
  const long long nchunk = (T + kTK - 1) / kTK;
  long long s = (512 + tiles - 1) / tiles;
  if (s > nchunk / 4) s = nchunk / 4;
  return (int)(s < 1 ? 1 : s);
}

bool sizes_ok(long long T, int N, int K) {
  return T >= 0 && T < (1ll << 40) && N >= 0 && K >= 0 && N <= (1 << 24) && K <= (1 << 24) &&
         (long long)((N + 127) / 128) * ((K + 127) / 128) < (1 << 22);
}

}  // namespace
}  // namespace vs

using namespace vs;

extern "C" long long vs_act8_wgrad_workspace_bytes(long long tokens, int N, int K) {
  if (!sizes_ok(tokens, N, K) || N == 0 || K == 0) return 0;
  const long long S = splits_of(tokens, N, K);
  if (S == 1) return 0;
  const long long tiles = (long long)((N + 127) / 128) * ((K + 127) / 128);
  return 4 * S * (tiles * 128 * 128 + N);
}

extern "C" int vs_act8_wgrad(int dtype, int out_dtype, const void* gy, long long ld_gy, const void* q,
                             const void* scale, void* dw, void* db, void* workspace, long long tokens, int N, int K,
                             void* stream) {
  VS_CHECK((dtype == VS_F32 || dtype == VS_BF16) && (out_dtype == VS_F32 || out_dtype == VS_BF16),
           "dtypes must be VS_F32 or VS_BF16");
  VS_CHECK(sizes_ok(tokens, N, K), "sizes out of range");
  if (N == 0) return VS_OK;
  VS_CHECK(ld_gy >= 0, "row stride >= 0");
  VS_CHECK((K == 0 || dw) && (tokens == 0 || (gy && (K == 0 || (q && scale)))), "null pointer");
  VS_CHECK(((uintptr_t)q & 15) == 0, "q must be 16-B aligned");
  VS_CHECK(K > 0, "K > 0");
  Wgrad8 a;
  a.gy = gy;
  a.q = (const unsigned char*)q;
  a.scale = (const unsigned char*)scale;
  a.dw = dw;
  a.db = db;
  a.ldg = ld_gy;
  a.T = tokens;
  a.N = N;
  a.K = K;
  a.P = padded32(K);
  a.S = splits_of(tokens, N, K);
  a.tiles_i = (K + 127) / 128;
  a.tiles = ((N + 127) / 128) * a.tiles_i;
  a.f32_out = out_dtype == VS_F32;
  VS_CHECK(a.S == 1 || (workspace && ((uintptr_t)workspace & 15) == 0),
           "workspace: 16-B aligned, sized by vs_act8_wgrad_workspace_bytes");
  a.part = (float*)workspace;
  a.pbias = a.part + (size_t)a.S * a.tiles * (128 * 128);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(a.S * a.tiles));
  if (dtype == VS_BF16) {
    hipLaunchKernelGGL((act8_wgrad_kernel<bf16>), grid, dim3(kThreads), 4 * kImg, st, a);
  } else {
    // 128 KB of LDS: above the default limit of a launch
    VS_HIP(hipFuncSetAttribute((const void*)act8_wgrad_kernel<float>, hipFuncAttributeMaxDynamicSharedMemorySize,
                               8 * kImg));
    hipLaunchKernelGGL((act8_wgrad_kernel<float>), grid, dim3(kThreads), 8 * kImg, st, a);
  }
  VS_LAUNCH_CHECK();
  if (a.S > 1) {
    const long long items = (long long)N * K + (db ? N : 0);
    hipLaunchKernelGGL(act8_wgrad_sum_kernel, dim3((unsigned)((items + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                       st, a);
    VS_LAUNCH_CHECK();
  }
  return VS_OK;
}
