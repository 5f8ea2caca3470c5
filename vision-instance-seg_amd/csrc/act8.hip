// 8-bit activation checkpoints (the format: act8.h): written from a tensor, read back, and the
// exact GELU that keeps its input in them.
//
// One pass over the data each, a chunk a thread: loads, ~20-40 vector instructions an element and
// stores, bound by memory.  Measured (a copy of 1 GiB runs at 5.15 TB/s): 262144 x 384 bf16, written
// in 52 us (5.9 TB/s: part of it stays in the last-level cache) and read back in 49;  65536 x 2048
// bf16, GELU forward 107 us (6.3 TB/s), backward 114-122 (5.9-5.5), with the activation again 160
// (5.9);  32768 x 2048 f32 (with the reciprocal's correction, act8.h; the same without), 105, 106 and
// 160;  50021 x 201 f32, written in 9.1 us and read back in 11.2 (4.6).  Two or four chunks a thread,
// all loaded before the first use, were no faster (GELU backward 122, 123 us where one took 114).
#include "act8.h"

namespace vs {
namespace {

constexpr int kThreads = 256;

// chunk g of a tensor of P / 8 chunks a row: its row and its place there.  FLAT (contiguous rows of
// a multiple of 32 features): chunk g is features 8 g.. of the whole buffer, with no division
// and no row ends to look for.
struct Place {
  long long row;
  int j;
};
__device__ __forceinline__ Place place_of(long long g, int cpr) {
  const uint32_t r = (uint32_t)g / (uint32_t)cpr;              // (fewer than 2^32 chunks)
  return {(long long)r, (int)((uint32_t)g - r * (uint32_t)cpr)};
}

template <typename T, bool FLAT>
__device__ __forceinline__ void load_at(Chunk<T>& c, const T* p, long long ld, long long g, const Place& pl, int C) {
  if (FLAT)
    c.load(p + 8 * g);
  else
    load_row_chunk(c, p + pl.row * ld, pl.j, C);
}
template <typename T, bool FLAT>
__device__ __forceinline__ void store_at(const Chunk<T>& c, T* p, long long g, const Place& pl, int C) {
  if (FLAT)
    c.store(p + 8 * g);
  else
    store_row_chunk(c, p + pl.row * C, pl.j, C);
}

// MODE 0: x -> q, scale.  1: x -> y = gelu(x), q, scale (q null: y only).
template <typename T, int MODE, bool FLAT>
__global__ void __launch_bounds__(kThreads) act8_fwd_kernel(const T* __restrict__ x, long long ld, T* __restrict__ y,
                                                            unsigned char* __restrict__ q,
                                                            unsigned char* __restrict__ scale, long long chunks,
                                                            int C, int cpr) {
  const long long g = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (g >= chunks) return;                       // (chunks is a multiple of 4: quads leave whole)
  Place pl = {};
  if (!FLAT) pl = place_of(g, cpr);
  Chunk<T> c;
  load_at<T, FLAT>(c, x, ld, g, pl, C);
  float v[8];
  c.unpack(v);
  if (MODE == 0 || q) {
    uint32_t sb;
    *reinterpret_cast<uint2*>(q + 8 * g) = pack_chunk(v, sb);
    if ((threadIdx.x & 3) == 0) scale[g >> 2] = (unsigned char)sb;
  }
  if (MODE == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu_value<T>(v[i]);
    c.pack(v);
    store_at<T, FLAT>(c, y, g, pl, C);
  }
}

// MODE 0: q, scale -> y (the values).  1: gy, q, scale -> gx = gy gelu'(h) (and y = gelu(h)).
template <typename T, int MODE, bool FLAT>
__global__ void __launch_bounds__(kThreads) act8_bwd_kernel(const T* __restrict__ gy, const unsigned char* __restrict__ q,
                                                            const unsigned char* __restrict__ scale,
                                                            T* __restrict__ gx, T* __restrict__ y, long long chunks,
                                                            int C, int cpr) {
  const long long g = (long long)blockIdx.x * kThreads + threadIdx.x;
  if (g >= chunks) return;
  const uint2 b = *reinterpret_cast<const uint2*>(q + 8 * g);
  const uint32_t sb = scale[g >> 2];
  Place pl = {};
  if (!FLAT) pl = place_of(g, cpr);
  Chunk<T> c;
  float h[8];
  if (MODE == 0) {
    unpack_chunk(b, sb, h);
    c.pack(h);
    store_at<T, FLAT>(c, y, g, pl, C);
    return;
  }
  load_at<T, FLAT>(c, gy, C, g, pl, C);
  unpack_chunk(b, sb, h);
  float d[8];
  c.unpack(d);
  if (y) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float slope;
      gelu_both<T>(h[i], h[i], slope);
      d[i] *= slope;
    }
    c.pack(h);
    store_at<T, FLAT>(c, y, g, pl, C);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] *= gelu_slope<T>(h[i]);
  }
  c.pack(d);
  store_at<T, FLAT>(c, gx, g, pl, C);
}

}  // namespace
}  // namespace vs

using namespace vs;

namespace {

int check_tensor(const char* who, int dtype, long long rows, int features, const void* q, long long& chunks,
                 long long& groups) {
  auto no = [who](const char* msg) {
    set_error(std::string(who) + ": " + msg);
    return VS_ERR_INVALID;
  };
  if (dtype != VS_F32 && dtype != VS_BF16) return no("dtype must be VS_F32 or VS_BF16");
  if (rows < 0 || features < 0 || features > (1 << 30)) return no("rows >= 0, 0 <= features <= 2^30");
  if (((uintptr_t)q & 7) != 0) return no("q must be 8-B aligned");
  const int cpr = padded32(features) / 8;
  // a launch has fewer than 2^32 threads, whole workgroups of them
  if (cpr && rows > ((1ll << 32) - kThreads) / cpr) return no("tensor too large (2^35 elements with the padding)");
  chunks = rows * cpr;
  groups = (chunks + kThreads - 1) / kThreads;
  return VS_OK;
}

template <typename T, int MODE>
void launch_fwd(bool flat, long long groups, hipStream_t st, const void* x, long long ld, void* y, void* q,
                void* scale, long long chunks, int C) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(kThreads), 0, st, (const T*)x, ld, (T*)y,
                       (unsigned char*)q, (unsigned char*)scale, chunks, C, padded32(C) / 8);
  };
  if (flat)
    go(act8_fwd_kernel<T, MODE, true>);
  else
    go(act8_fwd_kernel<T, MODE, false>);
}

template <typename T, int MODE>
void launch_bwd(bool flat, long long groups, hipStream_t st, const void* gy, const void* q, const void* scale,
                void* gx, void* y, long long chunks, int C) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(kThreads), 0, st, (const T*)gy, (const unsigned char*)q,
                       (const unsigned char*)scale, (T*)gx, (T*)y, chunks, C, padded32(C) / 8);
  };
  if (flat)
    go(act8_bwd_kernel<T, MODE, true>);
  else
    go(act8_bwd_kernel<T, MODE, false>);
}

}  // namespace

extern "C" int vs_act8_pack(int dtype, const void* x, long long ld_x, void* q, void* scale, long long rows,
                            int features, void* stream) {
  long long chunks, groups;
  const int rc = check_tensor(__func__, dtype, rows, features, q, chunks, groups);
  if (rc != VS_OK || chunks == 0) return rc;
  VS_CHECK(x && q && scale, "null pointer");
  VS_CHECK(ld_x >= 0, "row stride >= 0");
  const bool flat = features % kBlock == 0 && ld_x == features;
  if (dtype == VS_BF16)
    launch_fwd<bf16, 0>(flat, groups, (hipStream_t)stream, x, ld_x, nullptr, q, scale, chunks, features);
  else
    launch_fwd<float, 0>(flat, groups, (hipStream_t)stream, x, ld_x, nullptr, q, scale, chunks, features);
  VS_LAUNCH_CHECK();
  return VS_OK;
}

extern "C" int vs_act8_unpack(int dtype, const void* q, const void* scale, void* y, long long rows, int features,
                              void* stream) {
  long long chunks, groups;
  const int rc = check_tensor(__func__, dtype, rows, features, q, chunks, groups);
  if (rc != VS_OK || chunks == 0) return rc;
  VS_CHECK(q && scale && y, "null pointer");
  const bool flat = features % kBlock == 0;
  if (dtype == VS_BF16)
    launch_bwd<bf16, 0>(flat, groups, (hipStream_t)stream, nullptr, q, scale, nullptr, y, chunks, features);
  else
    launch_bwd<float, 0>(flat, groups, (hipStream_t)stream, nullptr, q, scale, nullptr, y, chunks, features);
  VS_LAUNCH_CHECK();
  return VS_OK;
}

extern "C" int vs_act8_gelu_forward(int dtype, const void* x, void* y, void* q, void* scale, long long rows,
                                    int features, void* stream) {
  long long chunks, groups;
  const int rc = check_tensor(__func__, dtype, rows, features, q, chunks, groups);
  if (rc != VS_OK || chunks == 0) return rc;
  VS_CHECK(x && y && (!q == !scale), "null pointer (q and scale: both or neither)");
  const bool flat = features % kBlock == 0;
  if (dtype == VS_BF16)
    launch_fwd<bf16, 1>(flat, groups, (hipStream_t)stream, x, features, y, q, scale, chunks, features);
  else
    launch_fwd<float, 1>(flat, groups, (hipStream_t)stream, x, features, y, q, scale, chunks, features);
  VS_LAUNCH_CHECK();
  return VS_OK;
}

extern "C" int vs_act8_gelu_backward(int dtype, const void* gy, const void* q, const void* scale, void* gx, void* y,
                                     long long rows, int features, void* stream) {
  long long chunks, groups;
  const int rc = check_tensor(__func__, dtype, rows, features, q, chunks, groups);
  if (rc != VS_OK || chunks == 0) return rc;
  VS_CHECK(gy && q && scale && gx, "null pointer");
  const bool flat = features % kBlock == 0;
  if (dtype == VS_BF16)
    launch_bwd<bf16, 1>(flat, groups, (hipStream_t)stream, gy, q, scale, gx, y, chunks, features);
  else
    launch_bwd<float, 1>(flat, groups, (hipStream_t)stream, gy, q, scale, gx, y, chunks, features);
  VS_LAUNCH_CHECK();
  return VS_OK;
}
