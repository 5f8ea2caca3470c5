// Weight and bias gradient of a Linear whose input was kept as an 8-bit checkpoint (act8.h):
//     dW[o, i] = sum_t gY[t, o] h[t, i],   db[o] = sum_t gY[t, o],   h[t, i] = q[t, i] 2^e[t, i / 32]
//
// The reduction runs over tokens, the strided dimension of both operands: 64-token chunks are
// staged in LDS in their natural [token][feature] order (images of 128 columns, padded row
// pitches: kPitchG, kPitchX) and read as MFMA operands with the transposing LDS read.  The
// checkpoint is widened to bf16 on its way into LDS, once a workgroup, exactly (act8.h).  f32
// gradients are cut into three bf16 parts by truncation, gY = hi + mid + lo: 8 bits of significand
// each, so that the sum is exact for |gY| >= 2^-110 (bf16's last bit is 2^-133, which the matrix
// units keep: below, what lies under it is cut, and a product is off by less than 2^-133 |h|), and
// three matrix products give what an f32 product of exact terms would; a non-finite value is its hi
// part alone.  Accumulation is f32 in the matrix units.  db is summed on the way into LDS, every
// workgroup of an output block its share of the chunks.
//
// A workgroup owns BO output rows x BI input columns of dW for one split of the tokens.  LDS holds
// two chunks: while chunk c is multiplied, chunk c + 1 goes from registers into LDS and chunk
// c + 2 from memory into the registers, piece by piece between the MFMAs; one barrier a chunk.
// Splits write f32 partials that a second kernel adds up in a fixed order (no atomics).
//
// What bounds it.  Vector arithmetic costs MFMA time almost in full (64 idle instructions more a
// chunk: 10 to 16 % more time), so the widening of the checkpoint, 2.5 instructions an element, is
// what an uncompressed operand would save; at the largest size below the matrix units are busy
// 64 to 67 % of the cycles and the clock falls from 1.8 to 1.5 GHz within four launches in a row.
// Measured on several cards (they differ by up to 15 %), tokens x outputs x inputs:  147456 x 1024 x
// 2048 bf16 530-610 us, 15 of it for the sum of the splits (1015-1165 TF/s; the library's 8192^3
// product 1475, its product at these sizes and layouts 570);  16384 x 1536 x 384 35-37 us, of it 7.6
// for the sum of 14 splits (33 MB of partials; the products alone are 13 us at the library's rate);
// 262144 x 96 x 384 43-50;  400 x 256 x 256 7 (seven chunks in a row);  f32 65536 x 768 x 768 206-250
// (310-375 TFLOP/s of the exact product, three times that of MFMA), 10007 x 299 x 203 19-22.
// Tried and slower: a ring of three 32-token chunks (637 us against 612 at the time), two or three
// chunks in flight in registers (the loads are not what it waits for; the first two asked for at once:
// no change), a 128 x 128 tile a wave (four waves of 256 x 256: spills), 32-token chunks of the
// smallest f32 tile with two workgroups a CU (10007 x 299 x 203: 20.5 us against 18.2).
#include <climits>
#include <type_traits>

#include "act8.h"
#include "lds_dma.h"

namespace vs {
namespace {

struct Wgrad8 {
  const void* gy;
  const unsigned char* q;
  const unsigned char* scale;
  void* dw;
  void* db;
  float* part;                                   // [S][tiles][BO * BI] in fragment order (S > 1)
  float* pbias;                                  // [S][tiles_i][N]
  long long ldg, T;
  int N, K, P;                                   // P: the checkpoint's pitch
  int S, tiles_i, tiles;
  int f32_out;
  int vec;                                       // dW's rows take 4-element stores
};

__device__ __forceinline__ void store_out(void* p, size_t i, bool f32, float v) {
  if (f32)
    reinterpret_cast<float*>(p)[i] = v;
  else
    reinterpret_cast<bf16*>(p)[i] = __float2bfloat16(v);
}

// dW[o, i .. i + 3], as far as it goes
__device__ __forceinline__ void store_four(const Wgrad8& a, int o, int i, float x, float y, float z, float w) {
  const size_t at = (size_t)o * a.K + i;
  if (a.vec && i < a.K) {                        // rows of a multiple of 4: i + 3 < K too
    if (a.f32_out)
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.dw) + at) = make_float4(x, y, z, w);
    else
      *reinterpret_cast<bf16x4_t*>(reinterpret_cast<bf16*>(a.dw) + at) =
          bf16x4_t{bf16_bits(x), bf16_bits(y), bf16_bits(z), bf16_bits(w)};
    return;
  }
  const float v[4] = {x, y, z, w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (i + e < a.K) store_out(a.dw, at + e, a.f32_out, v[e]);
}

// The bf16 parts of 8 f32 values (truncation; see the head of the file).  The rest of an infinity is
// taken as 0, so that it stays one; that of a NaN is a NaN, also where truncation makes its hi part an
// infinity.
__device__ __forceinline__ void split3(const float* v, uint4& hi, uint4& mid, uint4& lo) {
  float m[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float rest = __builtin_isinf(v[i]) ? 0.f : v[i] - __uint_as_float(__float_as_uint(v[i]) & 0xffff0000u);
    m[i] = rest;
    l[i] = rest - __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
  }
  auto two = [](const float* w, int i) {         // the upper halves of two values
    return __builtin_amdgcn_perm(__float_as_uint(w[i + 1]), __float_as_uint(w[i]), 0x07060302u);
  };
  hi = make_uint4(two(v, 0), two(v, 2), two(v, 4), two(v, 6));
  mid = make_uint4(two(m, 0), two(m, 2), two(m, 4), two(m, 6));
  lo = make_uint4(two(l, 0), two(l, 2), two(l, 4), two(l, 6));
}

__device__ __forceinline__ uint4 buffer16(__amdgpu_buffer_rsrc_t rs, int offset) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(rs, offset, 0, 0);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

typedef __attribute__((address_space(3))) unsigned char lds_byte;
__device__ __forceinline__ void lds16(lds_byte* p, uint4 a) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 v = {a.x, a.y, a.z, a.w};
  *(__attribute__((address_space(3))) u32x4*)p = v;
}

// LDS images of 128 columns of bf16, a row a token.  A transposing read takes four rows x 64 B at a
// time: the row pitches are chosen so that these lie in different banks (of 64 x 4 B) without an
// exclusive or in the address, whose steps -- columns, rows, parts -- are then immediate offsets of one
// register.  gY: 256 + 64 B.  h: a thread writes two neighbouring 16-B columns, 2 x and 2 x + 1, one
// after the other; the even columns are stored in front of the odd ones, so that eight lanes write
// 128 B of different banks, and the pitch is 256 + 32 B.
constexpr int kPitchG = 320, kPitchX = 288;
constexpr int images(int columns) { return (columns + 127) / 128; }

// How gY is loaded.  Rows: by address, each row and chunk checked against its end (any stride; the
// branches drain the loads in flight).  Dwords: buffer loads, of rows that begin on a dword.  Halves:
// buffer loads of the 20 B around a chunk of bf16, from the dword that its first value lies in, and a
// shift by 0 or 16 bits on the way into LDS (40001 x 1030 x 1030 bf16, row pitch 1030 / 1031 values:
// 130 / 139 us, by rows 238;  147456 x 1040 / 1039 x 2048 with db 683 / 745, without 676 / 727).
enum Feed { kRows, kDwords, kHalves };

// acc += h^T gY over the wave's TO x TI tiles of 32 x 32, chunk by chunk
template <typename T, int BO, int BI, int WO, int WI, int TK, int FEED>
__global__ void __launch_bounds__(64 * WO * WI) act8_wgrad_kernel(const Wgrad8 a) {
  constexpr int NP = std::is_same<T, float>::value ? 3 : 1;   // parts of a gradient
  constexpr int NT = 64 * WO * WI, TO = BO / WO / 32, TI = BI / WI / 32;
  constexpr int kImgG = TK * kPitchG, kImgX = TK * kPitchX;   // bytes of an image
  constexpr int NHO = images(BO), NHI = images(BI);           // images of a part of gY, of h
  constexpr int kStage = NP * NHO * kImgG + NHI * kImgX;
  constexpr int GC = BO / 8, XC = BI / 16;                    // pieces of a token: 8 gradients, 16 of q
  constexpr int GP = TK * GC / NT, XP = TK * XC / NT;         // pieces of a thread
  constexpr int KS = TK / 16;                                 // MFMA steps of a chunk
  static_assert(GP * NT == TK * GC && XP * NT == TK * XC && NT % GC == 0 && NT % (2 * XC) == 0, "whole pieces");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int wg = xcd_swizzle(blockIdx.x, gridDim.x);
  const int s = wg / a.tiles, tile = wg - s * a.tiles;        // a split's tiles are neighbours (one XCD's L2)
  const int ob = tile / a.tiles_i, ib = tile - ob * a.tiles_i;
  const int w = threadIdx.x >> 6, l = threadIdx.x & 63, r = l & 31, hh = l >> 5;
  const int qo = w % WO, qi = w / WO;
  const int wo = qo * (BO / WO), wi = qi * (BI / WI);
  const int nchunk = (int)((a.T + TK - 1) / TK);
  const int cb = (int)((long long)nchunk * s / a.S), ce = (int)((long long)nchunk * (s + 1) / a.S);

  const int gr = threadIdx.x / GC, gc = threadIdx.x % GC, xr = threadIdx.x / XC, xc = threadIdx.x % XC;
  const int gcol = ob * BO + gc * 8, xcol = ib * BI + xc * 16;
  Chunk<T> g[GP];
  uint32_t tail[FEED == kHalves ? GP : 1];       // the dword behind a chunk
  uint4 xq[XP];
  uint32_t xs[XP];
  // The next chunk to fetch: the three tensors from its first row on, and the rows left.  A buffer
  // load gives 0 behind the chunk's last row, which are the tokens behind the last one; columns
  // behind N or P hold whatever is there (the next row): they only reach rows and columns of dW
  // that do not exist.
  const long long cb_rows = (long long)cb * TK;
  const unsigned char* gbase = reinterpret_cast<const unsigned char*>(a.gy) + cb_rows * a.ldg * (long long)sizeof(T);
  const unsigned char* qbase = a.q + cb_rows * a.P;
  const unsigned char* sbase = a.scale + cb_rows * (a.P >> 5);
  const long long end = (long long)ce * TK;      // (behind the split's last chunk too: zeros)
  int left = (int)((end < a.T ? end : a.T) - cb_rows);
  const int gld = (int)(a.ldg * (long long)sizeof(T)), sld = a.P >> 5;        // (gld: the buffer loads')
  // kHalves: where gbase lies in its dword -- in every chunk, TK rows on, the same -- and a thread's
  // chunks in theirs: its rows are an even number apart
  static_assert(FEED != kHalves || (sizeof(T) == 2 && (NT / GC) % 2 == 0 && TK % 2 == 0), "one shift a thread");
  const int odd = FEED == kHalves ? (int)(reinterpret_cast<uintptr_t>(gbase) & 2) : 0;
  gbase -= odd;
  const int gbyte = odd + gr * gld + gcol * (int)sizeof(T), gshift = (gbyte & 2) * 8;
  const int goff = FEED == kHalves ? gbyte & ~3 : gbyte;
  const int xoff = xr * a.P + xcol, soff = xr * sld + (xcol >> 5);
  const int gap = gld - odd - a.N * (int)sizeof(T) - 3;      // (rows gld - gap) & ~3: to the last row's last dword
  // the chunk's bytes (readfirstlane: buffer descriptors live in scalar registers)
  int gsize, qsize, ssize;
  auto size_up = [&]() {
    const int rows = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : left < TK ? left : TK);
    gsize = __builtin_amdgcn_readfirstlane(rows > 0 ? (rows * gld - gap) & ~3 : 0);
    qsize = rows * a.P;
    ssize = rows * sld;
  };
  size_up();
  auto fetch_g = [&](int p) {
    if constexpr (FEED != kRows) {
      const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)gbase, 0, gsize, 0x00020000);
      int at = goff + p * (NT / GC) * gld;
      // (the row behind the last one can begin in the last one's last dword)
      if constexpr (FEED == kHalves) at = p * (NT / GC) < left - gr ? at : INT_MIN;
      g[p].a = buffer16(rs, at);
      if constexpr (FEED == kHalves) tail[p] = __builtin_amdgcn_raw_buffer_load_b32(rs, at + 16, 0, 0);
      if constexpr (NP == 3) g[p].b = buffer16(rs, at + 16);
    } else {
      const int row = p * (NT / GC) + gr;
      if (row < left)
        load_row_chunk(g[p], reinterpret_cast<const T*>(gbase) + row * a.ldg, gcol >> 3, a.N);
      else
        g[p].zero();
    }
  };
  auto fetch_x = [&](int p) {
    const auto rq = __builtin_amdgcn_make_buffer_rsrc((void*)qbase, 0, qsize, 0x00020000);
    const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)sbase, 0, ssize, 0x00020000);
    xq[p] = buffer16(rq, xoff + p * (NT / XC) * a.P);
    xs[p] = __builtin_amdgcn_raw_buffer_load_b8(rs, soff + p * (NT / XC) * sld, 0, 0);
  };
  auto advance = [&]() {
    gbase += TK * a.ldg * (long long)sizeof(T);
    qbase += (long long)TK * a.P;
    sbase += (long long)TK * sld;
    left -= TK;
    size_up();
  };
  // LDS addresses, all of the current stage: this thread's pieces and its wave's operands.  An operand
  // of 16 tokens x 32 columns is two transposing reads: rows 8 hh + (l & 15) / 4 and four rows on,
  // columns (l & 16) + 4 (l & 3)..
  typedef __attribute__((address_space(3))) bf16x4v_t lds_v4;
  lds_byte* const base = (lds_byte*)smem;
  lds_byte* at_g = base + (gc >> 4) * kImgG + gr * kPitchG + (gc & 15) * 16;
  lds_byte* at_x = base + NP * NHO * kImgG + (xc >> 3) * kImgX + xr * kPitchX + (xc & 7) * 16;
  const int orow = 8 * hh + ((l & 15) >> 2);
  lds_byte* at_b = base + (wo >> 7) * kImgG + orow * kPitchG + ((wo & 127) + (l & 16) + 4 * (l & 3)) * 2;
  lds_byte* at_a = base + NP * NHO * kImgG + (wi >> 7) * kImgX + orow * kPitchX + (wi & 127) + (l & 16) +
                   ((l & 2) >> 1) * 128 + (l & 1) * 8;
  static_assert(BO / WO <= 128 && BI / WI <= 128 && 128 % (BO / WO) == 0 && 128 % (BI / WI) == 0,
                "a wave's operands lie in one image");
  // db: this thread's columns of gY, summed as they pass.  The workgroups of an output block share a
  // split's chunks, this one's are [b0, b1); the first workgroup has them all where there is no
  // second kernel to add them up, and on the largest tile, which has no registers for a third loop
  // (47 us against 51 at 262144 x 96 x 384 on the smallest tile; 592 against 585 at 147456 x 1024 x
  // 2048 on the largest)
  constexpr bool SHARE = TO * TI < 8;
  const int shares = SHARE && a.S > 1 ? a.tiles_i : 1;
  const bool do_bias = a.db != nullptr && ib < shares;
  const int b0 = do_bias ? cb + (int)((long long)(ce - cb) * ib / shares) : cb;
  const int b1 = do_bias ? cb + (int)((long long)(ce - cb) * (ib + 1) / shares) : cb;
  float bsum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) bsum[i] = 0.f;
  auto put_g = [&](int p, auto bias_tag) {
    constexpr bool BIAS = decltype(bias_tag)::value;
    lds_byte* to = at_g + p * (NT / GC) * kPitchG;
    if constexpr (FEED == kHalves) {
      const uint4 d = g[p].a;
      g[p].a = make_uint4(__builtin_amdgcn_alignbit(d.y, d.x, gshift), __builtin_amdgcn_alignbit(d.z, d.y, gshift),
                          __builtin_amdgcn_alignbit(d.w, d.z, gshift), __builtin_amdgcn_alignbit(tail[p], d.w, gshift));
    }
    float v[8];
    if constexpr (NP == 3 || BIAS) g[p].unpack(v);
    if constexpr (BIAS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) bsum[i] += v[i];
    }
    if constexpr (NP == 3) {
      uint4 hi, mid, lo;
      split3(v, hi, mid, lo);
      lds16(to, hi);
      lds16(to + NHO * kImgG, mid);
      lds16(to + 2 * NHO * kImgG, lo);
    } else {
      lds16(to, g[p].a);
    }
  };
  auto put_x = [&](int p) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
      unpack_chunk(h == 0 ? make_uint2(xq[p].x, xq[p].y) : make_uint2(xq[p].z, xq[p].w), xs[p], v);
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)                // exact in bf16: the upper halves
        o[i] = __builtin_amdgcn_perm(__float_as_uint(v[2 * i + 1]), __float_as_uint(v[2 * i]), 0x07060302u);
      lds16(at_x + p * (NT / XC) * kPitchX + h * 128, make_uint4(o[0], o[1], o[2], o[3]));
    }
  };
  auto to_stage = [&](int step) {                // where the pieces go, `step` stages on
    at_g += step * kStage;
    at_x += step * kStage;
  };

  f32x16_t acc[TO][TI];
#pragma unroll
  for (int x = 0; x < TO; ++x)
#pragma unroll
    for (int y = 0; y < TI; ++y) zero16(acc[x][y]);

  // MODE 0: no db, 1: db from every chunk, 2: from [b0, b1)
  auto run = [&](auto mode_tag) {
    constexpr int MODE = decltype(mode_tag)::value;
    // the first chunk into LDS, the next one into the registers
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (j == 1) {
        if (MODE == 1 || (MODE == 2 && b0 == cb && b1 > cb)) {
#pragma unroll
          for (int p = 0; p < GP; ++p) put_g(p, std::true_type{});
        } else {
#pragma unroll
          for (int p = 0; p < GP; ++p) put_g(p, std::false_type{});
        }
#pragma unroll
        for (int p = 0; p < XP; ++p) put_x(p);
        to_stage(1);
      }
#pragma unroll
      for (int p = 0; p < GP; ++p) fetch_g(p);
#pragma unroll
      for (int p = 0; p < XP; ++p) fetch_x(p);
      advance();
    }
    lds_barrier();
    // operands of a step of 16 tokens, read one step ahead
    bf16x8_t xa[2][TI], gb[2][TO][NP];
    auto operand = [&](lds_byte* p, int pitch) {
      const bf16x4v_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)p);
      const bf16x4v_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(p + 4 * pitch));
      return bf16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto read = [&](int k, int f) {
#pragma unroll
      for (int ti = 0; ti < TI; ++ti) xa[f][ti] = operand(at_a + 16 * kPitchX * k + 32 * ti, kPitchX);
#pragma unroll
      for (int to = 0; to < TO; ++to)
#pragma unroll
        for (int p = 0; p < NP; ++p)
          gb[f][to][p] = operand(at_b + p * NHO * kImgG + 16 * kPitchG * k + 64 * to, kPitchG);
    };
    auto next_stage = [&](int step) {
      at_b += step * kStage;
      at_a += step * kStage;
    };
    static_assert(KS % 2 == 0, "the operands' two sets alternate over chunks");
    int flip = 1;                                // from the stage that is read to the other one
    read(0, 0);
    auto chunk = [&](auto bias_tag) {
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        if (k + 1 < KS) {
          read(k + 1, (k + 1) & 1);
        } else {
          // chunk c's last operands are in registers and chunk c + 1 is written: the barrier makes
          // it visible and its own place free, with the last step's MFMAs still to issue
          if constexpr (TO * TI >= 8) {
            // the steps before, MFMA by MFMA with a share of the operand reads and of the pieces'
            // arithmetic behind each (alone on the chip 1257 ns a chunk against 1374 as the compiler
            // has it; the smaller tiles lose by it).  2 and 4 vector instructions: 530 us at 147456 x
            // 1024 x 2048; 3 and 5: 537, 4 and 6: 547, one LDS read an MFMA: 573.  kHalves with db:
            // 6 (4: the loop spills, 1282 us at 147456 x 1025 x 2047 against 733)
            constexpr int kVector = !decltype(bias_tag)::value ? 2 : FEED == kHalves ? 6 : 4;
#pragma unroll
            for (int i = 0; i < (KS - 1) * TO * TI; ++i) {
              __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);      // MFMA
              __builtin_amdgcn_sched_group_barrier(0x2, kVector, 0);// vector arithmetic
              __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);    // LDS reads
            }
          }
          lds_barrier();                         // (the loads of chunk c + 2 stay in flight)
          next_stage(flip);
          read(0, 0);
        }
        const int f = k & 1;
#pragma unroll
        for (int to = 0; to < TO; ++to)
#pragma unroll
          for (int p = NP - 1; p >= 0; --p)      // the smallest part first
#pragma unroll
            for (int ti = 0; ti < TI; ++ti) acc[to][ti] = mfma16(xa[f][ti], gb[f][to][p], acc[to][ti]);
        // (behind the last chunk too: into places that are not read again)
        constexpr int PS = KS - 1;               // the steps that carry the pieces
        if (k < PS) {
#pragma unroll
          for (int p = GP * k / PS; p < GP * (k + 1) / PS; ++p) put_g(p, bias_tag);
#pragma unroll
          for (int p = XP * k / PS; p < XP * (k + 1) / PS; ++p) put_x(p);
#pragma unroll
          for (int p = GP * k / PS; p < GP * (k + 1) / PS; ++p) fetch_g(p);
#pragma unroll
          for (int p = XP * k / PS; p < XP * (k + 1) / PS; ++p) fetch_x(p);
        }
      }
      advance();
      to_stage(-flip);
      flip = -flip;
    };
    // (at chunk c, chunk c + 1 passes through the registers)
    int c = cb;
    if constexpr (MODE == 2) {
      for (; c < b0 - 1; ++c) chunk(std::false_type{});
      for (; c < b1 - 1; ++c) chunk(std::true_type{});
    }
    for (; c < ce; ++c) chunk(std::integral_constant<bool, MODE == 1>{});
    lds_barrier();
  };
  if constexpr (SHARE)
    run(std::integral_constant<int, 2>{});
  else if (do_bias)
    run(std::integral_constant<int, 1>{});
  else
    run(std::integral_constant<int, 0>{});
  if (do_bias) {          // the threads that hold the same columns, in order
    float* sum = reinterpret_cast<float*>(smem);
    constexpr int R = NT / GC;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[gr * BO + gc * 8 + i] = bsum[i];
    __syncthreads();
    const int o = ob * BO + (int)threadIdx.x;
    if ((int)threadIdx.x < BO && o < a.N) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < R; ++k) t += sum[k * BO + threadIdx.x];
      if (a.S > 1)
        a.pbias[((size_t)s * shares + ib) * a.N + o] = t;
      else
        store_out(a.db, o, a.f32_out, t);
    }
  }

  // C tile: lane column = o, registers 4 g.. = 4 consecutive i
  if (a.S > 1) {
    float* pw = a.part + ((size_t)s * a.tiles + tile) * (BO * BI) + (size_t)w * (TO * TI * 1024) + l * 4;
#pragma unroll
    for (int to = 0; to < TO; ++to)
#pragma unroll
      for (int ti = 0; ti < TI; ++ti)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq)
          *reinterpret_cast<float4*>(pw + ((to * TI + ti) * 4 + gq) * 256) = make_float4(
              acc[to][ti][4 * gq], acc[to][ti][4 * gq + 1], acc[to][ti][4 * gq + 2], acc[to][ti][4 * gq + 3]);
  }
#pragma unroll
  for (int to = 0; to < TO; ++to) {
    const int o = ob * BO + wo + 32 * to + r;
    if (o >= a.N) continue;
    if (a.S == 1) {
#pragma unroll
      for (int ti = 0; ti < TI; ++ti)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq)
          store_four(a, o, ib * BI + wi + 32 * ti + 8 * gq + 4 * hh, acc[to][ti][4 * gq], acc[to][ti][4 * gq + 1],
                     acc[to][ti][4 * gq + 2], acc[to][ti][4 * gq + 3]);
    }
  }
}

// dW = the splits' partials added in order, in the partials' own order: a wave reads 1 KB (the
// 32 x 8 values of a register group) of each split at a time.  A workgroup takes 64 float4 in
// NG interleaved slices of the splits, whose sums it adds in order; the workgroups behind dW's
// are db's.
template <int BO, int BI, int WO, int WI, int NG>
__global__ void __launch_bounds__(64 * NG) act8_wgrad_sum_kernel(const Wgrad8 a) {
  constexpr int TO = BO / WO / 32, TI = BI / WI / 32, GROUPS = BO * BI / 256;
  __shared__ float4 lds[NG][64];
  const int l = threadIdx.x & 63, sl = threadIdx.x >> 6;
  const long long n = (long long)a.tiles * GROUPS;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (blockIdx.x >= n) {                         // db: 16 columns x 4 NG slices of the partial rows
    float* sum = reinterpret_cast<float*>(&lds[0][0]);
    const int col = threadIdx.x & 15, slice = threadIdx.x >> 4;
    const long long o = (blockIdx.x - n) * 16 + col;
    const int rows = a.S * (TO * TI < 8 ? a.tiles_i : 1);      // (SHARE)
    float t = 0.f;
    if (o < a.N) {
#pragma unroll 8
      for (int s = slice; s < rows; s += 4 * NG) t += a.pbias[(size_t)s * a.N + o];
    }
    sum[slice * 16 + col] = t;
    __syncthreads();
    if (slice == 0 && o < a.N) {
#pragma unroll
      for (int k = 1; k < 4 * NG; ++k) t += sum[k * 16 + col];
      store_out(a.db, o, a.f32_out, t);
    }
    return;
  }
  const int tile = blockIdx.x / GROUPS, grp = blockIdx.x - tile * GROUPS;
  const int ob = tile / a.tiles_i, ib = tile - ob * a.tiles_i;
  const int gq = grp & 3, t = (grp >> 2) % (TO * TI), w = (grp >> 2) / (TO * TI);
  const int o = ob * BO + (w % WO) * (BO / WO) + 32 * (t / TI) + (l & 31);
  const int i = ib * BI + (w / WO) * (BI / WI) + 32 * (t % TI) + 8 * gq + 4 * (l >> 5);
  const float* p = a.part + (size_t)blockIdx.x * 256 + l * 4;
  const size_t stride = (size_t)a.tiles * BO * BI;
  if (o < a.N && i < a.K) {
#pragma unroll 4
    for (int s = sl; s < a.S; s += NG) {
      const float4 u = *reinterpret_cast<const float4*>(p + s * stride);
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
    }
  }
  lds[sl][l] = v;
  __syncthreads();
  if (sl == 0 && o < a.N) {
#pragma unroll
    for (int k = 1; k < NG; ++k) {
      const float4 u = lds[k][l];
      v.x += u.x;
      v.y += u.y;
      v.z += u.z;
      v.w += u.w;
    }
    store_four(a, o, i, v.x, v.y, v.z, v.w);
  }
}

// How a problem is run: the tile and the splits of the tokens, whichever has the smallest estimate
//     chunks of a workgroup x time of a chunk on a full chip + 4 us
//     + with splits: 5 us for the second launch and 0.2 us a MB of partials
// (us; a place is a workgroup that runs at a time: splits fill the places once, or a half, a
// quarter, ... of them).  Measured as tile 0 / 1 / 2, us:  147456 tokens x 1024 x 2048: 635 / 677 /
// 790;  65536 x 768 x 192: 48 / 42 / 52;  16384 x 1536 x 384: 45 / 37 / 41;  262144 x 96 x 384: 79 /
// 67 / 52.  Tile 2 / 3:  400 x 256 x 256: 8.6 / 7.0 (12 in two splits);  10007 x 203 x 299: 15.5 /
// 13.7;  262144 x 96 x 96: 22.3 / 26;  262144 x 96 x 384: 44 / 58;  300000 x 20 x 64: 24 / 15.  f32,
// tile 4 / 5: 65536 x 768 x 768: 271 / 210-250 (the cutting of the gradients serves twice the
// columns);  16384 x 384 x 384: 28.8 / 31;  4 / 6: 400 x 256 x 256: 9.8 / 8.7;  10007 x 203 x 299: 19.1 /
// 18.1;  16384 x 384 x 384: 26 / 35;  300000 x 18 x 20: 40 / 23.
struct Tile {
  int f32, bo, bi, tk, places;
  float chunk, alone;                            // alone: with at most half the places taken
};
constexpr Tile kTiles[] = {
    {0, 256, 256, 64, 256, 2.19f, 2.19f}, {0, 256, 128, 64, 256, 1.175f, 1.175f},
    {0, 128, 128, 64, 256, 0.8f, 0.8f},   {0, 64, 64, 64, 512, 0.49f, 0.385f},
    {1, 128, 128, 64, 256, 1.76f, 1.76f}, {1, 128, 256, 32, 256, 1.31f, 1.31f},
    {1, 64, 64, 64, 256, 0.62f, 0.62f},
};
struct Plan {
  int tile, bo, bi, S;
  long long tiles;
};

Plan plan_of(bool f32, long long T, int N, int K) {
  Plan best = {};
  float least = 0.f;
  for (int c = 0; c < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++c) {
    const Tile& t = kTiles[c];
    if ((t.f32 != 0) != f32) continue;
    const long long tiles = (long long)((N + t.bo - 1) / t.bo) * ((K + t.bi - 1) / t.bi);
    const long long nchunk = (T + t.tk - 1) / t.tk;
    long long S = t.places / tiles;
    if (S > nchunk / 2) S = nchunk / 2;
    if (S < 1) S = 1;
    for (; S >= 1; S >>= 1) {
      const long long turns = (tiles * S + t.places - 1) / t.places;
      float cost = (float)(turns * ((nchunk + S - 1) / S)) * (2 * tiles * S <= t.places ? t.alone : t.chunk) + 4.f;
      if (S > 1) cost += 5.f + 0.2e-6f * (float)(4 * S * tiles * t.bo * t.bi);
      if (best.S == 0 || cost < least) {
        best = {c, t.bo, t.bi, (int)S, tiles};
        least = cost;
      }
    }
  }
  return best;
}

bool sizes_ok(long long T, int N, int K) {
  return T >= 0 && T < (1ll << 31) && N >= 0 && K >= 0 && N <= (1 << 24) && K <= (1 << 24) &&
         (long long)((N + 127) / 128) * ((K + 127) / 128) < (1 << 20);
}

long long workspace_bytes(const Plan& p, int N, int K) {
  return p.S == 1 ? 0 : 4ll * p.S * (p.tiles * p.bo * p.bi + (long long)((K + p.bi - 1) / p.bi) * N);
}

template <typename T, int BO, int BI, int WO, int WI, int TK>
int launch(const Wgrad8& a, Feed feed, hipStream_t st) {
  constexpr int NP = std::is_same<T, float>::value ? 3 : 1;
  constexpr int kLds = 2 * TK * (NP * images(BO) * kPitchG + images(BI) * kPitchX);
  auto kernel = feed == kRows ? act8_wgrad_kernel<T, BO, BI, WO, WI, TK, kRows>
                              : act8_wgrad_kernel<T, BO, BI, WO, WI, TK, kDwords>;
  if constexpr (NP == 1)
    if (feed == kHalves) kernel = act8_wgrad_kernel<T, BO, BI, WO, WI, TK, kHalves>;
  if (kLds > 64 * 1024)                          // above the default limit of a launch
    VS_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  hipLaunchKernelGGL(kernel, dim3((unsigned)(a.S * a.tiles)), dim3(64 * WO * WI), kLds, st, a);
  VS_LAUNCH_CHECK();
  if (a.S > 1) {
    const long long groups = (long long)a.tiles * (BO * BI / 256) + (a.db ? (a.N + 15) / 16 : 0);
    auto sum = [&](auto slices) {
      constexpr int NG = decltype(slices)::value;
      hipLaunchKernelGGL((act8_wgrad_sum_kernel<BO, BI, WO, WI, NG>), dim3((unsigned)groups), dim3(64 * NG), 0, st, a);
    };
    if (a.S > 64)                                // us with 4 / 16: 300000 x 20 x 64 in 512 splits 21.0 / 15.2,
      sum(std::integral_constant<int, 16>{});    // 262144 x 96 x 96 in 256 24.4 / 22.3,
    else                                         // 4096 x 768 x 768 in 3 21.1 / 24.6
      sum(std::integral_constant<int, 4>{});
    VS_LAUNCH_CHECK();
  }
  return VS_OK;
}

}  // namespace
}  // namespace vs

using namespace vs;

extern "C" long long vs_act8_wgrad_workspace_bytes(int dtype, long long tokens, int N, int K) {
  if (!sizes_ok(tokens, N, K) || N == 0 || K == 0) return 0;
  return workspace_bytes(plan_of(dtype == VS_F32, tokens, N, K), N, K);
}

extern "C" int vs_act8_wgrad(int dtype, int out_dtype, const void* gy, long long ld_gy, const void* q,
                             const void* scale, void* dw, void* db, void* workspace, long long tokens, int N, int K,
                             void* stream) {
  VS_CHECK((dtype == VS_F32 || dtype == VS_BF16) && (out_dtype == VS_F32 || out_dtype == VS_BF16),
           "dtypes must be VS_F32 or VS_BF16");
  VS_CHECK(sizes_ok(tokens, N, K), "sizes out of range");
  if (N == 0) return VS_OK;
  if (tokens <= 1) ld_gy = (N + 7) & ~7;         // one row: its stride is not used
  VS_CHECK(ld_gy >= N, "row stride >= N");
  VS_CHECK((K == 0 || dw) && (tokens == 0 || (gy && (K == 0 || (q && scale)))), "null pointer");
  VS_CHECK(((uintptr_t)q & 15) == 0, "q must be 16-B aligned");
  VS_CHECK(K > 0, "K > 0");
  VS_CHECK(((uintptr_t)gy & (dtype == VS_F32 ? 3 : 1)) == 0, "gy must be aligned to its elements");
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
  const Plan plan = plan_of(dtype == VS_F32, tokens, N, K);
  a.S = plan.S;
  a.tiles_i = (K + plan.bi - 1) / plan.bi;
  a.tiles = (int)plan.tiles;
  a.f32_out = out_dtype == VS_F32;
  a.vec = K % 4 == 0 && ((uintptr_t)dw & 15) == 0;
  VS_CHECK(a.S == 1 || (workspace && ((uintptr_t)workspace & 15) == 0),
           "workspace: 16-B aligned, sized by vs_act8_wgrad_workspace_bytes");
  a.part = (float*)workspace;
  a.pbias = a.part + (size_t)a.S * a.tiles * (plan.bo * plan.bi);
  hipStream_t st = (hipStream_t)stream;
  // buffer loads: a chunk of rows within their 32-bit offsets
  const long long esz = dtype == VS_F32 ? 4 : 2;
  const Feed feed = 64 * (ld_gy + N) * esz >= (1ll << 31)                     ? kRows
                    : (((uintptr_t)gy & 3) == 0 && ld_gy * esz % 4 == 0) ? kDwords
                                                                         : kHalves;
  switch (plan.tile) {
    case 0: return launch<bf16, 256, 256, 2, 4, 64>(a, feed, st);
    case 1: return launch<bf16, 256, 128, 4, 2, 64>(a, feed, st);
    case 2: return launch<bf16, 128, 128, 2, 4, 64>(a, feed, st);
    case 3: return launch<bf16, 64, 64, 2, 2, 64>(a, feed, st);
    case 4: return launch<float, 128, 128, 2, 4, 64>(a, feed, st);
    case 5: return launch<float, 128, 256, 2, 4, 32>(a, feed, st);
    default: return launch<float, 64, 64, 2, 2, 64>(a, feed, st);
  }
}
