// int8_rows.cu -- rows of activations to 8-bit integers with one scale a row, and back.
//
//   int8(v) of a row v[0 .. K):  m = max(max_k |v_k|, 2^-100),  scale = m / 127,
//                                code_k = rint(v_k * (127 / m))          (ties to even)
// The floor 2^-100 keeps the scale and its reciprocal normal numbers for an all-zero or a
// subnormal row; |v_k * (127 / m)| <= 127 (1 + 2^-22), so no code needs clamping.  A row
// that holds an infinity or a NaN gets scale NaN and codes 0: its products are NaN.
//
// v is the row itself (quantize), silu(gate) * up of a packed gate|up row (swiglu), or the
// weighted root-mean-square norm of x + residual (rmsnorm); everything up to the code is
// kept in fp32, and the sum x + residual is rounded once, when it is stored.
#include <math.h>

#include <atomic>

#include "sd_common.cuh"
#include "sd_internal.h"

namespace sd {

constexpr float kInt8Max = 127.f;
constexpr int kInt8MaxRow = 1 << 24;
constexpr float kInt8Floor = 7.888609052210118e-31f;  // 2^-100

template <typename T>
SD_DEV float widen(T v);
template <>
SD_DEV float widen<float>(float v) {
  return v;
}
template <>
SD_DEV float widen<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
SD_DEV T narrow(float v);
template <>
SD_DEV float narrow<float>(float v) {
  return v;
}
template <>
SD_DEV __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

constexpr int kWarpRows = 4;
enum RowOp { kRowQuantize = 0, kRowSwiglu = 1, kRowNorm = 2, kRowNormAdd = 3 };  // Add: with a residual

struct RowArgs {
  const void* x;
  int64_t x_stride;  // elements between rows of x (residual and summed: r_stride, s_stride)
  const void* residual;
  int64_t r_stride;
  const void* weight;
  float eps;
  void* summed;
  int64_t s_stride;
  int8_t* codes;
  int64_t c_stride;
  float* scale;
  int64_t rows;
  int32_t width;
  int32_t lose;  // of the self-test: no copy is started, every wait for one runs out
};

// rint(y) for |y| < 2^22 in the low byte of the sum with 1.5 * 2^23 (a product and a sum, each
// rounded: the codes are those of the formula in IEEE fp32)
SD_DEV uint32_t code_of(float v, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f)); }

// max that returns NaN when an operand is one (fmaxf drops it)
SD_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// the largest magnitude of `m` and N values, two values an instruction (sm_100's three-operand maximum)
template <int N>
SD_DEV float amax_values(float m, const float (&v)[N]) {
  if constexpr (N == 1) {
    return max_nan(m, fabsf(v[0]));
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 2)
      asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[k]), "f"(v[k + 1]));
    return m;
  }
}

// silu(g) * u with the hardware exponential and reciprocal: for |g| < 16 within 2^-19 of the exact
// value, far under what decides a code; the exponent's rounding is |g| 2^-24 of it further out, 2^-17 at
// g = -87, and -0 below, where exp(-g) passes 2^126 (the exact value is under 2^-119 |u|)
SD_DEV float silu_mul(float g, float u) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(g * -1.4426950408889634f)));
  return g * r * u;
}

// N consecutive values (N = 1, or 16 bytes of them) as they lie in memory
template <typename T, int N>
struct Piece {
  T e[N];
};
template <typename T>
struct alignas(16) Piece<T, 16 / sizeof(T)> {
  T e[16 / sizeof(T)];
};
template <typename T, int N>
SD_DEV Piece<T, N> load_piece(const T* p) {
  return *reinterpret_cast<const Piece<T, N>*>(p);
}
template <typename T, int N>
SD_DEV void store_values(T* p, const float (&v)[N]) {
  Piece<T, N> raw;
#pragma unroll
  for (int k = 0; k < N; ++k) raw.e[k] = narrow<T>(v[k]);
  *reinterpret_cast<Piece<T, N>*>(p) = raw;
}
SD_DEV uint32_t pack_codes(const float* v, float inv) {
  const uint32_t lo = __byte_perm(code_of(v[0], inv), code_of(v[1], inv), 0x0040);
  const uint32_t hi = __byte_perm(code_of(v[2], inv), code_of(v[3], inv), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
template <int N>
SD_DEV void store_codes(int8_t* p, const float (&v)[N], float inv) {
  if constexpr (N == 1)
    *p = static_cast<int8_t>(code_of(v[0], inv) & 0xFFu);
  else if constexpr (N == 4)
    *reinterpret_cast<uint32_t*>(p) = pack_codes(v, inv);
  else
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_codes(v, inv), pack_codes(v + 4, inv));
}

// Sum of squares and largest magnitude of a row over the G threads that hold it, in every thread (the
// maximum keeps a NaN).  `part`: a pair per warp, used once between two block-wide barriers.
template <int G, bool SUM>
SD_DEV float2 row_reduce(float2 v, float2* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (SUM) v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y = max_nan(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
  }
  if constexpr (G > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[threadIdx.x & (G / 32 - 1)];
#pragma unroll
    for (int o = G / 64; o > 0; o >>= 1) {
      if (SUM) v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y = max_nan(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
    }
  }
  return v;
}

// What is quantised, before the norm's factors, from the values x and (second half of a gate|up row,
// or the residual) y
template <int OP>
SD_DEV float row_value(float x, float y) {
  if (OP == kRowSwiglu) return silu_mul(x, y);
  return OP == kRowNormAdd ? x + y : x;
}
template <int OP>
constexpr bool kTwoInputs = OP == kRowSwiglu || OP == kRowNormAdd;
template <int OP>
constexpr bool kIsNorm = OP == kRowNorm || OP == kRowNormAdd;
template <typename T, int OP>
SD_DEV const T* second_row(const RowArgs& a, int64_t row) {
  if (OP == kRowSwiglu) return static_cast<const T*>(a.x) + row * a.x_stride + a.width;
  return static_cast<const T*>(a.residual) + row * a.r_stride;
}
// The norm's y = s * weight / rms is kept as z = s * weight until the one reduction of a row has given
// both the sum of s^2 and the largest |z|; 1 / rms then joins the factors of the codes and the scale.
struct RowScale {
  float rms, inv, scale;  // code = rint(z * rms * inv); inv = 0 and scale NaN for a row that is not finite
};
template <int OP>
SD_DEV RowScale row_scale(const RowArgs& a, float2 r) {
  RowScale s;
  s.rms = 1.f;
  bool finite = true;
  if (kIsNorm<OP>) {
    finite = r.x <= 3.4028234663852886e38f;  // an infinite sum of finite values would make 1 / rms, and the row, zero
    s.rms = __fdiv_rn(1.f, __fsqrt_rn(r.x / static_cast<float>(a.width) + a.eps));
    r.y *= s.rms;
  }
  if (!finite || !(r.y <= 3.4028234663852886e38f)) {
    s.rms = s.inv = 0.f;
    s.scale = __int_as_float(0x7FC00000);
    return s;
  }
  const float m = fmaxf(r.y, kInt8Floor);
  s.inv = __fdiv_rn(kInt8Max, m);
  s.scale = __fdiv_rn(m, kInt8Max);
  return s;
}

// G threads a row (32: kWarpRows rows a block, no block-wide step; else a row per block), each with up
// to CH pieces of N values held in registers as fp32 from the load to the store: a row is read once,
// and the only wait is the reduction.
template <typename T, int OP, int G, int N, int CH>
__global__ void __launch_bounds__(G == 32 ? 32 * kWarpRows : G) int8_rows_kernel(const RowArgs a) {
  __shared__ float2 part[G == 32 ? 1 : G / 32];
  const int t = threadIdx.x & (G - 1);
  const int64_t row = G == 32 ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  grid_dep_wait();  // launched programmatically: x is the preceding work's output
  grid_dep_launch();
  if (G == 32 && row >= a.rows) return;
  // every load of the row is under way before the first value is used
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* yr = second_row<T, OP>(a, row);
  const T* w = static_cast<const T*>(a.weight);
  Piece<T, N> px[CH] = {}, py[CH] = {};
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (t + G * c) * N;
    if (i < a.width) px[c] = load_piece<T, N>(xr + i);
    if (kTwoInputs<OP> && i < a.width) py[c] = load_piece<T, N>(yr + i);
  }
  float v[CH][N];
  float2 r = make_float2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (t + G * c) * N;
#pragma unroll
    for (int k = 0; k < N; ++k) v[c][k] = row_value<OP>(widen<T>(px[c].e[k]), widen<T>(py[c].e[k]));
    if constexpr (kIsNorm<OP>) {
      if (OP == kRowNormAdd && i < a.width)
        store_values<T, N>(static_cast<T*>(a.summed) + row * a.s_stride + i, v[c]);
      if (i < a.width) py[c] = load_piece<T, N>(w + i);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        r.x += v[c][k] * v[c][k];
        v[c][k] *= widen<T>(py[c].e[k]);
      }
    }
    r.y = amax_values(r.y, v[c]);
  }
  const RowScale s = row_scale<OP>(a, row_reduce<G, kIsNorm<OP>>(r, part));
  if (s.inv == 0.f) {  // the same for the whole row: its codes are 0, whatever it holds
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int k = 0; k < N; ++k) v[c][k] = 0.f;
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (t + G * c) * N;
    if constexpr (kIsNorm<OP>)
#pragma unroll
      for (int k = 0; k < N; ++k) v[c][k] *= s.rms;
    if (i < a.width) store_codes<N>(a.codes + row * a.c_stride + i, v[c], s.inv);
  }
  if (t == 0) a.scale[row] = s.scale;
}

// 16 bytes from `sh` (a multiple of sizeof(T), the same for a warp) bytes into a pair of granules.  A
// branch picks the words: selecting them took three times the instructions, and this is what bounds an
// unaligned row.
template <typename T>
SD_DEV uint4 shift_granules(const uint4* g, uint32_t sh) {
  const uint4 a = g[0], b = g[1];
  uint32_t w0, w1, w2, w3, w4;
  switch (sh >> 2) {
    case 0: w0 = a.x, w1 = a.y, w2 = a.z, w3 = a.w, w4 = b.x; break;
    case 1: w0 = a.y, w1 = a.z, w2 = a.w, w3 = b.x, w4 = b.y; break;
    case 2: w0 = a.z, w1 = a.w, w2 = b.x, w3 = b.y, w4 = b.z; break;
    default: w0 = a.w, w1 = b.x, w2 = b.y, w3 = b.z, w4 = b.w; break;
  }
  if (sizeof(T) == 4) return make_uint4(w0, w1, w2, w3);
  const uint32_t bits = (sh & 2) * 8;
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                    __funnelshift_r(w3, w4, bits));
}

// Rows of any alignment, or too long for the registers of a few warps, through shared memory: W warps
// work on a row (1: eight independent warps a block with a ring each; 4 to 16: the block), and the
// copies of the next rows are always under way (cp.async.bulk into a ring of `slots` rows), so neither
// the reduction nor the arithmetic leaves HBM idle.  A copy takes the 16-byte granules inside the row;
// the values at the two ends of an unaligned row are loaded by lanes, one row ahead.  A thread holds up
// to stream_pieces(W) pieces of 16 bytes a row from the ring to the store.  VEC: all rows are 16-byte
// aligned and whole pieces; else a piece is shifted out of two granules of the ring, and the values past
// the last whole piece are taken by a lane each.  Outputs and weight are aligned either way.
constexpr int kStreamSlots = 4;
constexpr int kStreamSmem = 222 * 1024;
constexpr int stream_threads(int W) { return W == 1 ? 256 : 32 * W; }
constexpr int stream_pieces(int W) { return W == 1 ? 7 : 5; }
template <typename T, int OP, int W, bool VEC>
__global__ void __launch_bounds__(stream_threads(W)) int8_stream_rows_kernel(const RowArgs a, int slots, int row_bytes) {
  constexpr int kGroups = W == 1 ? 8 : 1, kThreads = 32 * W, kStreams = kTwoInputs<OP> ? 2 : 1;
  constexpr int kN = 16 / static_cast<int>(sizeof(T)), kCh = stream_pieces(W);
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t full[kGroups][kStreamSlots];
  __shared__ float2 part[2][W];
  __shared__ uint32_t late;  // W > 1: 1 + `odd` of the row at which a thread's wait gave up (threads may be a row apart)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = W == 1 ? warp : 0, t = W == 1 ? lane : threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  uint8_t* mine = ring + group * slots * kStreams * row_bytes;
  if (t == 0) {
    for (int s = 0; s < slots; ++s) mbar_init(&full[group][s], 1);
    fence_barrier_init();
    if (W > 1) late = 0;
  }
  __syncthreads();
  grid_dep_wait();
  grid_dep_launch();

  const auto row_ptr = [&](int k, int64_t row) {
    return reinterpret_cast<uintptr_t>(k == 0 ? static_cast<const T*>(a.x) + row * a.x_stride : second_row<T, OP>(a, row));
  };
  const uint32_t width_bytes = static_cast<uint32_t>(a.width) * sizeof(T);
  // bytes of row `row` of input k into its first granule
  const uint32_t base0 = static_cast<uint32_t>(row_ptr(0, 0)), base1 = kStreams == 2 ? static_cast<uint32_t>(row_ptr(1, 0)) : 0;
  const uint32_t pitch0 = static_cast<uint32_t>(a.x_stride) * sizeof(T);
  const uint32_t pitch1 = static_cast<uint32_t>(OP == kRowSwiglu ? a.x_stride : a.r_stride) * sizeof(T);
  const auto row_shift = [&](int k, int64_t row) {
    return VEC ? 0u : ((k == 0 ? base0 : base1) + static_cast<uint32_t>(row) * (k == 0 ? pitch0 : pitch1)) & 15u;
  };
  const auto slot_ptr = [&](int k, int slot) { return mine + (slot * kStreams + k) * row_bytes; };
  // the granules inside row `row`, by one thread
  const auto copy_row = [&](int64_t row, int slot) {
    uint32_t skip[2], bytes[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < kStreams; ++k) {
      const uint32_t sh = row_shift(k, row);
      skip[k] = (16 - sh) & 15;
      if (width_bytes > skip[k]) bytes[k] = (width_bytes - skip[k]) & ~15u;
    }
    fence_proxy_async();  // the ends of the slot's last row were written by ordinary stores
    mbar_arrive_expect_tx(&full[group][slot], bytes[0] + bytes[1]);
#pragma unroll
    for (int k = 0; k < kStreams; ++k)
      if (bytes[k])
        bulk_g2s(slot_ptr(k, slot) + (skip[k] ? 16 : 0), reinterpret_cast<const void*>(row_ptr(k, row) + skip[k]),
                 bytes[k], &full[group][slot]);
  };
  // the values of `row` outside its granules, one a lane (16 lanes an input): index, or -1
  const int end_input = lane >> 4;
  const auto end_index = [&](int64_t row) {
    if (end_input >= kStreams) return -1;
    const int l = lane & 15;
    const uint32_t sh = row_shift(end_input, row);
    const int head = min(a.width, static_cast<int>(((16 - sh) & 15) / sizeof(T)));
    const int tail = sh != 0 && sh + width_bytes < 16 ? 0 : static_cast<int>(((sh + width_bytes) & 15) / sizeof(T));
    return l < head ? l : l < head + tail ? a.width - tail + (l - head) : -1;
  };
  const auto load_end = [&](int64_t row, int at) {
    return at < 0 ? T(0.f) : reinterpret_cast<const T*>(row_ptr(end_input, row))[at];
  };
  const auto store_end = [&](int64_t row, int slot, int at, T v) {
    if (at >= 0) reinterpret_cast<T*>(slot_ptr(end_input, slot) + row_shift(end_input, row))[at] = v;
  };

  if (t == 0 && !a.lose)
    for (int s = 0; s < slots - (W > 1); ++s)
      if (row0 + s * step < a.rows) copy_row(row0 + s * step, s);
  const bool ends = !VEC && (W == 1 || warp == 0);
  if (ends && row0 < a.rows) {
    const int at = end_index(row0);
    store_end(row0, 0, at, load_end(row0, at));
  }
  if (W > 1)
    __syncthreads();
  else
    __syncwarp();

  const T* w = static_cast<const T*>(a.weight);
  const int whole = a.width / kN * kN;                                   // values in whole pieces
  const int tail = !VEC && t < a.width - whole ? whole + t : -1;         // this thread's value past them
  int slot = 0;
  uint32_t parity = 0, odd = 0;
  for (int64_t row = row0; row < a.rows; row += step, odd ^= 1) {
    const int next_slot = slot + 1 == slots ? 0 : slot + 1;
    // the next row's ends are on their way while this row is worked on
    int at = -1;
    T end_value = T(0.f);
    if (ends && row + step < a.rows) {
      at = end_index(row + step);
      end_value = load_end(row + step, at);
    }
    bool ok = mbar_wait(&full[group][slot], parity);
    if (W == 1)
      ok = __all_sync(0xffffffffu, ok);
    else if (!ok)
      late = odd + 1;
    const uint32_t shx = row_shift(0, row), shy = kStreams == 2 ? row_shift(1, row) : 0;
    const uint8_t *xs = slot_ptr(0, slot), *ys = slot_ptr(kStreams - 1, slot);
    // 16 bytes from value i on of an input's row
    const auto piece = [&](const uint8_t* at, uint32_t sh, int i) {
      Piece<T, kN> p;
      const uint4* g = reinterpret_cast<const uint4*>(at + i * sizeof(T));
      *reinterpret_cast<uint4*>(&p) = VEC ? g[0] : shift_granules<T>(g, sh);
      return p;
    };
    float v[kCh][kN], tv[1] = {0.f};
    float2 r = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int i = (t + kThreads * c) * kN;
      if (i >= whole) break;
      const Piece<T, kN> px = piece(xs, shx, i), py = kStreams == 2 ? piece(ys, shy, i) : px;
#pragma unroll
      for (int k = 0; k < kN; ++k) v[c][k] = row_value<OP>(widen<T>(px.e[k]), widen<T>(py.e[k]));
      if constexpr (OP == kRowNormAdd)
        store_values<T, kN>(static_cast<T*>(a.summed) + row * a.s_stride + i, v[c]);
      if constexpr (kIsNorm<OP>) {
        const Piece<T, kN> pw = load_piece<T, kN>(w + i);
#pragma unroll
        for (int k = 0; k < kN; ++k) {
          r.x += v[c][k] * v[c][k];
          v[c][k] *= widen<T>(pw.e[k]);
        }
      }
      r.y = amax_values(r.y, v[c]);
    }
    if (tail >= 0) {
      const auto at_tail = [&](const uint8_t* at, uint32_t sh) { return widen<T>(reinterpret_cast<const T*>(at + sh)[tail]); };
      tv[0] = row_value<OP>(at_tail(xs, shx), kStreams == 2 ? at_tail(ys, shy) : 0.f);
      if constexpr (OP == kRowNormAdd) static_cast<T*>(a.summed)[row * a.s_stride + tail] = narrow<T>(tv[0]);
      if constexpr (kIsNorm<OP>) {
        r.x += tv[0] * tv[0];
        tv[0] *= widen<T>(w[tail]);
      }
      r.y = amax_values(r.y, tv);
    }
    if (ends) {
      store_end(row + step, next_slot, at, end_value);
      fence_proxy_async();  // before a later copy into these bytes
    }
    r = row_reduce<kThreads, kIsNorm<OP>>(r, part[odd]);
    if (W > 1) ok = late != odd + 1;
    if (!ok) {
      // copies that did not land within the wait's limit: what is left is marked, the others are awaited
      // (bounded, too), and the block ends
      if constexpr (OP == kRowNormAdd) {
        if (W == 1) __syncwarp();  // this row's sums, of whatever was there, are written
        for (int64_t left = row; left < a.rows; left += step)
          for (int i = t; i < a.width; i += kThreads)
            static_cast<T*>(a.summed)[left * a.s_stride + i] = narrow<T>(__int_as_float(0x7FC00000));
      }
      if (t == 0) {
        for (int64_t left = row; left < a.rows; left += step) a.scale[left] = __int_as_float(0x7FC00000);
        for (int i = 0; !a.lose && i < slots - (W > 1) && row + i * step < a.rows; ++i)
          (void)mbar_wait(&full[group][(slot + i) % slots], slot + i < slots ? parity : parity ^ 1);
      }
      break;
    }
    // W > 1: past the barrier of this row's reduction nobody reads the previous row's slot; W = 1: the
    // shuffles of the reduction come after every lane's reads of this row's
    if (t == 0) {
      if (W > 1 && row + (slots - 1) * step < a.rows)
        copy_row(row + (slots - 1) * step, slot == 0 ? slots - 1 : slot - 1);
      if (W == 1 && row + slots * step < a.rows) copy_row(row + slots * step, slot);
    }
    const RowScale s = row_scale<OP>(a, r);
    int8_t* codes = a.codes + row * a.c_stride;
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int i = (t + kThreads * c) * kN;
      if (i >= whole) break;
      if (s.inv == 0.f)
#pragma unroll
        for (int k = 0; k < kN; ++k) v[c][k] = 0.f;
      if constexpr (kIsNorm<OP>)
#pragma unroll
        for (int k = 0; k < kN; ++k) v[c][k] *= s.rms;
      store_codes<kN>(codes + i, v[c], s.inv);
    }
    if (tail >= 0) {
      tv[0] = s.inv == 0.f ? 0.f : tv[0] * s.rms;
      store_codes<1>(codes + tail, tv, s.inv);
    }
    if (t == 0) a.scale[row] = s.scale;
    if (W == 1) __syncwarp();
    if (next_slot == 0) parity ^= 1;
    slot = next_slot;
  }
}

// Rows too long for a ring in shared memory (a block's registers hold 20480 bf16 values, the ring three rows of 18944
// and a second input; f32 half as many): read again in each pass, a value a lane and load.  8192 x 28672 bf16: quantise 203 us (108 of bytes), norm 290, with residual 551 (251), swiglu 390 (180).
template <typename T, int OP>
__global__ void __launch_bounds__(1024) int8_long_rows_kernel(const RowArgs a) {
  __shared__ float2 part[32];
  const int64_t row = blockIdx.x;
  grid_dep_wait();
  grid_dep_launch();
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* yr = second_row<T, OP>(a, row);
  const T* w = static_cast<const T*>(a.weight);
  const auto value = [&](int i) { return row_value<OP>(widen<T>(xr[i]), kTwoInputs<OP> ? widen<T>(yr[i]) : 0.f); };
  float2 r = make_float2(0.f, 0.f);
  for (int i = threadIdx.x; i < a.width; i += 1024) {
    float v = value(i);
    if (kIsNorm<OP>) {
      r.x += v * v;
      v *= widen<T>(w[i]);
    }
    r.y = max_nan(r.y, fabsf(v));
  }
  const RowScale s = row_scale<OP>(a, row_reduce<1024, kIsNorm<OP>>(r, part));
  for (int i = threadIdx.x; i < a.width; i += 1024) {
    float v[1] = {value(i)};
    if (OP == kRowNormAdd) static_cast<T*>(a.summed)[row * a.s_stride + i] = narrow<T>(v[0]);
    if (kIsNorm<OP>) v[0] *= widen<T>(w[i]);
    v[0] = s.inv == 0.f ? 0.f : v[0] * s.rms;
    store_codes<1>(a.codes + row * a.c_stride + i, v, s.inv);
  }
  if (threadIdx.x == 0) a.scale[row] = s.scale;
}

// code * scale: a warp per row and 1024 columns.  VEC: 16 codes a lane and load.  Else the outputs'
// alignment leads: a lane stores the 16 aligned bytes of outputs from value i on, its codes shifted out
// of the words around them, and the values before the first and after the last such piece (at most 11 each)
// are one lane's each.  (No __restrict__: codes and scales are written by the preceding kernel, which may
// still run when this one starts, so their loads must not count as independent of grid_dep_wait.)
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize_int8_kernel(const int8_t* codes, int64_t c_stride, const float* scale,
                                                              T* out, int64_t o_stride, int64_t rows, int width) {
  constexpr int kOut = 16 / static_cast<int>(sizeof(T));
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  grid_dep_wait();
  grid_dep_launch();
  if (row >= rows) return;
  const float s = scale[row];
  const int8_t* c = codes + row * c_stride;
  T* o = out + row * o_stride;
  if constexpr (VEC) {
    const int begin = blockIdx.y * 1024, end = min(width, begin + 1024);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = begin + (j * 32 + lane) * 16;
      if (i >= end) break;
      const uint4 raw = *reinterpret_cast<const uint4*>(c + i);
      const int8_t* e = reinterpret_cast<const int8_t*>(&raw);
#pragma unroll
      for (int k = 0; k < 16; k += kOut) {
        float v[kOut];
#pragma unroll
        for (int q = 0; q < kOut; ++q) v[q] = static_cast<float>(e[k + q]) * s;
        store_values<T, kOut>(o + i + k, v);
      }
    }
  } else {
    // pieces end 4 codes before the row does, so that the words around their codes are the row's
    int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / static_cast<int>(sizeof(T));
    if (head < 4 && (reinterpret_cast<uintptr_t>(c) & 3)) head += kOut;  // nor before its first code
    const int pieces = max(0, width - head - 4) / kOut, most = 1024 / kOut;
    const int last = min(pieces, static_cast<int>(blockIdx.y + 1) * most);
    for (int j = blockIdx.y * most + lane; j < last; j += 32) {
      const int i = head + j * kOut;
      const uintptr_t at = reinterpret_cast<uintptr_t>(c + i);
      const uint32_t* words = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
      const uint32_t bits = static_cast<uint32_t>(at & 3) * 8;
      uint32_t raw[kOut / 4 + 1];
#pragma unroll
      for (int q = 0; q <= kOut / 4; ++q) raw[q] = words[q];
      float v[kOut];
#pragma unroll
      for (int q = 0; q < kOut; ++q) {
        const uint32_t word = __funnelshift_r(raw[q / 4], raw[q / 4 + 1], bits);
        v[q] = static_cast<float>(static_cast<int8_t>(word >> (8 * (q % 4)))) * s;
      }
      store_values<T, kOut>(o + i, v);
    }
    if (blockIdx.y == 0) {
      const int first = min(head, width), i = lane < first ? lane : head + pieces * kOut + lane - first;
      if (i < width) o[i] = narrow<T>(static_cast<float>(c[i]) * s);
    }
  }
}

static int check_rows(const char* what, const void* x, int64_t x_stride, int64_t need, const void* codes,
                      int64_t c_stride, const void* scale, int32_t dtype, int64_t rows, int32_t width) {
  if (rows < 0 || rows > 0x7fffffff) return fail(SPECDEC_ERR_INVALID, "%s: row count out of range", what);
  if (width <= 0) return fail(SPECDEC_ERR_INVALID, "%s: empty row", what);
  if (width > kInt8MaxRow) return fail(SPECDEC_ERR_INVALID, "%s: row longer than %d", what, kInt8MaxRow);
  if (dtype != SPECDEC_F32 && dtype != SPECDEC_BF16)
    return fail(SPECDEC_ERR_INVALID, "%s supports float32 and bfloat16", what);
  if (rows == 0) return SPECDEC_OK;
  if (!x || !codes || !scale) return fail(SPECDEC_ERR_INVALID, "%s: tensors must be CUDA", what);
  if (x_stride < need || c_stride < width)
    return fail(SPECDEC_ERR_INVALID, "%s: a row stride is smaller than its row", what);
  if (reinterpret_cast<uintptr_t>(x) % (dtype == SPECDEC_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(scale) % 4)
    return fail(SPECDEC_ERR_INVALID, "%s: a tensor is not aligned to its elements", what);
  return SPECDEC_OK;
}

template <typename T, int OP, int G, int N, int CH>
static int launch_rows_as(const char* what, const RowArgs& a, cudaStream_t st) {
  const int64_t blocks = G == 32 ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows;
  return launch_pdl(what, int8_rows_kernel<T, OP, G, N, CH>, dim3(static_cast<unsigned>(blocks)),
                    dim3(G == 32 ? 32 * kWarpRows : G), 0, st, a);
}

template <typename T, int OP, int W, bool VEC>
static int launch_stream_as(const char* what, const RowArgs& a, int slots, int row_bytes, cudaStream_t st) {
  constexpr int kGroups = W == 1 ? 8 : 1;
  const int smem = kGroups * slots * row_bytes * (kTwoInputs<OP> ? 2 : 1);
  auto* kern = int8_stream_rows_kernel<T, OP, W, VEC>;
  static std::atomic<bool> attr_set[64];  // threads may be here at once
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamSmem);
    if (e != cudaSuccess) return fail(SPECDEC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    attr_set[dev].store(true, std::memory_order_release);
  }
  // blocks that fit an SM's shared memory, and 1024 threads
  int per_sm = 220 * 1024 / (smem + 2048);
  per_sm = per_sm < 1 ? 1 : per_sm > 1024 / stream_threads(W) ? 1024 / stream_threads(W) : per_sm;
  const int64_t need = (a.rows + kGroups - 1) / kGroups;
  const int64_t most = static_cast<int64_t>(device_sm_count()) * per_sm;
  return launch_pdl(what, kern, dim3(static_cast<unsigned>(need < most ? need : most)), dim3(stream_threads(W)),
                    static_cast<size_t>(smem), st, a, slots, row_bytes);
}
// SPECDEC_ERR_UNSUPPORTED when three rows do not fit the ring (the one at work, the next, and the one
// whose ends are being written)
template <typename T, int OP>
static int launch_stream(const char* what, const RowArgs& a, bool vec, cudaStream_t st) {
  constexpr int kStreams = kTwoInputs<OP> ? 2 : 1;
  const int64_t bytes = (static_cast<int64_t>(sizeof(T)) * a.width + 15) / 16 * 16 + (vec ? 0 : 32);
  const int64_t pieces = (a.width + 16 / static_cast<int>(sizeof(T)) - 1) / (16 / static_cast<int>(sizeof(T)));
  if (pieces > 512 * stream_pieces(16) || 3 * kStreams * bytes > kStreamSmem) return SPECDEC_ERR_UNSUPPORTED;
  const int row = static_cast<int>(bytes);
  if (!vec && pieces <= 32 * stream_pieces(1)) return launch_stream_as<T, OP, 1, false>(what, a, 2, row, st);
  if (!vec && pieces <= 128 * stream_pieces(4)) return launch_stream_as<T, OP, 4, false>(what, a, kStreamSlots, row, st);
  int slots = (kStreamSmem / 2 + 8 * 1024) / (row * kStreams);  // two blocks an SM, if they have three rows each
  if (slots < 3) slots = kStreamSmem / (row * kStreams);
  if (slots > kStreamSlots) slots = kStreamSlots;
  if (pieces <= 256 * stream_pieces(8))
    return vec ? launch_stream_as<T, OP, 8, true>(what, a, slots, row, st)
               : launch_stream_as<T, OP, 8, false>(what, a, slots, row, st);
  return vec ? launch_stream_as<T, OP, 16, true>(what, a, slots, row, st)
             : launch_stream_as<T, OP, 16, false>(what, a, slots, row, st);
}

// Which kernel takes the rows; measured for bf16 rows of 896, 1536, 4864 and 8960 values, 5 to 32768 of
// them.  Aligned rows that a few warps can hold: a warp, or two to eight, a row, three to six pieces a
// thread, which keeps the most loads in flight (a block of 1024 threads a row: 3.3 us for 5 rows of
// swiglu's 8960, 13.5 for 600; 256 threads: 2.5 and 7.3; 32768 rows of swiglu's 1536: 49 us with a warp a
// row, 39 with two); short rows in small number are spread as wide as they go, a piece a thread (`few`:
// under eight rows an SM).  Longer ones, swiglu's long ones in large
// number (its arithmetic hides behind the ring's copies: 8192 x 8960 62 us, 90 in registers) and unaligned
// ones in large number through shared memory; unaligned rows in small number by single values, a block a
// row, and so are rows whose outputs are not aligned.
// The thresholds are in pieces of 16 bytes and decide f32, too (registers and ring, us: quantise 8192 x 2048
// 13.6 and 21.6, norm with residual 8192 x 4096 65.0 and 71.5, swiglu 8192 x 4096 45.6 and 46.1, which is the
// ring's), but for two: one f32 input in large number keeps a warp a row up to 320 pieces (a warp and four, us:
// 32768 x 1280 quantise 31.1 and 34.8, norm 35.1 and 37.9; x 1408 34.2 and 35.2, 44.0 and 39.3; x 1536 37.0 and
// 36.5, 44.2 and 40.7); and single values take unaligned f32 rows of 897 to 1024 values, which a
// block of 256 threads still holds while the ring needs four warps each (norm without a residual, 1001 values:
// 600 rows 3.4 us either way, 2000 5.5 and 7.1 in the ring, 8000 17.2 and 19.6).  Unaligned norms without a
// residual by single values and in the ring, us: 600 x 501 bf16 3.1 and 2.9, 1000 x 1501 bf16 11.8 and 4.5,
// 8000 x 1501 bf16 81.6 and 14.9, f32 79.4 and 22.3.
template <typename T, int OP>
static int launch_rows_t(const char* what, const RowArgs& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int64_t sms = device_sm_count();
  const bool few = a.rows < 8 * sms, two = kTwoInputs<OP>;
  const uintptr_t out_bits = reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.summed) |
                             static_cast<uintptr_t>(a.s_stride) * sizeof(T);
  const bool out_vec = out_bits % 16 == 0 &&
                       (reinterpret_cast<uintptr_t>(a.codes) | static_cast<uintptr_t>(a.c_stride)) % V == 0;
  const uintptr_t in_bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.residual) |
                            static_cast<uintptr_t>(a.x_stride | a.r_stride) * sizeof(T);
  const bool vec = out_vec && in_bits % 16 == 0 && a.width % V == 0;
  const int need = vec ? a.width / V : a.width;
  if (vec) {
    if (need <= 64 && !few) return launch_rows_as<T, OP, 32, V, 2>(what, a, st);
    if (need <= 128) return few ? launch_rows_as<T, OP, 128, V, 1>(what, a, st) : launch_rows_as<T, OP, 32, V, 4>(what, a, st);
    if (need <= 256 && a.rows <= 2 * sms) return launch_rows_as<T, OP, 256, V, 1>(what, a, st);
    if (need <= 192) return few || two ? launch_rows_as<T, OP, 64, V, 3>(what, a, st) : launch_rows_as<T, OP, 32, V, 6>(what, a, st);
    if (need <= 256) return few || two ? launch_rows_as<T, OP, 128, V, 2>(what, a, st) : launch_rows_as<T, OP, 32, V, 8>(what, a, st);
    if (need <= 320 && V == 4 && !few && !two) return launch_rows_as<T, OP, 32, V, 48 / V>(what, a, st);
    if (need <= 384) return launch_rows_as<T, OP, 128, V, 3>(what, a, st);
    if (need <= 640) return launch_rows_as<T, OP, 128, V, 5>(what, a, st);
    if (need <= 768) return launch_rows_as<T, OP, 256, V, 3>(what, a, st);
    if (need <= 1280 && (few || OP != kRowSwiglu)) return launch_rows_as<T, OP, 256, V, 5>(what, a, st);
  }
  const bool held = !vec && a.width <= 1024 && a.width > 32 * stream_pieces(1) * V;
  if (out_vec && !held && (vec || need > 8192 || a.rows > (need > 1024 ? 1 : 4) * sms))
    if (const int rc = launch_stream<T, OP>(what, a, vec, st); rc != SPECDEC_ERR_UNSUPPORTED) return rc;
  if (a.width <= 1024) return launch_rows_as<T, OP, 256, 1, 4>(what, a, st);
  if (a.width <= 8192) return launch_rows_as<T, OP, 1024, 1, 8>(what, a, st);
  return launch_pdl(what, int8_long_rows_kernel<T, OP>, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, st, a);
}
template <int OP>
static int launch_rows(const char* what, const RowArgs& a, int32_t dtype, cudaStream_t st) {
  return dtype == SPECDEC_F32 ? launch_rows_t<float, OP>(what, a, st) : launch_rows_t<__nv_bfloat16, OP>(what, a, st);
}

template <typename T>
static int launch_dequantize(const int8_t* codes, int64_t c_stride, const float* scale, T* out, int64_t o_stride,
                             int64_t rows, int32_t width, cudaStream_t st) {
  const bool vec = (reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(out) |
                    static_cast<uintptr_t>(c_stride) | static_cast<uintptr_t>(o_stride) * sizeof(T) |
                    static_cast<uintptr_t>(width)) %
                       16 == 0;
  const dim3 grid(static_cast<unsigned>((rows + 7) / 8), static_cast<unsigned>((width + 1023) / 1024));
  return launch_pdl("dequantize_int8", vec ? dequantize_int8_kernel<T, true> : dequantize_int8_kernel<T, false>, grid,
                    dim3(256), 0, st, codes, c_stride, scale, out, o_stride, rows, width);
}

}  // namespace sd

using namespace sd;

extern "C" int specdec_quantize_int8(const void* x, int64_t x_stride, void* codes, int64_t codes_stride, float* scale,
                                     int32_t dtype, int64_t rows, int32_t width, specdec_stream_t stream) {
  if (int rc = check_rows("quantize_int8", x, x_stride, width, codes, codes_stride, scale, dtype, rows, width))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  RowArgs a = {};
  a.lose = wait_limit_ns() == 0;
  a.x = x;
  a.x_stride = x_stride;
  a.codes = static_cast<int8_t*>(codes);
  a.c_stride = codes_stride;
  a.scale = scale;
  a.rows = rows;
  a.width = width;
  return launch_rows<kRowQuantize>("quantize_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int specdec_swiglu_int8(const void* gate_up, int64_t x_stride, void* codes, int64_t codes_stride,
                                   float* scale, int32_t dtype, int64_t rows, int32_t inter, specdec_stream_t stream) {
  if (int rc = check_rows("swiglu_int8", gate_up, x_stride, 2 * static_cast<int64_t>(inter), codes, codes_stride,
                          scale, dtype, rows, inter))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  RowArgs a = {};
  a.lose = wait_limit_ns() == 0;
  a.x = gate_up;
  a.x_stride = x_stride;
  a.codes = static_cast<int8_t*>(codes);
  a.c_stride = codes_stride;
  a.scale = scale;
  a.rows = rows;
  a.width = inter;
  return launch_rows<kRowSwiglu>("swiglu_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int specdec_rmsnorm_int8(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                    const void* weight, float eps, void* summed, int64_t summed_stride, void* codes,
                                    int64_t codes_stride, float* scale, int32_t dtype, int64_t rows, int32_t hidden,
                                    specdec_stream_t stream) {
  if (int rc = check_rows("rmsnorm_int8", x, x_stride, hidden, codes, codes_stride, scale, dtype, rows, hidden))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  if (!weight) return fail(SPECDEC_ERR_INVALID, "rmsnorm_int8: tensors must be CUDA");
  if ((residual == nullptr) != (summed == nullptr))
    return fail(SPECDEC_ERR_INVALID, "rmsnorm_int8: residual and summed come together");
  if (residual && (residual_stride < hidden || summed_stride < hidden))
    return fail(SPECDEC_ERR_INVALID, "rmsnorm_int8: a row stride is smaller than its row");
  if ((reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(residual) |
       reinterpret_cast<uintptr_t>(summed)) % (dtype == SPECDEC_F32 ? 4 : 2))
    return fail(SPECDEC_ERR_INVALID, "rmsnorm_int8: a tensor is not aligned to its elements");
  RowArgs a = {};
  a.lose = wait_limit_ns() == 0;
  a.x = x;
  a.x_stride = x_stride;
  a.residual = residual;
  a.r_stride = residual ? residual_stride : 0;  // of no account without one: they would decide the kernel
  a.weight = weight;
  a.eps = eps;
  a.summed = summed;
  a.s_stride = residual ? summed_stride : 0;
  a.codes = static_cast<int8_t*>(codes);
  a.c_stride = codes_stride;
  a.scale = scale;
  a.rows = rows;
  a.width = hidden;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return residual ? launch_rows<kRowNormAdd>("rmsnorm_int8", a, dtype, st)
                  : launch_rows<kRowNorm>("rmsnorm_int8", a, dtype, st);
}

extern "C" int specdec_dequantize_int8(const void* codes, int64_t codes_stride, const float* scale, void* out,
                                       int64_t out_stride, int32_t dtype, int64_t rows, int32_t width,
                                       specdec_stream_t stream) {
  if (int rc = check_rows("dequantize_int8", out, out_stride, width, codes, codes_stride, scale, dtype, rows, width))
    return rc;
  if (rows == 0) return SPECDEC_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int8_t* c = static_cast<const int8_t*>(codes);
  return dtype == SPECDEC_F32
             ? launch_dequantize(c, codes_stride, scale, static_cast<float*>(out), out_stride, rows, width, st)
             : launch_dequantize(c, codes_stride, scale, static_cast<__nv_bfloat16*>(out), out_stride, rows, width, st);
}
