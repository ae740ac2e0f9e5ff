// MatMulNBits: products with 4-bit weights that have a scale, and where given
// a zero point, for each group of consecutive k:
//   y[m, n] = sum_g s[n, g] * sum_{k in g} a[m, k] * (q[n, k] - z[n, g]) + bias[n]
// A group's inner sum and the sum over groups are fp32; the result is rounded
// to the tensor type once. bf16 and fp32 inner sums are formed 2^-12 times too
// small, so that they stay finite wherever the result does (15 * 256 < 2^12).
//
// For few rows the floor is the codes' bytes. At their rate an SM gets some 46
// codes a cycle, about a third as many as it has lanes, so a code may cost no
// more than two instructions: the products run on the tensor cores, with 16
// weight rows as the M operand and 8 activation rows as N, and a word of 8
// codes becomes 8 operands in 9 (fp16) or 11 instructions.
#include <algorithm>
#include <atomic>
#include <new>
#include <type_traits>

#include "decode.cuh"

namespace nnrcu {
namespace {

// The laid-out weights. Rows in tiles of 16, k in spans of 64. In one span of
// one tile, lane (g, t) of a warp holds codes of rows g and g + 8:
//   word h (of 4) has k = 32 (h / 2) + 8 t + 4 (h % 2) + {0, 1, 2, 3}: of row g
//   in nibbles 0, 4, 2, 6 and of row g + 8 in nibbles 1, 5, 3, 7,
// so that masking word >> 4 i for i = 0..3 leaves the four registers of a
// 16x8x16 operand, in pairs of neighbouring k: those of row g for even i. A lane's 16 bytes lie together,
// and so do the 8 activations that it wants of each half of the span.
// Scales: [tile][span][scales of a span][8] pairs (row g, row g + 8); with
// zero points each is followed by such a pair of them, as the number that is
// taken from the code's operand.
constexpr int kSpan = 64;

template <typename T>
struct Traits {  // of the operands
  using type = T;
  static constexpr int kParts = 1;
};
template <>
struct Traits<float> {  // fp32: the sum of three bf16, 8 bits each
  using type = __nv_bfloat16;
  static constexpr int kParts = 3;
};

// (code - zero) as a pair of operands, of row g and of row g + 8, whose codes
// lie 4 bits higher in x. fp16: 1024 + q, less 1024 + z; (1024 + 16 q) / 16,
// less 64 + z. bf16: (128 + q) 2^-12, less (128 + z) 2^-12. All are exact.
// The constants come as kernel parameters: known ones the compiler would set
// up again before each use, an instruction for each pair of codes.
template <typename M>
struct Unpack {
  static constexpr bool kF16 = std::is_same_v<M, __half>;
  uint32_t mask = 0x000F000Fu, high = 0x00F000F0u, ones = kF16 ? 0x64006400u : 0x43004300u;
  uint32_t small = kF16 ? 0x2C002C00u : 0x39803980u;  // 2^-4; 2^-12
  uint32_t eight[2];                                  // what stands for zero points where there are none
  __device__ __forceinline__ uint32_t row(uint32_t x, uint32_t zero) const {
    uint32_t r;
    if constexpr (kF16)
      asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(and_or(x, mask, ones)), "r"(zero));
    else
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(and_or(x, mask, ones)), "r"(small), "r"(zero));
    return r;
  }
  __device__ __forceinline__ uint32_t row8(uint32_t x, uint32_t zero) const {
    if constexpr (kF16) {
      uint32_t r;
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(and_or(x, high, ones)), "r"(small), "r"(zero));
      return r;
    } else {
      return row(x >> 4, zero);
    }
  }
};
// What is taken from, or added to, the codes of row g (e = 0) or g + 8.
template <typename M>
__host__ __device__ constexpr uint16_t zero_bits(int z, int e) {
  // 1024 + z or -(64 + z) in fp16; -(128 + z) 2^-12 in bf16 (128 + z has at most 8 bits)
  return std::is_same_v<M, __half> ? (e ? 0xD400 + 16 * z : 0x6400 + z) : 0xBD00 + z;
}

// c (zeros if FIRST) + a b.
template <typename M, bool FIRST>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
#define NNRCU_MMA(type, in)                                                                                          \
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." type "." type                                                \
               ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"                                      \
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                      \
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(in[0]), "f"(in[1]), "f"(in[2]),   \
                 "f"(in[3]))
  const float zeros[4] = {0.f, 0.f, 0.f, 0.f};
  if constexpr (std::is_same_v<M, __half>) {
    if constexpr (FIRST)
      NNRCU_MMA("f16", zeros);
    else
      NNRCU_MMA("f16", c);
  } else {
    if constexpr (FIRST)
      NNRCU_MMA("bf16", zeros);
    else
      NNRCU_MMA("bf16", c);
  }
#undef NNRCU_MMA
}

struct NbitsArgs {
  const void* a;
  void* y;
  long long lda, ldy;
  int m, n, k, spans;
  const uint4* codes;
  const void* scales;
  const void* bias;
  int spans_log2, scale_spans;  // a scale serves 2^spans_log2 spans; scales of a tile's row (pairs, for groups of 32)
  int items, more;              // of a block; that many blocks have one more
  int wide;            // a's rows start at multiples of: 2: 16 bytes, 1: 4 bytes
};

// A pair of scales, and of zero points, as they are laid out and as they are used.
template <typename T, bool ZERO>
struct Scale {
  static constexpr int kBytes = (std::is_same_v<T, float> ? 8 : 4) + (ZERO ? 4 : 0);
  float s0, s1;
  uint32_t z0, z1;
  __device__ __forceinline__ void load(const uint8_t* p, const uint32_t (&eight)[2]) {
    uint32_t zero = 0;
    if constexpr (std::is_same_v<T, float>) {
      s0 = reinterpret_cast<const float*>(p)[0], s1 = reinterpret_cast<const float*>(p)[1];
      if constexpr (ZERO) zero = reinterpret_cast<const uint32_t*>(p)[2];
    } else {
      uint32_t x;
      if constexpr (ZERO) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        x = v.x, zero = v.y;
      } else {
        x = *reinterpret_cast<const uint32_t*>(p);
      }
      if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
        s0 = f.x, s1 = f.y;
      } else {
        s0 = __uint_as_float(x << 16), s1 = __uint_as_float(x & 0xFFFF0000u);
      }
    }
    if constexpr (ZERO) {
      z0 = __byte_perm(zero, 0, 0x1010), z1 = __byte_perm(zero, 0, 0x3232);
    } else {
      z0 = eight[0], z1 = eight[1];
    }
  }
};

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(src), "n"(BYTES) : "memory");
}

// This lane's activations of one span, 8 of each half: as they lie (load) and
// as the operand pairs of its 4 steps (pairs). An fp32 value is the sum of
// three bf16, its leading 8 bits, the next and the last (an infinity has but
// the first).
template <typename T>
struct Activations {
  static constexpr int kWords = sizeof(T) * 2;  // 32-bit words of 8 of them
  uint32_t v[2][kWords];
  // `wide` as in NbitsArgs, 0 for the span that k ends in
  __device__ __forceinline__ void load(const T* row, int at, int k, int wide) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (wide == 2) {
#pragma unroll
        for (int j = 0; j < kWords; j += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(row + at + 32 * i + j * 4 / sizeof(T));
          v[i][j] = x.x, v[i][j + 1] = x.y, v[i][j + 2] = x.z, v[i][j + 3] = x.w;
        }
      } else if (sizeof(T) == 2 && wide == 1) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) v[i][j] = *reinterpret_cast<const uint32_t*>(row + at + 32 * i + 2 * j);
      } else {
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          const int n = at + 32 * i + j * 4 / (int)sizeof(T);
          if constexpr (sizeof(T) == 2) {
            const uint16_t* const r = reinterpret_cast<const uint16_t*>(row);
            v[i][j] = (n < k ? r[n] : 0u) | (n + 1 < k ? (uint32_t)r[n + 1] << 16 : 0u);
          } else {
            v[i][j] = n < k ? __float_as_uint(row[n]) : 0u;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void pairs(uint32_t (&b)[Traits<T>::kParts][4][2]) const {
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = h % 2 * 4 + 2 * e;
        if constexpr (sizeof(T) == 2) {
          b[0][h][e] = v[h / 2][at / 2];
        } else {
          uint32_t next[2], last[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t bits = v[h / 2][at + i];
            const float x = __uint_as_float(bits);
            const float rest = fabsf(x) == INFINITY ? 0.f : x - __uint_as_float(bits & 0xFFFF0000u);  // exact
            next[i] = __float_as_uint(rest);
            last[i] = __float_as_uint(rest - __uint_as_float(next[i] & 0xFFFF0000u));
          }
          b[0][h][e] = __byte_perm(v[h / 2][at], v[h / 2][at + 1], 0x7632);
          b[1][h][e] = __byte_perm(next[0], next[1], 0x7632);
          b[2][h][e] = __byte_perm(last[0], last[1], 0x7632);
        }
      }
  }
};

// Sizes of one kernel: tensor type, zero points or not, groups of 32 or more,
// RT times 8 activation rows (each 8 columns of operands, fp32: three times 8,
// for its parts), TT tiles of 16 outputs, and a block's warps.
template <typename T, bool ZERO, int BLOCK, int RT, int TT, int WARPS>
struct Cfg {
  static constexpr int kParts = Traits<T>::kParts;
  static constexpr int kRows = 8 * RT, CT = RT * kParts;  // activation rows of a block, tiles of columns
  static constexpr int kOuts = 16 * TT;
  static constexpr int kScales = BLOCK == 32 ? 2 : 1;   // of a span
  static constexpr int kLane = Scale<T, ZERO>::kBytes * kScales;
  static constexpr int kStage = TT * 32 * (16 + kLane); // what one warp brings of one span
  static constexpr int kColumns = 8 * CT + 2;
  static constexpr int kJoin = WARPS * kOuts * kColumns * 4;  // bytes in which the warps are joined
  static constexpr int kFit = (216 * 1024 - kJoin) / (WARPS * kStage), kWant = TT == 1 ? 8 : 5;
  static constexpr int kStages = kFit < kWant ? kFit : kWant;
  static_assert(kStages >= 3, "a ring of three at least");
  // The next span's activations are loaded before this one's products, where registers allow.
  static constexpr bool kEarly = RT * sizeof(T) <= 2;
  static constexpr int kSmem = WARPS * kStages * kStage + kJoin;
  static constexpr int kBlocks = WARPS == 16 ? 1 : (CT >= 4 ? 1 : (CT >= 2 ? 2 : 3));  // on an SM at least
};

// One block: items of TT tiles of 16 outputs, `items` of them one after the
// other. The spans of k are divided over the block's warps, which are joined
// through shared memory in a fixed order. Each lane brings its own 16 bytes of
// codes of a span, and its scales, through a ring of cp.async stages that runs
// on across the items; nobody else reads them, so nothing waits for another.
// On the device: 1x4096x4096 5.5 us, 1x16384x4096 13.5 us (2.6 TB/s of codes
// and scales), 16x14336x4096 17.6 us. Its instructions, some 115 a tile and span
// of which 60 are unpacking and products, take half of the issue slots at most
// (1x14336x4096: IPC 2.2, 16x14336x4096: 1.6); what is left are latencies with 16
// to 24 warps on an SM, and ends where some blocks have an item less than others.
template <typename T, bool ZERO, int BLOCK, int RT, int TT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, Cfg<T, ZERO, BLOCK, RT, TT, WARPS>::kBlocks)
    nbits_kernel(const __grid_constant__ NbitsArgs p, const Unpack<typename Traits<T>::type> operand) {
  using C = Cfg<T, ZERO, BLOCK, RT, TT, WARPS>;
  using M = typename Traits<T>::type;
  constexpr int kBytes = Scale<T, ZERO>::kBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * C::kRows, tiles = (p.n + 15) / 16;

  // Columns 8 (kParts i + part) + g are row row0 + 8 i + g. Those past the last
  // row repeat it and are not kept.
  constexpr int CT = C::CT;
  const T* rows[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
    rows[i] = static_cast<const T*>(p.a) + (long long)min(row0 + 8 * i + g, p.m - 1) * p.lda;

  const int my_spans = p.spans > warp ? (p.spans - warp + WARPS - 1) / WARPS : 0;
  const int share = blockIdx.x, first = share * p.items + min(share, p.more);
  const int last = first + p.items + (share < p.more);
  uint8_t* const ring = smem + warp * C::kStages * C::kStage + lane * 16;
  uint8_t* const ring_scales = smem + warp * C::kStages * C::kStage + TT * 512 + lane * C::kLane;
  // The next span to bring, and where it lies for each tile of its item. The
  // warp's spans are WARPS apart, a multiple of those that share a scale.
  int f_item = first, f_left = my_spans, f_slot = 0;
  const int f_step = (WARPS >> p.spans_log2) * (C::kScales * 8 * kBytes);
  const uint32_t f_ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const uint32_t f_ring_scales = static_cast<uint32_t>(__cvta_generic_to_shared(ring_scales));
  const uint4* f_codes[TT];
  const uint8_t* f_scales[TT];
  auto begin_item = [&]() {
#pragma unroll
    for (int j = 0; j < TT; ++j) {
      const long long tile = min(f_item * TT + j, tiles - 1);
      f_codes[j] = p.codes + (tile * p.spans + warp) * 32 + lane;
      f_scales[j] = static_cast<const uint8_t*>(p.scales) +
                    ((tile * p.scale_spans + (warp >> p.spans_log2)) * C::kScales * 8 + g) * kBytes;
    }
  };
  begin_item();
  auto fetch = [&]() {
    if (f_item < last && my_spans > 0) {
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        copy_async<16>(f_ring + f_slot + j * 512, f_codes[j]);
        f_codes[j] += 32 * WARPS;
        const uint8_t* const from = f_scales[j];
        const uint32_t to_scales = f_ring_scales + f_slot + j * 32 * C::kLane;
        f_scales[j] += f_step;
#pragma unroll
        for (int i = 0; i < C::kScales; ++i) {
          if constexpr (kBytes == 12) {
#pragma unroll
            for (int e = 0; e < 12; e += 4) copy_async<4>(to_scales + i * 12 + e, from + i * 96 + e);
          } else {
            copy_async<kBytes>(to_scales + i * kBytes, from + i * 8 * kBytes);
          }
        }
      }
      if (--f_left == 0) {
        f_left = my_spans, ++f_item;
        begin_item();
      }
      f_slot = f_slot == (C::kStages - 1) * C::kStage ? 0 : f_slot + C::kStage;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) fetch();

  Activations<T> x[RT];
  auto load_activations = [&](int i) {
    const int at = (warp + i * WARPS) * kSpan;
    const int wide = at + kSpan <= p.k ? p.wide : 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) x[r].load(rows[r], at + 8 * t, p.k, wide);
  };
  if (C::kEarly && my_spans > 0) load_activations(0);

  int slot = 0;
  for (int item = first; item < last; ++item) {
    float sum[TT][CT][4];
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
      for (int c = 0; c < CT; ++c) sum[j][c][0] = sum[j][c][1] = sum[j][c][2] = sum[j][c][3] = 0.f;
    for (int i = 0; i < my_spans; ++i) {
      uint32_t b[RT][C::kParts][4][2];
      if constexpr (!C::kEarly) load_activations(i);
#pragma unroll
      for (int r = 0; r < RT; ++r) x[r].pairs(b[r]);
      if constexpr (C::kEarly) load_activations(i + 1 < my_spans ? i + 1 : 0);  // the next item begins with span 0 again
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
      uint4 w4[TT];
      Scale<T, ZERO> scale[TT][C::kScales];
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        w4[j] = *reinterpret_cast<const uint4*>(ring + slot + j * 512);
#pragma unroll
        for (int e = 0; e < C::kScales; ++e)
          scale[j][e].load(ring_scales + slot + j * 32 * C::kLane + e * kBytes, operand.eight);
      }
      slot = slot == (C::kStages - 1) * C::kStage ? 0 : slot + C::kStage;
      fetch();
      __syncwarp();
#pragma unroll
      for (int j = 0; j < TT; ++j) {
        const uint32_t w[4] = {w4[j].x, w4[j].y, w4[j].z, w4[j].w};
        float acc[CT][4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const Scale<T, ZERO>& f = scale[j][C::kScales == 2 ? h / 2 : 0];
          const uint32_t a[4] = {operand.row(w[h], f.z0), operand.row8(w[h], f.z1), operand.row(w[h] >> 8, f.z0),
                                 operand.row8(w[h] >> 8, f.z1)};
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            if (h == 0 || (C::kScales == 2 && h == 2))
              mma<M, true>(acc[c], a, b[c / C::kParts][c % C::kParts][h][0], b[c / C::kParts][c % C::kParts][h][1]);
            else
              mma<M, false>(acc[c], a, b[c / C::kParts][c % C::kParts][h][0], b[c / C::kParts][c % C::kParts][h][1]);
            if (h == 3 || (C::kScales == 2 && h == 1)) {
              float(&y)[4] = sum[j][c];
              y[0] = fmaf(acc[c][0], f.s0, y[0]), y[1] = fmaf(acc[c][1], f.s0, y[1]);
              y[2] = fmaf(acc[c][2], f.s1, y[2]), y[3] = fmaf(acc[c][3], f.s1, y[3]);
            }
          }
        }
      }
    }

    // [warp][output][column], columns 2 t + e of 8 c
    float* const part_sum = reinterpret_cast<float*>(smem + WARPS * C::kStages * C::kStage);
#pragma unroll
    for (int j = 0; j < TT; ++j)
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const float(&y)[4] = sum[j][c];
        float* const to = part_sum + (warp * C::kOuts + 16 * j + g) * C::kColumns + 8 * c + 2 * t;
        *reinterpret_cast<float2*>(to) = make_float2(y[0], y[1]);
        *reinterpret_cast<float2*>(to + 8 * C::kColumns) = make_float2(y[2], y[3]);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < C::kOuts * C::kRows; i += WARPS * 32) {
      const int o = i % C::kOuts, r = i / C::kOuts, at = item * C::kOuts + o;
      if (at < p.n && row0 + r < p.m) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
#pragma unroll
          for (int j = 0; j < C::kParts; ++j)
            y += part_sum[(w * C::kOuts + o) * C::kColumns + (r / 8 * C::kParts + j) * 8 + r % 8];
        if (!std::is_same_v<M, __half>) y *= 0x1p12f;
        if (p.bias) y += to_f32(static_cast<const T*>(p.bias)[at]);
        static_cast<T*>(p.y)[(long long)(row0 + r) * p.ldy + at] = from_f32<T>(y);
      }
    }
    __syncthreads();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// One thread lays out one word (8 codes) of the weights.
__global__ void __launch_bounds__(256) pack_codes_kernel(const uint8_t* __restrict__ b, uint32_t* __restrict__ out, int n,
                                                         int k, int row_bytes, int spans, long long words) {
  const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (i >= words) return;
  const int h = (int)(i & 3), lane = (int)(i >> 2 & 31), g = lane >> 2, t = lane & 3;
  const long long span = i >> 7;
  const long long row = span / spans * 16 + g;
  const int at = (int)(span % spans) * kSpan + 32 * (h / 2) + 8 * t + 4 * (h % 2);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long r = row + 8 * e;
      uint32_t q = 8;  // past the end: met by zeros, or not kept
      if (r < n && at + j < k) q = (b[r * row_bytes + (at + j) / 2] >> (4 * ((at + j) & 1))) & 15;
      // of row g (e = 0): nibbles 0, 4, 2, 6; of row g + 8: 1, 5, 3, 7
      w |= q << (4 * ((j & 1) * 4 + (j >> 1) * 2 + e));
    }
  out[i] = w;
}

// One thread lays out one pair of scales (and zero points).
template <typename T, bool ZERO>
__global__ void __launch_bounds__(256)
    pack_scales_kernel(const T* __restrict__ scales, const uint8_t* __restrict__ zero, uint8_t* __restrict__ out, int n,
                       int groups, int padded, long long pairs) {
  using M = typename Traits<T>::type;
  const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (i >= pairs) return;
  const int g = (int)(i & 7), grp = (int)(i / 8 % padded);
  const long long tile = i / 8 / padded;
  uint8_t* p = out + i * Scale<T, ZERO>::kBytes;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const long long r = tile * 16 + g + 8 * e;
    const bool there = r < n && grp < groups;
    reinterpret_cast<T*>(p)[e] = there ? scales[r * groups + grp] : from_f32<T>(0.f);
    if (ZERO) {
      const int z = there ? (zero[r * ((groups + 1) / 2) + grp / 2] >> (4 * (grp & 1))) & 15 : 8;
      reinterpret_cast<uint16_t*>(p + 2 * sizeof(T))[e] = zero_bits<M>(z, e);
    }
  }
}

struct Staged {  // operands brought to the device for the time of laying them out
  void* p[3] = {};
  ~Staged() {
    for (void* x : p)
      if (x) cudaFree(x);
  }
};

int pack(Op* op, const uint8_t* b, const void* scales, const uint8_t* zero_points, const void* bias) {
  const size_t size = dtype_size(op->nb_dtype);
  const int n = op->N, k = op->K, block = op->nb_block;
  const long long groups = (k + block - 1) / block, tiles = (n + 15) / 16, spans = (k + kSpan - 1) / kSpan;
  const int kept = block == 32 ? (int)(2 * spans) : (int)groups;  // scales of a tile's row
  Staged staged;
  auto bring = [&](int i, const void* src, size_t bytes) {
    NNRCU_CUDA(cudaMalloc(&staged.p[i], bytes));
    NNRCU_CUDA(cudaMemcpy(staged.p[i], src, bytes, cudaMemcpyDefault));
    return (int)NNRCU_OK;
  };
  int rc = bring(0, b, n * groups * (block / 2));
  if (rc == NNRCU_OK) rc = bring(1, scales, n * groups * size);
  if (rc == NNRCU_OK && zero_points) rc = bring(2, zero_points, n * ((groups + 1) / 2));
  if (rc != NNRCU_OK) return rc;
  const long long words = tiles * spans * 128, pairs = tiles * kept * 8;
  NNRCU_CUDA(cudaMalloc(&op->wB, words * 4));
  NNRCU_CUDA(cudaMalloc(&op->nb_scale, pairs * (2 * size + (zero_points ? 4 : 0))));
  pack_codes_kernel<<<(unsigned)((words + 255) / 256), 256>>>(static_cast<const uint8_t*>(staged.p[0]),
                                                            static_cast<uint32_t*>(op->wB), n, k,
                                                            (int)(groups * (block / 2)), (int)spans, words);
  NNRCU_CUDA(cudaGetLastError());
  rc = with_type(op->nb_dtype, [&](auto t) {
    using T = decltype(t);
    auto* kernel = zero_points ? pack_scales_kernel<T, true> : pack_scales_kernel<T, false>;
    kernel<<<(unsigned)((pairs + 255) / 256), 256>>>(static_cast<const T*>(staged.p[1]),
                                                   static_cast<const uint8_t*>(staged.p[2]),
                                                   static_cast<uint8_t*>(op->nb_scale), n, (int)groups, kept, pairs);
    return cuda_check(cudaGetLastError(), "MatMulNBits layout launch");
  });
  if (rc != NNRCU_OK) return rc;
  if (bias) {
    NNRCU_CUDA(cudaMalloc(reinterpret_cast<void**>(&op->bias), n * size));
    NNRCU_CUDA(cudaMemcpy(op->bias, bias, n * size, cudaMemcpyDefault));
  }
  return cuda_check(cudaStreamSynchronize(nullptr), "MatMulNBits layout");
}

template <typename T, bool ZERO, int BLOCK, int RT, int TT, int WARPS>
int launch(const NbitsArgs& p, cudaStream_t st) {
  using C = Cfg<T, ZERO, BLOCK, RT, TT, WARPS>;
  auto* kernel = nbits_kernel<T, ZERO, BLOCK, RT, TT, WARPS>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use its shared memory
  int device = 0;
  NNRCU_CUDA(cudaGetDevice(&device));
  if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
    NNRCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    ready.fetch_or(1ull << device, std::memory_order_relaxed);
  }
  const int blocks = (int)(((long long)p.m + C::kRows - 1) / C::kRows), items = (p.n + C::kOuts - 1) / C::kOuts;
  for (int y0 = 0; y0 < blocks; y0 += 65535) {  // what a grid holds
    NbitsArgs q = p;
    const long long skip = (long long)y0 * C::kRows;
    q.a = static_cast<const T*>(p.a) + skip * p.lda;
    q.y = static_cast<T*>(p.y) + skip * p.ldy;
    q.m = (int)(p.m - skip);
    const int rows = blocks - y0 < 65535 ? blocks - y0 : 65535;
    // As many blocks as the SMs take at once, whose shares of the items differ
    // by one at most; the larger ones come first, one to each SM.
    const long long places = (long long)num_sms() * C::kBlocks;
    const int grid = (int)std::min<long long>(items, std::max(1LL, places / rows));
    q.items = items / grid;
    q.more = items % grid;
    using M = typename Traits<T>::type;
    Unpack<M> operand;
    for (int e = 0; e < 2; ++e) operand.eight[e] = zero_bits<M>(8, e) * 0x10001u;
    kernel<<<dim3(grid, rows), WARPS * 32, C::kSmem, st>>>(q, operand);
    NNRCU_CUDA(cudaGetLastError());
  }
  return NNRCU_OK;
}

// The more tiles a warp takes, the less it reads the activations and counts
// along again: two where every SM has work that way (1x16384x4096: 14.2 us and
// 15.8 with one; 16x14336x4096: 18.1 and 22.0). fp32 activations cost more to take
// apart than their codes to read, so there two are taken as soon as one a block
// leaves SMs with two blocks to do (8x2560x8192: 16.2 us and 18.5, 16x2400x4096:
// 14.3 and 20.5, 40x3000x3000: 20.5 and 30.7; single rows are the same). Where one
// tile a block leaves SMs without work, those that have some get twice the
// warps, so that twice the bytes are on their way (1x2048x4096: 4.2 us and 4.9,
// 16x2048x8192: 7.6 and 9.2).
template <typename T, bool ZERO, int BLOCK, int RT>
int launch_tiles(const NbitsArgs& p, cudaStream_t st) {
  const int tiles = (p.n + 15) / 16, sms = num_sms();
  if (tiles >= 2 * sms) return launch<T, ZERO, BLOCK, RT, 2, 8>(p, st);
  if constexpr (sizeof(T) == 4)
    if (tiles > sms && p.spans > 8) return launch<T, ZERO, BLOCK, RT, 2, RT == 1 ? 16 : 8>(p, st);
  if (tiles <= sms && p.spans > 8) return launch<T, ZERO, BLOCK, RT, 1, 16>(p, st);
  return launch<T, ZERO, BLOCK, RT, 1, 8>(p, st);
}

// Rows of a block: as many as there are, up to what the registers hold, for
// each block of rows reads and unpacks the codes again.
template <typename T, bool ZERO, int BLOCK>
int launch_rows(const NbitsArgs& p, cudaStream_t st) {
  if (p.m <= 8) return launch_tiles<T, ZERO, BLOCK, 1>(p, st);
  if (p.m <= 16 || sizeof(T) == 4) return launch_tiles<T, ZERO, BLOCK, 2>(p, st);
  return launch_tiles<T, ZERO, BLOCK, sizeof(T) == 4 ? 2 : 4>(p, st);
}

}  // namespace
}  // namespace nnrcu

using namespace nnrcu;

extern "C" {

int nnrcu_matmul_nbits_create(int k, int n, int block_size, int dtype, const uint8_t* b, const void* scales,
                              const uint8_t* zero_points, const void* bias, nnrcu_op** out) {
  if (!b || !scales || !out) return set_error(NNRCU_ERR_INVALID, "NULL argument");
  *out = nullptr;
  if (k < 1 || n < 1 || k > (1 << 30) || n > (1 << 30))
    return set_error(NNRCU_ERR_INVALID, "k and n must be positive and at most 2^30, got %d and %d", k, n);
  if (!dtype_ok(dtype)) return set_error(NNRCU_ERR_INVALID, "dtype must be fp32, bf16 or fp16");
  if (block_size != 32 && block_size != 64 && block_size != 128 && block_size != 256)
    return set_error(NNRCU_ERR_UNSUPPORTED, "block_size must be 32, 64, 128 or 256, got %d", block_size);
  nnrcu_op* op = new (std::nothrow) nnrcu_op();
  if (!op) return set_error(NNRCU_ERR_NOMEM, "out of host memory");
  op->kind = OP_MATMUL_NBITS;
  op->N = n;
  op->K = k;
  op->nb_block = block_size;
  op->nb_dtype = dtype;
  op->nb_zero = zero_points != nullptr;
  op->num_ops = 2LL * n * k;
  int rc = cuda_check(cudaGetDevice(&op->device), "cudaGetDevice");
  if (rc == NNRCU_OK) rc = pack(op, b, scales, zero_points, bias);
  if (rc != NNRCU_OK) {
    nnrcu_op_destroy(op);
    return rc;
  }
  *out = op;
  return NNRCU_OK;
}

int nnrcu_matmul_nbits_run(nnrcu_op* op, const void* a, int m, long long lda, void* y, long long ldy, void* stream) {
  if (!op || !a || !y) return set_error(NNRCU_ERR_INVALID, "NULL argument");
  if (op->kind != OP_MATMUL_NBITS) return set_error(NNRCU_ERR_INVALID, "not a MatMulNBits operator");
  int device = 0;
  NNRCU_CUDA(cudaGetDevice(&device));
  if (device != op->device)
    return set_error(NNRCU_ERR_INVALID, "the weights are on device %d, the current device is %d", op->device, device);
  if (m < 1 || (m > 1 && (lda < op->K || ldy < op->N)))
    return set_error(NNRCU_ERR_INVALID, "m = %d rows with strides %lld and %lld of k = %d and n = %d", m, lda, ldy,
                     op->K, op->N);
  NbitsArgs p{};
  p.a = a;
  p.y = y;
  p.lda = lda;
  p.ldy = ldy;
  p.m = m;
  p.n = op->N;
  p.k = op->K;
  p.spans = (op->K + kSpan - 1) / kSpan;
  p.codes = static_cast<const uint4*>(op->wB);
  p.scales = op->nb_scale;
  p.bias = op->bias;
  p.spans_log2 = op->nb_block == 256 ? 2 : (op->nb_block == 128 ? 1 : 0);
  p.scale_spans = (p.spans + (1 << p.spans_log2) - 1) >> p.spans_log2;
  auto starts_at = [&](int bytes) {
    return reinterpret_cast<uintptr_t>(a) % bytes == 0 && (m == 1 || lda * dtype_size(op->nb_dtype) % bytes == 0);
  };
  p.wide = starts_at(16) ? 2 : (starts_at(4) ? 1 : 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return with_type(op->nb_dtype, [&](auto t) {
    using T = decltype(t);
    if (op->nb_zero) return op->nb_block == 32 ? launch_rows<T, true, 32>(p, st) : launch_rows<T, true, 64>(p, st);
    return op->nb_block == 32 ? launch_rows<T, false, 32>(p, st) : launch_rows<T, false, 64>(p, st);
  });
}

}  // extern "C"
