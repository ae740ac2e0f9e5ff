// Attention of many query rows over the same keys: a prefix that the batch
// shares, or a chunk of a prompt. There the products bound it, 4 dim
// operations for each row and key, and they run on tcgen05: blocks of 128 rows
// by tiles of 128 keys,
//   S [rows x keys] = q C^T,   O [rows x channels] += (p r) D
// with S and O in tensor memory. The codes become fp16 in shared memory once
// for the 128 rows, exactly; scales meet logits and weights in fp32, as in
// kv_attention.cuh, whose division of the work and numbers this kernel keeps.
//
// Warps 0-7:  softmax, two threads a row (each half of a tile's keys), which
//             agree on what the row's weights are relative to.
// Warps 8-11: codes; each thread brings its own 16 bytes two tiles ahead
//             (cp.async) and makes them fp16. Warp 12: the products.
// Two S are in flight, so that the products of one tile overlap the softmax of
// another; keys and values are made fp16 in one buffer each, since they are
// wanted at different times. A tile is 1048 cycles of products
// (dim 128); the softmax warps keep theirs near that by working on pairs
// (packed fp32), 64 logits a thread, in code short enough for the instruction
// cache. With its chain from the codes through S, the weights and O a tile takes
// some 4000 cycles, of which the softmax passes are half; the start, with q and
// the first tiles, and the end, with the segments' means, take some 15000
// together. 128 rows of each of 8 heads over a
// prefix of 16384 (8 bits, dim 128, bf16), the whole call: 47 us, and 84 with the
// kernel for few rows; 256 rows: 67 us, in fp16 with its second product 78.
#include "kv_attention.cuh"
#include "ptx.cuh"

namespace nnrcu {
namespace attn {
namespace {

constexpr int kM = 128, kN = 128, kRing = 4;  // rows, keys of a tile, tiles whose scales are kept
constexpr int kThreads = 416;

enum Bar { K_FULL, K_EMPTY, V_FULL, V_EMPTY, S_FULL, S_FREE = S_FULL + 2, P_FULL = S_FREE + 2, O_DONE, Q_FULL, MEET, BARS = MEET + 4 };

template <int BITS, int DIM>
struct Many {
  static constexpr int kSlab = kM * 128;  // 128 rows of 64 fp16
  static constexpr int kTileBytes = DIM / 64 * kSlab;
  static constexpr int kQ = 0, kK = kQ + kTileBytes, kV = kK + kTileBytes, kP = kV + kTileBytes;
  static constexpr int kCodes = kN * DIM * BITS / 8;     // a tile's keys or values as they lie in the cache
  static constexpr int kRaw = kP + 2 * kSlab;            // [2 tiles][keys, values]
  static constexpr int kScales = kRaw + 2 * 2 * kCodes;  // [kRing][128] of keys, then of values
  static constexpr int kMasks = kScales + 2 * kRing * kN * 4;
  static constexpr int kWidest = kMasks + kRing * 16;    // [kRing][4 warps]
  static constexpr int kMeet = kWidest + kRing * 16;  // [2][half][row]
  static constexpr int kBars = kMeet + 2 * 2 * kM * 4;
  static constexpr int kEnd = kBars + (BARS + 8) * 8;
  static constexpr int kSmem = kEnd + 1024;  // the tiles start at a multiple of 1024
};

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// As above, 16 columns, without waiting.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// D += A B with A in tensor memory: a lane a row, two 16-bit numbers a column.
__device__ __forceinline__ void mma_f16_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc)
      : "memory");
}

// Waits for the phase with this parity without asking to be suspended (a tile
// passes five such waits in turn); bounded as ptx::mbar_wait is.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint32_t at = ptx::smem_u32(bar);
  long long t0 = 0;
  for (uint32_t i = 0;; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(at), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 255u) == 255u) {
      if (*abort_flag) return false;
      const long long now = clock64();
      if (t0 == 0)
        t0 = now;
      else if (now - t0 > (long long)(2 * NNRCU_WAIT_NS))
        return false;
    }
  }
}

// A 16-byte chunk of one row in a slab of 128-byte rows with the 128-byte swizzle.
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// Descriptor of an operand whose contiguous direction is not the summed one
// (values: channels contiguous, keys summed) in slabs of 64 channels: 8 keys
// are 1024 bytes, the next 64 channels a slab further.
__device__ __forceinline__ uint64_t desc_values(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(16384 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// FINE: fp16 tensors, whose weights are held in two parts (see kv_attention.cuh).
// The second goes to the 64 columns of tensor memory that S and O leave, as the
// operand of a second product.
template <int BITS, int DIM, bool FINE>
__global__ void __launch_bounds__(kThreads, 1) attend_many_kernel(const __grid_constant__ Args p, const bool own) {
  using L = Many<BITS, DIM>;
  constexpr int kChunks = DIM * BITS / 128;     // 16-byte chunks of a row's codes
  constexpr int kLoads = kChunks;               // of a loading thread for its warp's 32 keys
  constexpr int kRowsAtOnce = 32 / kChunks;     // rows that a warp brings at once
  extern __shared__ uint8_t raw[];
  uint8_t* const smem = raw + ((1024 - (ptx::smem_u32(raw) & 1023)) & 1023);  // tiles start at a multiple of 1024
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  int* const words = reinterpret_cast<int*>(bars + BARS);  // 0: tensor memory, 1: abort, 2, 3: any_lo, any_hi
  volatile int* const abort_flag = words + 1;
  float* const scales = reinterpret_cast<float*>(smem + L::kScales);
  uint32_t* const masks = reinterpret_cast<uint32_t*>(smem + L::kMasks);
  float* const widests = reinterpret_cast<float*>(smem + L::kWidest);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch();
  if (warp == 12) ptx::tmem_alloc(reinterpret_cast<uint32_t*>(words), 512);
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < BARS; ++i) {
      const bool from_mma = i == K_EMPTY || i == V_EMPTY || i == S_FULL || i == S_FULL + 1 || i == O_DONE;
      const bool from_softmax = i == S_FREE || i == S_FREE + 1 || i == P_FULL || i == Q_FULL;
      ptx::mbar_init(bars + i, from_mma ? 1 : (from_softmax ? 256 : (i >= MEET ? 64 : 128)));
    }
    ptx::fence_mbar_init();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = words[0], t_o = tmem + 256, t_rest = tmem + 384;

  const Args::Part w = own ? p.own : p.prefix;
  const Shares shares = shares_of(p, own, lane, 0);
  int at_quad = blockIdx.x * shares.share;
  const int stop = min(shares.total, at_quad + shares.share);
  Start at{};
  const bool any = at_quad < stop && first_unit(p, own, lane, at_quad, at);
  int done = 0;  // tiles of earlier segments: what the barriers' phases go by
  int segments = 0, met = 0;
  // Waits for the phase in which a barrier completes for the n-th time (from 0).
  auto wait = [&](int bar, int n) {
    if (wait_phase(bars + bar, n & 1, abort_flag)) return true;
    *abort_flag = 1;
    report(p.status, ST_WAIT);
    return false;
  };

  for (bool more = any; more;) {
    const int n_quads = min(at.quads - at.quad, stop - at_quad);
    const int head = at.unit / w.blocks, first_row = (at.unit - head * w.blocks) * kM;
    const int len = own ? length_of(p, at.b) : 0;
    const int rows = own ? p.q_len * p.share : p.batch * p.q_len * p.share;
    if (own && threadIdx.x == 0 && len != p.lens[at.b]) report(p.status, ST_LENGTH);
    // Each softmax thread's row: its place in q and y and the keys that it sees.
    long long row_q = 0, row_y = -1;
    int lo = 0, hi = 1 << 30;
    if (threadIdx.x == 0) words[2] = 1 << 30, words[3] = 0;
    __syncthreads();
    const int row = threadIdx.x % kM;
    if (warp < 8 && first_row + row < rows) {
      int b, i, h;
      locate(p, at.b, head, first_row + row, b, i, h);
      visible(p, own, own ? len : length_of(p, b), i, lo, hi);
      row_q = b * p.q_batch + i * p.q_token + h * p.q_head;
      row_y = ((long long)b * p.q_len + i) * p.q_heads + h;
      if (hi > lo) atomicMin(words + 2, lo), atomicMax(words + 3, hi);
    }
    __syncthreads();
    const int any_lo = words[2], any_hi = words[3];
    const int quad_key = first_key(p, own, len) + at.quad * kQuad;
    const int end = min(quad_key + n_quads * kQuad, any_hi);
    const int begin = max(quad_key, any_lo / kKeys * kKeys);
    const int tiles = end > begin ? (end - begin + kN - 1) / kN : 0;

    if (warp < 8) {
      // ---------------------------------------------------------------- softmax
      const int half = warp / 4, r = row;
      const uint32_t lanes = (uint32_t)(warp % 4 * 32) << 16;
      float* const meet = reinterpret_cast<float*>(smem + L::kMeet);
      // The other half's value of x; `met` counts these meetings.
      auto other = [&](float x, bool& ok) {
        float* const at2 = meet + (met & 1) * 2 * kM;
        at2[half * kM + r] = x;
        ptx::mbar_arrive(bars + MEET + warp % 4);
        ok = __all_sync(~0u, wait(MEET + warp % 4, met));
        ++met;
        return at2[(1 - half) * kM + r];
      };
      float row_scale = 0.f;
      bool ok = true;
      if (tiles > 0) {  // q: each half its channels, scaled by a power of two so that the whole row lies below 2^15
        float x[DIM / 2], most = 0.f;
#pragma unroll
        for (int c = 0; c < DIM / 16; ++c) {
          const long long at_q = row_q + half * (DIM / 2) + 8 * c;
          if (row_y < 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[8 * c + j] = 0.f;
          } else {
            load_q<std::conditional_t<FINE, __half, __nv_bfloat16>, 8>(x + 8 * c, p.q, at_q, p.q_wide16);
          }
        }
#pragma unroll
        for (int j = 0; j < DIM / 2; ++j) most = fmaxf(most, fabsf(x[j]));
        __syncwarp();
        most = fmaxf(most, other(most, ok));
        const uint32_t exponent = min(max(__float_as_uint(most) >> 23, 15u), 254u);
        const float f = __uint_as_float((268 - exponent) << 23) * p.q_sign;
        row_scale = __uint_as_float((exponent - 14) << 23);  // key scales carry the rest, see kv_attention.cuh
#pragma unroll
        for (int c = 0; c < DIM / 16; ++c) {
          uint32_t y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t z[1];
            split_pair<1>(x[8 * c + 2 * j] * f, x[8 * c + 2 * j + 1] * f, z);
            y[j] = z[0];
          }
          const int chunk = half * (DIM / 16) + c;
          *reinterpret_cast<uint4*>(smem + L::kQ + chunk / 8 * L::kSlab + chunk_at(r, chunk % 8)) =
              make_uint4(y[0], y[1], y[2], y[3]);
        }
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(bars + Q_FULL);
      }
      float ref = -INFINITY;
      float2 l = make_float2(0.f, 0.f), l2 = make_float2(0.f, 0.f);
      int unit = kFirstUnit;
      float room = 268.f - kFirstUnit;  // what p's and r's exponents may be together for a weight to stay below 2^15
      for (int n = 0; n < tiles && ok; ++n) {
        const int g = done + n, buf = g & 1, slot = g % kRing;
        const int first = begin + n * kN;
        ok = __all_sync(~0u, wait(S_FULL + buf, g >> 1));  // the tile's scales came before its keys
        if (!ok) break;
        ptx::tc_fence_after();
        const float* const ks = scales + slot * kN;
        const float* const vs = scales + (kRing + slot) * kN;
        // Which of 32 keys, from the c-th 32 of the tile, this row sees.
        auto seen = [&](int c) -> uint32_t {
          const int from = lo - (first + 32 * c), to = hi - (first + 32 * c);
          const uint32_t above = from <= 0 ? ~0u : (from >= 32 ? 0u : ~0u << from);
          const uint32_t below = to >= 32 ? ~0u : (to <= 0 ? 0u : ~(~0u << to));
          return masks[slot * 4 + c] & above & below;
        };
        // This half's 64 logits less the row's factor.
        float2 x[2][16];
        uint32_t vis[2];
        {
          uint32_t s[2][32];
#pragma unroll
          for (int c = 0; c < 2; ++c) ptx::tmem_ld32_async(tmem + lanes + buf * 128 + 64 * half + 32 * c, s[c]);
#pragma unroll
          for (int c = 0; c < 2; ++c) vis[c] = seen(2 * half + c);
#pragma unroll
          for (int c = 0; c < 2; ++c) ptx::tmem_wait_ld(s[c]);
          ptx::tc_fence_before();
          ptx::mbar_arrive(bars + S_FREE + buf);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 f = *reinterpret_cast<const float4*>(ks + 64 * half + 32 * c + 4 * j);
              x[c][2 * j] = __fmul2_rn(make_float2(__uint_as_float(s[c][4 * j]), __uint_as_float(s[c][4 * j + 1])),
                                       make_float2(f.x, f.y));
              x[c][2 * j + 1] = __fmul2_rn(make_float2(__uint_as_float(s[c][4 * j + 2]), __uint_as_float(s[c][4 * j + 3])),
                                           make_float2(f.z, f.w));
            }
        }
        const bool partial = __any_sync(~0u, (vis[0] & vis[1]) != ~0u);
        if (partial) {
          __syncwarp();  // keeps this a branch: few tiles have hidden keys
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (!((vis[c] >> (2 * j)) & 1)) x[c][j].x = -INFINITY;
              if (!((vis[c] >> (2 * j + 1)) & 1)) x[c][j].y = -INFINITY;
            }
        }
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < 16; ++j) most[j & 3] = fmaxf(most[j & 3], fmaxf(x[c][j].x, x[c][j].y));
        float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * row_scale;
        top = fmaxf(top, other(top, ok));
        if (!ok) break;
        // the exponent of the largest value scale of a key that some row sees
        const float4 four = *reinterpret_cast<const float4*>(widests + slot * 4);
        const float widest = fmaxf(fmaxf(four.x, four.y), fmaxf(four.z, four.w));
        // p passes 2^8, or a weight may pass 2^15: p is at most 2^(top - ref)
        const float above = top - ref;
        const bool moves = __any_sync(~0u, above > 8.f || above + widest > room);
        ok = __all_sync(~0u, n == 0 || wait(O_DONE, g - 1));  // the last tile's weights are used, and O holds it
        if (!ok) break;
        const float2 factor = make_float2(row_scale, row_scale);
        if (moves) {  // the same in both halves
          const float next = fmaxf(ceilf(top), ref);
          const int rise = rise_of(ref, next);
          const float keep = shrink_by(rise), base = next == -INFINITY ? 0.f : next;
          ref = next;
          l.x *= keep, l.y *= keep, l2.x *= keep, l2.y *= keep;
          unit += rise;  // what O, as it stands, is in now
          float m[2] = {0.f, 0.f};  // the tile's largest weight
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float2 r = *reinterpret_cast<const float2*>(vs + 64 * half + 32 * c + 2 * j);
              const float2 q = __ffma2_rn(x[c][j], factor, make_float2(-base, -base));
              m[0] = fmaxf(m[0], exp2_fast(q.x) * fabsf(r.x)), m[1] = fmaxf(m[1], exp2_fast(q.y) * fabsf(r.y));
            }
          float most_weight = fmaxf(m[0], m[1]);
          most_weight = fmaxf(most_weight, other(most_weight, ok));
          if (!ok) break;
          const int fit = unit_for(most_weight, unit), by = unit - fit;
          unit = fit, room = 268.f - (float)fit;
          if (n > 0 && __any_sync(~0u, by != 0)) {
            const float f = shrink_by(by);
            ptx::tc_fence_after();
#pragma unroll 1
            for (int i = half * (DIM / 64); i < (half + 1) * (DIM / 64); ++i) {
              uint32_t o[32];
              ptx::tmem_ld32(t_o + lanes + 32 * i, o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st32(t_o + lanes + 32 * i, o);
            }
          }
        }
        if constexpr (FINE) ptx::tc_fence_after();  // the last tile's second product has used what is written below
        const float base = ref == -INFINITY ? 0.f : ref, times = __uint_as_float(unit << 23);
        const float2 minus = make_float2(-base, -base), per_unit = make_float2(times, times);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float4 f = *reinterpret_cast<const float4*>(vs + 64 * half + 32 * c + 2 * j);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float2 q = __ffma2_rn(x[c][j + e], factor, minus);
              q = make_float2(exp2_fast(q.x), exp2_fast(q.y));
              (j & 2 ? l2 : l) = __fadd2_rn(j & 2 ? l2 : l, q);
              x[c][j + e] = __fmul2_rn(__fmul2_rn(q, per_unit), e ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
            }
          }
          if (partial) {  // nothing of a hidden key, whatever its scale is
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (!((vis[c] >> (2 * j)) & 1)) x[c][j].x = 0.f;
              if (!((vis[c] >> (2 * j + 1)) & 1)) x[c][j].y = 0.f;
            }
          }
          uint32_t rest[16];
#pragma unroll
          for (int j = 0; j < 4; ++j) {  // the chunk's 4 of the row's 16
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t z[FINE ? 2 : 1];
              split_pair<FINE ? 2 : 1>(x[c][4 * j + e].x, x[c][4 * j + e].y, z);
              y[e] = z[0];
              if constexpr (FINE) rest[4 * j + e] = z[1];
            }
            *reinterpret_cast<uint4*>(smem + L::kP + half * L::kSlab + chunk_at(r, 4 * c + j)) =
                make_uint4(y[0], y[1], y[2], y[3]);
          }
          if constexpr (FINE) tmem_st16(t_rest + lanes + 32 * half + 16 * c, rest);
        }
        if constexpr (FINE) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before();
        ptx::mbar_arrive(bars + P_FULL);
      }
      float sum = (l.x + l.y) + (l2.x + l2.y);
      if (tiles > 0) {
        bool meets = true;
        if (ok) sum += other(sum, meets);
        ok = ok && meets;
        if (ok) ok = __all_sync(~0u, wait(O_DONE, done + tiles - 1));
      }
      ptx::tc_fence_after();
      const bool whole = n_quads == at.quads && !p.prefix_len;
      const long long segment = ((own ? (long long)at.b * w.units : 0) + at.unit + blockIdx.x) * kM + r;
      const float real = tiles > 0 && ok && sum != 0.f ? __uint_as_float((254 - unit) << 23) : 0.f;
      const float part = real == 0.f ? 0.f : 1.f / sum;  // the mean is kept, as in kv_attention.cuh
      // O by 32 channels through shared memory (every product has ended), so
      // that a store is one row's 32 and not one channel of 32 rows.
      float* const turn = reinterpret_cast<float*>(smem + L::kK) + warp * 32 * 33;
      const uint32_t kept = __ballot_sync(~0u, row_y >= 0);
#pragma unroll 1
      for (int i = half * (DIM / 64); i < (half + 1) * (DIM / 64); ++i) {
        uint32_t o[32];
        if (tiles > 0 && ok) {
          ptx::tmem_ld32(t_o + lanes + 32 * i, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0;
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) turn[lane * 33 + j] = __uint_as_float(o[j]) * part * real;
        __syncwarp();
        if (whole) {
#pragma unroll 4
          for (int j = 0; j < 32; ++j) {
            const long long to = __shfl_sync(~0u, row_y, j);
            if (to >= 0) store_y(p, to * DIM + 32 * i + lane, turn[j * 33 + lane]);
          }
        } else {
          float* const to = w.o + (segment - lane) * DIM + 32 * i + lane;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if ((kept >> j) & 1) to[j * DIM] = turn[j * 33 + lane];
        }
        __syncwarp();
      }
      if (row_y >= 0 && !whole && half == 0) w.ml[segment] = make_float2(ref, sum);
      ptx::tc_fence_before();
    } else if (warp < 12) {
      // ---------------------------------------------------------------- codes
      const int key = threadIdx.x - 256;  // of the tile; the warp brings its 32 keys' codes, chunk c of row r0 + i kRowsAtOnce
      const int c = lane % kChunks, r0 = lane / kChunks, row0 = (warp - 8) * 32;
      const int32_t* const table = own ? p.table + at.b * p.table_stride : p.prefix_table;
      const Unpack& codes = p.codes;
      uint8_t* const raw_mine = smem + L::kRaw + key * 16;  // this thread's 16 bytes, 2048 apart
      auto page_of = [&](int n) -> int {
        const int j = begin + n * kN + key;
        return n < tiles && j < end ? table[div_by(j, p.page)] : -1;
      };
      int next_page = page_of(0);
      long long rows_k = 0, rows_v = 0;  // key `key` of the newest tile of keys on its way, and of the one before
      auto copy_codes = [&](const uint8_t* base, long long my_row, uint32_t to) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          copy_async16(to + i * 2048,
                       base + __shfl_sync(~0u, my_row, r0 + i * kRowsAtOnce) * (DIM * BITS / 8) + c * 16);
      };
      const uint32_t raw_at = ptx::smem_u32(raw_mine);
      // Begins to bring tile n's scales and keys (its pages came a tile earlier) ...
      auto bring_keys = [&](int n) {
        rows_v = rows_k;
        if (n < tiles) {
          const int j = begin + n * kN + key, page = next_page, slot = (done + n) % kRing;
          next_page = page_of(n + 1);
          const bool there = j < end && (unsigned)page < (unsigned)p.pages;
          if (j < end && !there && j >= any_lo) report(p.status, ST_PAGE);  // as in kv_attention.cuh
          const uint32_t mask = __ballot_sync(~0u, there);
          rows_k = there ? ((long long)page * p.heads + head) * p.page.d + (j - div_by(j, p.page) * p.page.d) : 0;
          copy_async<4>(ptx::smem_u32(scales + slot * kN + key), p.k_scale + rows_k, there);
          copy_async<4>(ptx::smem_u32(scales + (kRing + slot) * kN + key), p.v_scale + rows_k, there);
          if (lane == 0) masks[slot * 4 + warp - 8] = mask;
          copy_codes(p.k, rows_k, raw_at + (n & 1) * 2 * L::kCodes);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      // ... and its values; the newest keys on their way are those of `of`, n or n + 1.
      auto bring_values = [&](int n, int of) {
        if (n < tiles) copy_codes(p.v, of == n ? rows_k : rows_v, raw_at + (n & 1) * 2 * L::kCodes + L::kCodes);
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      auto convert = [&](const uint8_t* from, uint8_t* to) {
        uint4 x[kLoads];  // all at once: the stores below may not pass loads
#pragma unroll
        for (int i = 0; i < kLoads; ++i) x[i] = *reinterpret_cast<const uint4*>(from + i * 2048);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int at_row = row0 + r0 + i * kRowsAtOnce;
          const uint32_t word[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
          constexpr int kOut = 64 / BITS / 4;  // 16-byte chunks of fp16 that one of codes becomes: 2 or 4
          uint4 y[kOut];
          if constexpr (BITS == 8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a = word[2 * h] ^ codes.sign, b = word[2 * h + 1] ^ codes.sign;
              y[h] = make_uint4(codes.from8(a, 0x4140), codes.from8(a, 0x4342), codes.from8(b, 0x4140), codes.from8(b, 0x4342));
            }
          } else {
#pragma unroll
            for (int h = 0; h < 4; ++h) {  // nibbles n and n + 4 come together
              const uint32_t a = codes.from4(word[h]), b = codes.from4(word[h] >> 4), d = codes.from4(word[h] >> 8),
                             e = codes.from4(word[h] >> 12);
              y[h] = make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(d, e, 0x5410), __byte_perm(a, b, 0x7632),
                                __byte_perm(d, e, 0x7632));
            }
          }
#pragma unroll
          for (int h = 0; h < kOut; ++h) {
            const int chunk = c * kOut + h;
            *reinterpret_cast<uint4*>(to + chunk / 8 * L::kSlab + chunk_at(at_row, chunk % 8)) = y[h];
          }
        }
      };
      // Keys a tile ahead of values: S of the next tile is wanted before O of this one.
      auto keys = [&](int n) {
        const int g = done + n, slot = g % kRing;
        if (!__all_sync(~0u, g == 0 || wait(K_EMPTY, g - 1))) return false;
        const int j = begin + n * kN + key;
        scales[slot * kN + key] *= p.scale_log2;
        const uint32_t r_bits = __float_as_uint(scales[(kRing + slot) * kN + key]) & 0x7FFFFFFFu;
        const bool counts = j >= any_lo && j < any_hi && r_bits < 0x7F800000u;  // a hidden key's is 0
        const uint32_t widest = __reduce_max_sync(~0u, counts ? r_bits >> 23 : 0u);
        if (lane == 0) widests[slot * 4 + warp - 8] = (float)widest;
        convert(raw_mine + (n & 1) * 2 * L::kCodes, smem + L::kK);
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(bars + K_FULL);
        __syncwarp();
        return true;
      };
      bring_keys(0);
      bring_values(0, 0);
      bring_keys(1);
      bring_values(1, 1);
      asm volatile("cp.async.wait_group 3;" ::: "memory");
      bool ok = tiles == 0 || keys(0);
      bring_keys(2);
      for (int n = 0; n < tiles && ok; ++n) {
        const int g = done + n;
        // On their way, oldest first: values n, keys n + 1 (or these two the
        // other way round), values n + 1 and keys n + 2 (likewise).
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        if (n + 1 < tiles) ok = keys(n + 1);
        if (!ok) break;
        ok = __all_sync(~0u, g == 0 || wait(V_EMPTY, g - 1));  // tile n - 1 is done with: so are its scales
        if (!ok) break;
        bring_keys(n + 3);
        convert(raw_mine + (n & 1) * 2 * L::kCodes + L::kCodes, smem + L::kV);
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(bars + V_FULL);
        __syncwarp();
        bring_values(n + 2, n + 3);
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else if (lane == 0) {
      // ---------------------------------------------------------------- products
      const uint32_t base = ptx::smem_u32(smem);
      const uint32_t idesc_s = ptx::umma_idesc(1, 0, 0, kM, kN);
      const uint32_t idesc_o = ptx::umma_idesc(1, 0, 0, kM, DIM) | 1u << 16;  // values: not transposed in memory
      bool ok = tiles == 0 || wait(Q_FULL, segments);
      auto scores = [&](int g) {
        const int buf = g & 1;
        if (!wait(K_FULL, g) || (g >= 2 && !wait(S_FREE + buf, (g >> 1) - 1))) return false;
        ptx::tc_fence_after();
#pragma unroll
        for (int s = 0; s < DIM / 16; ++s) {
          const uint32_t off = s / 4 * L::kSlab + s % 4 * 32;
          ptx::mma_f16(tmem + buf * 128, ptx::umma_desc_sw128(base + L::kQ + off),
                       ptx::umma_desc_sw128(base + L::kK + off), idesc_s, s > 0);
        }
        ptx::mma_commit(bars + S_FULL + buf);
        ptx::mma_commit(bars + K_EMPTY);
        return true;
      };
      if (ok && tiles > 0) ok = scores(done);
      for (int n = 0; n < tiles && ok; ++n) {
        const int g = done + n;
        if (n + 1 < tiles && !scores(g + 1)) break;
        if (!wait(V_FULL, g) || !wait(P_FULL, g)) break;
        ptx::tc_fence_after();
#pragma unroll
        for (int s = 0; s < kN / 16; ++s)
          ptx::mma_f16(t_o, ptx::umma_desc_sw128(base + L::kP + s / 4 * L::kSlab + s % 4 * 32),
                       desc_values(base + L::kV + s * 2048), idesc_o, n > 0 || s > 0);
        if constexpr (FINE) {
#pragma unroll
          for (int s = 0; s < kN / 16; ++s)  // 16 keys are 8 columns
            mma_f16_tmem(t_o, t_rest + 8 * s, desc_values(base + L::kV + s * 2048), idesc_o);
        }
        ptx::mma_commit(bars + V_EMPTY);
        ptx::mma_commit(bars + O_DONE);
      }
    }
    done += tiles;
    segments += tiles > 0;
    at_quad += n_quads;
    __syncwarp();
    __syncthreads();
    more = at_quad < stop && !*abort_flag && next_unit(p, own, w.units, at);
  }
  if (*abort_flag) ptx::settle_ns(200000);  // let what was issued end
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 12) ptx::tmem_dealloc(tmem, 512);
  after_prefix(p, own);
}

template <int BITS, int DIM, bool FINE>
int launch(const Args& p, bool own, cudaStream_t st) {
  auto* kernel = attend_many_kernel<BITS, DIM, FINE>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use its shared memory
  int device = 0;
  NNRCU_CUDA(cudaGetDevice(&device));
  if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
    NNRCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<BITS, DIM>::kSmem));
    ready.fetch_or(1ull << device, std::memory_order_relaxed);
  }
  return launch_part(kernel, p, own, kThreads, Many<BITS, DIM>::kSmem, st);
}

}  // namespace

int launch_many(const Args& p, int bits, bool own, cudaStream_t st) {
  auto go = [&](auto fine) {
    constexpr bool F = decltype(fine)::value;
    if (p.dim == 64) return bits == 8 ? launch<8, 64, F>(p, own, st) : launch<4, 64, F>(p, own, st);
    return bits == 8 ? launch<8, 128, F>(p, own, st) : launch<4, 128, F>(p, own, st);
  };
  return p.dtype == NNRCU_DT_F16 ? go(std::true_type()) : go(std::false_type());
}

}  // namespace attn
}  // namespace nnrcu
