// Causal attention of each sequence's newest tokens over a paged cache in 8
// or 4 bits, with a prefix that the whole batch shares:
//   y = sum_j p_j v_j,  p = softmax_j(scale * q . k_j) over the visible j.
// With key j's codes c_j and scale s_j (for each group of channels where
// there are several) and value j's codes d_j and scale r_j,
//   x_j = scale * s_j * (q . c_j),   y = sum_j (p_j r_j) d_j
// so both products run on the codes, which are exact in fp16, and the scales
// meet the logits and the weights in fp32.
#pragma once
#include <atomic>
#include <type_traits>

#include "decode.cuh"

namespace nnrcu {
namespace attn {

constexpr int kKeys = 32;   // keys of one warp's tile
constexpr int kWarps = 4;

// Codes to pairs of fp16, exactly. 8 bits (w with its sign bits flipped): the
// bytes that `sel` names under the top byte of 1024, less 1024 + 128. 4 bits:
// the nibbles at bits 0 and 16, 1024 + n less 1032.
// (The constants come as kernel parameters: known ones the compiler would set
// up again before each use, an instruction for each pair of codes.)
struct Unpack {
  uint32_t top = 0x64646464u, sign = 0x80808080u, eight_bits = 0x64806480u;
  uint32_t mask = 0x000F000Fu, ones = 0x64006400u, four_bits = 0x64086408u;
  __device__ __forceinline__ uint32_t from8(uint32_t w, uint32_t sel) const {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(__byte_perm(w, top, sel)), "r"(eight_bits));
    return r;
  }
  __device__ __forceinline__ uint32_t from4(uint32_t w) const {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(and_or(w, mask, ones)), "r"(four_bits));
    return r;
  }
};

struct Args {
  const void* q;
  void* y;
  long long q_batch, q_token, q_head;
  int dtype, batch, q_len, q_heads, heads, share, dim;
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  int pages, groups;      // groups: scales of a row
  int run;                // tokens that are sure to lie in a row on one page, from a multiple of it: 32, 16 or 1
  Divisor page;
  const int32_t* table;
  long long table_stride;
  const int32_t* lens;
  const int32_t* prefix_table;
  int max_len, prefix_len, window;
  float scale_log2;       // |scale| * log2(e)
  float q_sign;           // of scale
  int q_wide;             // q may be read 4 or 8 channels at a time, as a lane wants them
  int q_wide16;           // and 8 16-bit channels
  // Work on each sequence's own tokens, and on the prefix. A unit is one block
  // of rows of one cache head (of one sequence); it has a number of quads of
  // 128 keys. All units' quads in a row are shared out evenly over `grid`
  // blocks; one block's stretch of one unit is a segment, numbered unit +
  // block, which no other segment has. Each leaves for its rows
  //   ml: what p is relative to (a logit, log2 units) and the sum of p,
  //   o:  the mean of the values by p (their sum might pass fp32's range),
  // unless it is all of its unit and there is nothing to join.
  struct Part {
    int rows, blocks, units, grid;  // rows of a block; blocks of one head; units of one sequence
    float2* ml;                     // [segments][rows]
    float* o;                       // [segments][rows][dim]
  } own, prefix;
  int* status;
  Unpack codes;
};

__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Operands are fp16: codes are exact in it; q is scaled by a power of two for
// each row to lie below 2^15, where fp16 has 11 bits down to 2^-29 of that and
// steps of 2^-39 below. So are the weights p_j r_j, by a unit of each row's that
// puts the largest so far at 2^6 or more: a weight keeps 11 bits down to 2^-20
// of the largest weight, whatever larger values the row all but leaves out.
// A value of PARTS = 2 is the sum of two of them (22 bits): the weights of fp16
// and fp32 tensors, and fp32 queries. One would be enough for bf16 results,
// which keep 8 bits, but in fp16 it would cost as much as the result's own
// rounding does (error against 64 bits, 32 sequences of 5000: 2.9e-4 of the
// output with one, 2.1e-4 with two).
template <int PARTS>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&out)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const __half2 h = __floats2half2_rn(a, b);
    out[i] = *reinterpret_cast<const uint32_t*>(&h);
    if (i + 1 < PARTS) {
      const float2 f = __half22float2(h);
      a -= f.x, b -= f.y;
    }
  }
}

// A row's unit is 2^(e - 127), e from 6 to 245; its weights stay below 2^15.
constexpr int kFirstUnit = 245;
// The unit that puts a largest weight m at 2^6 or more (as far as the range
// goes); `before` is the unit in which the earlier weights' largest is there.
__device__ __forceinline__ int unit_for(float m, int before) {
  return 260 - min(max(max((int)(__float_as_uint(m) >> 23), 260 - before), 260 - kFirstUnit), 254);
}
// 2^-n for n from 0 on, 0 past fp32's range.
__device__ __forceinline__ float shrink_by(int n) { return n > 126 ? 0.f : __uint_as_float((127 - n) << 23); }
// By how many powers of two what is relative to ref shrinks when that rises to next.
__device__ __forceinline__ int rise_of(float ref, float next) { return next == -INFINITY ? 0 : (int)fminf(next - ref, 400.f); }

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t b0, const uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(there ? BYTES : 0)
               : "memory");
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Blocks on an SM at once: what registers and shared memory leave room for.
// (Three of 24 rows spilled: 79 us where two took 69.)
constexpr int blocks_of_sm(int dim, bool fp32, int rows) {
  if (dim > 128) return 2;
  if (rows == 24) return 2;
  if (rows == 8) return fp32 && dim > 64 ? 2 : 4;
  return fp32 && dim > 64 ? 2 : 3;
}

// Sizes of one kernel: fp16 parts of queries and of weights, head_dim padded to
// DP (EXACT: it is DP), 8 NT query rows.
template <int PARTS, int WPARTS, int BITS, bool GROUPED, int DP, bool EXACT, int NT>
struct Cfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kRowBytes = DP * BITS / 8;
  static constexpr int kChunks = kRowBytes / 16;          // 16-byte chunks of a row
  static constexpr int kChunkDim = 128 / BITS;            // channels of a chunk
  static constexpr int kSteps = kChunkDim / 16;           // tensor instructions over a chunk's channels
  static constexpr int kGroups = GROUPED ? DP / 32 : 1;
  static constexpr int kCodeBytes = kKeys * kRowBytes;    // of keys or of values
  static constexpr int kScaleBytes = kKeys * kGroups * 4;
  static constexpr int kSlot = kCodeBytes + kScaleBytes;  // keys or values of a tile
  static constexpr int kSlots = 3;
  // The products of 32 channels are summed apart: for each group's scale, and of
  // fp32 queries since the tensor cores cut off where an addition would round.
  static constexpr bool kApart = GROUPED || PARTS == 2;
  static constexpr bool kQShared = PARTS * NT * DP > 512;  // q's operands in shared memory, not in registers
  static constexpr int kQBytes = kQShared ? PARTS * DP * kRows * 2 : 0;
  static constexpr int kWarpBytes = kSlots * kSlot;
  static constexpr int kMergeRow = DP + 8;                // floats of a row when the warps are joined
  static constexpr int kMergeBytes = kWarps * kRows * kMergeRow * 4;
  static constexpr int kBody = kWarps * kWarpBytes > kMergeBytes ? kWarps * kWarpBytes : kMergeBytes;
  static constexpr int kSmem = kBody + kQBytes;
  static constexpr int kBlocks = blocks_of_sm(DP, PARTS == 2, kRows);
  // A chunk's place in its row: eight consecutive rows' chunks lie in
  // different banks.
  __device__ static uint32_t place(int row, int chunk) {
    constexpr int kRowsOfLine = kRowBytes >= 128 ? 1 : 128 / kRowBytes;
    constexpr int kMask = kRowBytes >= 128 ? 7 : kChunks - 1;
    return row * kRowBytes + ((chunk ^ ((row / kRowsOfLine) & kMask)) << 4);
  }
};

__device__ __forceinline__ int length_of(const Args& p, int b) {
  const int len = p.lens[b];
  return min(max(len, 0), p.max_len);
}

// One row's place: its sequence, token and query head (b < 0: the prefix, rows
// over the whole batch).
__device__ __forceinline__ void locate(const Args& p, int unit_b, int head, int r, int& b, int& i, int& h) {
  const int per = p.q_len * p.share;
  b = unit_b < 0 ? r / per : unit_b;
  const int in = unit_b < 0 ? r - b * per : r;
  i = in / p.share;
  h = head * p.share + in - i * p.share;
}

// The keys [lo, hi) of the unit's kind (own or prefix) that token i of a
// sequence with len tokens of its own sees. (Any window up to the largest int is
// taken, and positions before 0 see nothing: the comparisons stay in range.)
__device__ __forceinline__ void visible(const Args& p, bool own, int len, int i, int& lo, int& hi) {
  const int pos = p.prefix_len + len - p.q_len + i;
  const int first = p.window && pos >= p.window ? pos - p.window + 1 : 0;
  lo = own ? max(0, first - p.prefix_len) : first;
  hi = own ? min(len, pos + 1 - p.prefix_len) : min(p.prefix_len, pos + 1);
}

constexpr int kQuad = kWarps * kKeys;
// Where the keys of a sequence's units start, a multiple of kKeys, and how
// many quads they are (one at least, so that every row is written).
__device__ __forceinline__ int first_key(const Args& p, bool own, int len) {
  return own && p.window && len - p.q_len >= p.window ? (len - p.q_len - p.window + 1) / kKeys * kKeys : 0;
}
__device__ __forceinline__ int quads_of(const Args& p, bool own, int b) {
  const int len = own ? length_of(p, b) : p.prefix_len;
  return max(1, (len - first_key(p, own, len) + kQuad - 1) / kQuad);
}
// How the quads are shared out (a warp's lanes add up those of all sequences;
// the host sees to it that there are fewer than 2^31).
struct Shares {
  int total, share, before;  // before: those of the sequences before b
};
__device__ __forceinline__ Shares shares_of(const Args& p, bool own, int lane, int b) {
  const Args::Part w = own ? p.own : p.prefix;
  int sum = 0, before = 0;
  for (int at = lane; at < (own ? p.batch : 1); at += 32) {
    const int n = quads_of(p, own, at);
    sum += n;
    before += at < b ? n : 0;
  }
  Shares s;
  s.total = __reduce_add_sync(~0u, sum) * w.units;
  s.before = __reduce_add_sync(~0u, before) * w.units;
  s.share = (s.total + w.grid - 1) / w.grid;
  return s;
}

// The kernel for the sequences' own tokens may run beside the end of the one
// for their prefix: it waits for that before it ends itself, so that what comes
// after it has both.
__device__ __forceinline__ void after_prefix(const Args& p, bool own) {
  if (own && p.prefix_len) pdl_wait();
}

// Where in a part's work a block is: sequence (-1: the prefix), unit, quad of
// the unit and how many the unit has.
struct Start {
  int b, unit, quad, quads;
};
// Where quad at_quad of all is; false only if lengths change while this runs.
__device__ __forceinline__ bool first_unit(const Args& p, bool own, int lane, int at_quad, Start& at) {
  const Args::Part w = own ? p.own : p.prefix;
  int before = 0;
  at.b = -1;
  if (own) {
    for (int b0 = 0; b0 < p.batch && at.b < 0; b0 += 32) {
      int sum = b0 + lane < p.batch ? quads_of(p, own, b0 + lane) : 0;
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += x;
      }
      const uint32_t past = __ballot_sync(~0u, at_quad < (before + sum) * w.units);
      const int hit = past ? __ffs(past) - 1 : 32;
      if (hit > 0) before += __shfl_sync(~0u, sum, hit - 1);
      if (past) at.b = b0 + hit;
    }
    if (at.b < 0 || at.b >= p.batch) return false;
  }
  at.quads = quads_of(p, own, at.b);
  const int in = at_quad - before * w.units;
  at.unit = in / at.quads;
  at.quad = in - at.unit * at.quads;
  return at.unit < w.units;
}
// The next unit's first quad; false if there is none.
__device__ __forceinline__ bool next_unit(const Args& p, bool own, int units, Start& at) {
  at.quad = 0;
  if (++at.unit < units) return true;
  at.unit = 0;
  if (!own || ++at.b >= p.batch) return false;
  at.quads = quads_of(p, own, at.b);
  return true;
}

// N consecutive channels of q.
template <typename T, int N>
__device__ __forceinline__ void load_q(float* x, const void* base, long long at, bool wide) {
  const T* src = static_cast<const T*>(base) + at;
  if (wide) {
    struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Wide {
      T v[N];
    };
    const Wide w = *reinterpret_cast<const Wide*>(src);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = to_f32(w.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = to_f32(src[j]);
  }
}

__device__ __forceinline__ void store_y(const Args& p, long long at, float v) {
  if (p.dtype == NNRCU_DT_F32)
    static_cast<float*>(p.y)[at] = v;
  else if (p.dtype == NNRCU_DT_BF16)
    static_cast<__nv_bfloat16*>(p.y)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p.y)[at] = __float2half_rn(v);
}

// One block's segments, one after the other: 8 NT query rows that share a
// cache head, over a stretch of keys.
// Each warp takes every fourth tile of 32 keys through its own ring of three
// cp.async slots, which hold the keys of a tile, its values and the next
// tile's keys in turn, and keeps its own running softmax; the four are joined
// at the end. The products are taken transposed,
//   S^T [keys x rows] = C q^T,   O^T [channels x rows] += D^T (p r)^T
// so that the codes are the 16-row operands and few query rows cost few
// registers and little softmax; the weights change places between lanes by
// one 8x8 transposition for each 8 keys.
// 8 rows over 8 bits (32 sequences of 8192, 8 heads, bf16): 353 MB in 67 us,
// 5.3 TB/s, bound by the cache's way from HBM with 16 warps on an SM (fp16, whose
// weights have two parts: 70 us). 24 rows over 4 bits (7 sequences, 20001 of
// 30000 visible, scales of 32 channels): the whole call 60 us in bf16 and 70 in
// fp16, where 28.4 M warp instructions, some 1600 a tile, take less than half of
// the issue slots: 8 warps on an SM, for which the registers suffice, do not hide
// their latencies.
template <int PARTS, int WPARTS, int BITS, bool GROUPED, int DP, bool EXACT, int NT>
__global__ void __launch_bounds__(kWarps * 32, Cfg<PARTS, WPARTS, BITS, GROUPED, DP, EXACT, NT>::kBlocks)
    attend_kernel(const __grid_constant__ Args p, const bool own) {
  using C = Cfg<PARTS, WPARTS, BITS, GROUPED, DP, EXACT, NT>;
  constexpr int kOf = C::kChunkDim / 4;  // channels of a chunk that one lane holds
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int dim = EXACT ? DP : p.dim, groups = EXACT ? C::kGroups : p.groups;

  pdl_launch();
  const Args::Part w = own ? p.own : p.prefix;
  const Shares shares = shares_of(p, own, lane, 0);
  int at_quad = blockIdx.x * shares.share;
  const int stop = min(shares.total, at_quad + shares.share);
  Start at{};
  if (at_quad >= stop || !first_unit(p, own, lane, at_quad, at)) return after_prefix(p, own);

  // Each row's place in q and y and the keys that it sees.
  __shared__ long long row_q[C::kRows], row_y[C::kRows];
  __shared__ int row_lo[C::kRows], row_hi[C::kRows];
  __shared__ float2 warp_ml[kWarps][C::kRows];
  __shared__ float4 row_part[C::kRows];
  for (;;) {
    const int n_quads = min(at.quads - at.quad, stop - at_quad);
    const int head = at.unit / w.blocks, first_row = (at.unit - head * w.blocks) * C::kRows;
    const int len = own ? length_of(p, at.b) : 0;
    const int rows = own ? p.q_len * p.share : p.batch * p.q_len * p.share;
    if (own && threadIdx.x == 0 && len != p.lens[at.b]) report(p.status, ST_LENGTH);
    if (threadIdx.x < C::kRows) {
      const int r = first_row + threadIdx.x;
      row_lo[threadIdx.x] = 0, row_hi[threadIdx.x] = 1 << 30;  // a row past the end sees everything and is not kept
      row_y[threadIdx.x] = -1;
      if (r < rows) {
        int b, i, h;
        locate(p, at.b, head, r, b, i, h);
        visible(p, own, own ? len : length_of(p, b), i, row_lo[threadIdx.x], row_hi[threadIdx.x]);
        row_q[threadIdx.x] = b * p.q_batch + i * p.q_token + h * p.q_head;
        row_y[threadIdx.x] = ((long long)b * p.q_len + i) * p.q_heads + h;
      }
    }
    __syncthreads();
    // What all of this lane's rows 8 n + 2 t + e see, and any does.
    int all_lo = 0, all_hi = 1 << 30, any_lo = 1 << 30, any_hi = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int lo = row_lo[8 * n + 2 * t + e], hi = row_hi[8 * n + 2 * t + e];
        if (row_y[8 * n + 2 * t + e] >= 0 && hi > lo) any_lo = min(any_lo, lo), any_hi = max(any_hi, hi);
        all_lo = max(all_lo, lo), all_hi = min(all_hi, hi);
      }
    any_lo = __reduce_min_sync(~0u, any_lo);
    any_hi = __reduce_max_sync(~0u, any_hi);
    all_lo = __reduce_max_sync(~0u, all_lo);
    all_hi = __reduce_min_sync(~0u, all_hi);
    // tiles start at multiples of kKeys, so that runs of rows on a page stay together
    const int unit_key = first_key(p, own, len), first_quad_key = unit_key + at.quad * kQuad;
    const int end = min(first_quad_key + n_quads * kQuad, any_hi);
    const int begin = max(first_quad_key, any_lo / kKeys * kKeys);
    const int tiles = end > begin ? (end - begin + kKeys - 1) / kKeys : 0;
    const int my_tiles = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;

    uint8_t* const mine = smem + warp * C::kWarpBytes;
    const uint32_t mine_s = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
    const int32_t* const table = own ? p.table + at.b * p.table_stride : p.prefix_table;

    // The page of key `lane` of a tile, one tile ahead of its copies.
    auto page_of = [&](int n) -> int {
      const int j = begin + (n * kWarps + warp) * kKeys + lane;
      return n < my_tiles && j < end ? table[div_by(j, p.page)] : -1;
    };
    int next_page = page_of(0);
    long long row = 0;     // key `lane` of the newest tile on its way, as a row of the buffers
    uint32_t next_valid;   // that tile's mask of keys that are there
    // Copies one tile's codes and scales, of keys or of values. What is copied
    // for keys that are not there lies in the cache too and is hidden; their
    // scales are zeros.
    auto copy = [&](int slot, const uint8_t* codes, const float* scale) {
      const uint32_t base = mine_s + slot * C::kSlot;
      const uint32_t scales = base + C::kCodeBytes + lane * C::kGroups * 4;
      const bool there = (next_valid >> lane) & 1;
      if constexpr (!GROUPED) {
        copy_async<4>(scales, scale + row, there);
      } else if (groups % 4 == 0) {
        for (int e = 0; e < groups; e += 4) copy_async<16>(scales + e * 4, scale + row * groups + e, there);
      } else {
        for (int e = 0; e < groups; ++e) copy_async<4>(scales + e * 4, scale + row * groups + e, there);
      }
      const int bytes = dim * BITS / 8;
      constexpr int kAtOnce = 32 / C::kChunks;  // rows that the warp copies at once
      const int c = lane % C::kChunks, r = lane / C::kChunks;
      if (p.run > 1) {  // two runs of 16 rows
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint8_t* const from = codes + (__shfl_sync(~0u, row, half * 16) + r) * bytes + c * 16;
          if (c * 16 < bytes) {
#pragma unroll
            for (int i = 0; i < 16; i += kAtOnce) copy_async16(base + C::place(half * 16 + i + r, c), from + i * bytes);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kKeys; i += kAtOnce) {
          const uint8_t* const from = codes + __shfl_sync(~0u, row, i + r) * bytes + c * 16;
          if (c * 16 < bytes) copy_async16(base + C::place(i + r, c), from);
        }
      }
    };
    auto fetch_keys = [&](int n, int slot) {
      next_valid = 0;
      if (n < my_tiles) {
        const int j = begin + (n * kWarps + warp) * kKeys + lane;
        const int page = next_page;
        next_page = page_of(n + 1);
        const bool in = j < end, there = in && (unsigned)page < (unsigned)p.pages;
        if (in && !there && j >= any_lo) report(p.status, ST_PAGE);  // a key that no row sees may lack its page
        next_valid = __ballot_sync(~0u, there);
        row = there ? ((long long)page * p.heads + head) * p.page.d + (j - div_by(j, p.page) * p.page.d) : 0;
        copy(slot, p.k, p.k_scale);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto fetch_values = [&](int n, int slot) {
      if (n < my_tiles) copy(slot, p.v, p.v_scale);
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch_keys(0, 0);
    fetch_values(0, 1);

    // q as operands: row 8 n + g, channels in the order in which the key codes
    // come, each row scaled by a power of two to lie below 2^15
    uint32_t qf[C::kQShared ? 1 : PARTS][NT][C::kQShared ? 1 : DP / 16][2];
    uint2* const q_shared = reinterpret_cast<uint2*>(smem + C::kBody);
    // Of rows 2 t + e: what their logits are in. A power of two, so that the
    // largest logit and what it is less than by one multiplication and addition
    // are the same number however large it is; key scales carry the rest.
    float row_scale[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool real = row_y[8 * n + g] >= 0;
      const long long at = real ? row_q[8 * n + g] : 0;
      float x[C::kChunks][kOf];
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        const int ch = c * C::kChunkDim + t * kOf;
#pragma unroll
        for (int j = 0; j < kOf; ++j) x[c][j] = 0.f;
        if (real && ch < dim && tiles > 0) {
          if (PARTS == 2)
            load_q<float, kOf>(x[c], p.q, at + ch, p.q_wide);
          else if (WPARTS == 1)
            load_q<__nv_bfloat16, kOf>(x[c], p.q, at + ch, p.q_wide);
          else
            load_q<__half, kOf>(x[c], p.q, at + ch, p.q_wide);
        }
#pragma unroll
        for (int j = 0; j < kOf; ++j) most = fmaxf(most, fabsf(x[c][j]));
      }
      most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
      most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
      const uint32_t exponent = min(max(__float_as_uint(most) >> 23, 15u), 254u);
      const float f = __uint_as_float((268 - exponent) << 23) * p.q_sign;  // 2^(14 - E), E = exponent - 127
      const float back = __uint_as_float((exponent - 14) << 23);
#pragma unroll
      for (int e = 0; e < 2; ++e) row_scale[n][e] = __shfl_sync(~0u, back, (2 * t + e) * 4);
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
        for (int s = 0; s < C::kSteps; ++s) {
          uint32_t w[2][PARTS];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // 8 bits: channels 2 half, 2 half + 1; 4 bits: i and i + 4, i = 2 s + half
            const int a0 = BITS == 8 ? 2 * half : 2 * s + half, a1 = BITS == 8 ? a0 + 1 : a0 + 4;
            split_pair<PARTS>(x[c][a0] * f, x[c][a1] * f, w[half]);
          }
#pragma unroll
          for (int i = 0; i < PARTS; ++i) {
            if constexpr (C::kQShared) {
              if (c % kWarps == warp)
                q_shared[((i * NT + n) * (DP / 16) + c * C::kSteps + s) * 32 + lane] = make_uint2(w[0][i], w[1][i]);
            } else {
              qf[i][n][c * C::kSteps + s][0] = w[0][i], qf[i][n][c * C::kSteps + s][1] = w[1][i];
            }
          }
        }
    }
    if constexpr (C::kQShared) __syncthreads();

    const Unpack& codes = p.codes;
    constexpr int kTiles = DP / 16;  // 16 channels each
    float o[kTiles][NT][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
    // ref: what p is relative to, a whole number at most 6 below the largest
    // logit; unit: of the weights p r and of o
    float ref[NT][2], l[NT][2];
    int unit[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) ref[n][e] = -INFINITY, l[n][e] = 0.f, unit[n][e] = kFirstUnit;
    float most_unit = 0.f;  // the largest of the warp's rows that have seen a key

    int slot = 0;  // of this tile's keys; its values are in the next one
    for (int n_tile = 0; n_tile < my_tiles; ++n_tile) {
      const uint32_t mask = next_valid;
      const int slot_v = slot == 2 ? 0 : slot + 1, slot_next = slot == 0 ? 2 : slot - 1;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      fetch_keys(n_tile + 1, slot_next);
      __syncwarp();  // the copies' lanes part where a row is short, and what follows wants them together
      const uint32_t k_s = mine_s + slot * C::kSlot, v_s = mine_s + slot_v * C::kSlot;
      const float* const ks = reinterpret_cast<const float*>(mine + slot * C::kSlot + C::kCodeBytes);
      const float* const vs = reinterpret_cast<const float*>(mine + slot_v * C::kSlot + C::kCodeBytes);

      // logits: s[i][n][e]: key 16 i + g + 8 (e >> 1), row 8 n + 2 t + (e & 1)
      float s[kKeys / 16][NT][4];
#pragma unroll
      for (int i = 0; i < kKeys / 16; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
        float part[NT][4];
#pragma unroll
        for (int c = 0; c < C::kChunks; c += 2) {
          if (c * C::kChunkDim < dim) {
            uint32_t w[4];  // {keys 0-7, chunk c}, {0-7, c + 1}, {8-15, c}, {8-15, c + 1}
            ldsm4<false>(w, k_s + C::place(i * 16 + (lane >> 4) * 8 + (lane & 7), c + ((lane >> 3) & 1)));
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              if (C::kApart && (BITS == 4 || cc == 0))
#pragma unroll
                for (int n = 0; n < NT; ++n) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.f;
              const uint32_t x0 = BITS == 8 ? w[cc] ^ codes.sign : w[cc];
              const uint32_t x1 = BITS == 8 ? w[2 + cc] ^ codes.sign : w[2 + cc];
#pragma unroll
              for (int st = 0; st < C::kSteps; ++st) {
                const uint32_t a[4] = {BITS == 8 ? codes.from8(x0, 0x4140) : codes.from4(x0 >> (8 * st)),
                                       BITS == 8 ? codes.from8(x1, 0x4140) : codes.from4(x1 >> (8 * st)),
                                       BITS == 8 ? codes.from8(x0, 0x4342) : codes.from4(x0 >> (8 * st + 4)),
                                       BITS == 8 ? codes.from8(x1, 0x4342) : codes.from4(x1 >> (8 * st + 4))};
                const int step = (c + cc) * C::kSteps + st;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int j = 0; j < PARTS; ++j) {
                    uint2 b;
                    if constexpr (C::kQShared)
                      b = q_shared[((j * NT + n) * (DP / 16) + step) * 32 + lane];
                    else
                      b = make_uint2(qf[j][n][step][0], qf[j][n][step][1]);
                    mma(C::kApart ? part[n] : s[i][n], a, b.x, b.y);
                  }
              }
              if constexpr (GROUPED) {  // 8 bits: two chunks are a group; 4 bits: one is
                const int grp = BITS == 4 ? c + cc : c / 2;
                if ((BITS == 4 || cc == 1) && grp < groups) {
                  const float f0 = ks[(i * 16 + g) * C::kGroups + grp] * p.scale_log2;
                  const float f1 = ks[(i * 16 + 8 + g) * C::kGroups + grp] * p.scale_log2;
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    s[i][n][0] = fmaf(part[n][0], f0, s[i][n][0]), s[i][n][1] = fmaf(part[n][1], f0, s[i][n][1]);
                    s[i][n][2] = fmaf(part[n][2], f1, s[i][n][2]), s[i][n][3] = fmaf(part[n][3], f1, s[i][n][3]);
                  }
                }
              } else if constexpr (C::kApart) {
                if (BITS == 4 || cc == 1)
#pragma unroll
                  for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][n][e] += part[n][e];
              }
            }
          }
        }
        if constexpr (!GROUPED) {
          const float f0 = ks[i * 16 + g] * p.scale_log2, f1 = ks[i * 16 + 8 + g] * p.scale_log2;
#pragma unroll
          for (int n = 0; n < NT; ++n) s[i][n][0] *= f0, s[i][n][1] *= f0, s[i][n][2] *= f1, s[i][n][3] *= f1;
        }
      }
      const int first = begin + (n_tile * kWarps + warp) * kKeys;
      const bool partial = mask != ~0u || first < all_lo || first + kKeys > all_hi;
      if (partial) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const int lo = row_lo[8 * n + 2 * t + f], hi = row_hi[8 * n + 2 * t + f];
#pragma unroll
            for (int i = 0; i < kKeys / 16; ++i)
#pragma unroll
              for (int e = f; e < 4; e += 2) {
                const int in = i * 16 + 8 * (e >> 1) + g, at = first + in;
                const bool hidden = (((mask >> in) & 1) == 0) | (at < lo) | (at >= hi);
                s[i][n][e] = hidden ? -INFINITY : s[i][n][e];
              }
          }
      }

      // The values have come; the next ones take the keys' slot.
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      fetch_values(n_tile + 1, slot);
      __syncwarp();
      slot = slot_next;

      // Running softmax. What p is relative to moves only when a logit passes it
      // by 2^6: p stays below that, and o is seldom rescaled. Nor does the unit
      // move before some r_j could take a weight past 2^15.
      bool grown = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[0][n][e], s[0][n][2 + e]);
#pragma unroll
          for (int i = 1; i < kKeys / 16; ++i) x = fmaxf(x, fmaxf(s[i][n][e], s[i][n][2 + e]));
          top[n][e] = x * row_scale[n][e];
          grown |= top[n][e] > ref[n][e] + 6.f;
        }
      // The largest r_j of key j.
      auto largest = [&](int key) {
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < C::kGroups; ++e)
          if (e == 0 || e < groups) x = fmaxf(x, fabsf(vs[key * C::kGroups + e]));
        return x;
      };
      grown |= largest(lane) * most_unit >= 0x1p9f;
      const bool moves = __any_sync(~0u, grown);
      if (moves) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[n][e];
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
            x = fmaxf(ceilf(x), ref[n][e]);
            const int rise = rise_of(ref[n][e], x);
            ref[n][e] = x;
            l[n][e] *= shrink_by(rise);
            unit[n][e] += rise;  // what o, as it stands, is in now
          }
      }
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float r0 = ref[n][0] == -INFINITY ? 0.f : ref[n][0], r1 = ref[n][1] == -INFINITY ? 0.f : ref[n][1];
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[i][n][e] = exp2_fast(fmaf(s[i][n][e], row_scale[n][e & 1], -(e & 1 ? r1 : r0)));
            l[n][e & 1] += s[i][n][e];
          }
      }
      if (moves) {
        float r[kKeys / 16][2];
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i) r[i][0] = largest(i * 16 + g), r[i][1] = largest(i * 16 + 8 + g);
        most_unit = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < kKeys / 16; ++i) x = fmaxf(x, fmaxf(s[i][n][e] * r[i][0], s[i][n][2 + e] * r[i][1]));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
            x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
            const int next = unit_for(x, unit[n][e]);
            const float by = shrink_by(unit[n][e] - next);
            unit[n][e] = next;
            if (ref[n][e] > -INFINITY) most_unit = fmaxf(most_unit, __uint_as_float(next << 23));
#pragma unroll
            for (int i = 0; i < kTiles; ++i) o[i][n][e] *= by, o[i][n][2 + e] *= by;
          }
        most_unit = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(most_unit)));
      }
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < kKeys / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][n][e] *= __uint_as_float(unit[n][e & 1] << 23);

      // o += D^T (p r)^T
#pragma unroll
      for (int i = 0; i < kKeys / 16; ++i) {
        uint32_t b[NT][WPARTS][2];
        auto weights = [&](int grp) {
          const float f0 = vs[(i * 16 + g) * C::kGroups + grp], f1 = vs[(i * 16 + 8 + g) * C::kGroups + grp];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float w[4] = {s[i][n][0] * f0, s[i][n][1] * f0, s[i][n][2] * f1, s[i][n][3] * f1};
            if (partial) {  // nothing of a hidden key, whatever its scale is
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (s[i][n][e] == 0.f) w[e] = 0.f;
            }
            uint32_t x[WPARTS], y[WPARTS];
            split_pair<WPARTS>(w[0], w[1], x);
            split_pair<WPARTS>(w[2], w[3], y);
#pragma unroll
            for (int j = 0; j < WPARTS; ++j) b[n][j][0] = transpose8x8(x[j]), b[n][j][1] = transpose8x8(y[j]);
          }
        };
        if constexpr (!GROUPED) weights(0);
#pragma unroll
        for (int c = 0; c < C::kChunks; c += 2) {
          if (c * C::kChunkDim < dim) {
            if constexpr (GROUPED && BITS == 8) weights(c / 2);
            uint32_t w[4];  // keys 0-7 and 8-15 of chunk c, then of chunk c + 1
            ldsm4<true>(w, v_s + C::place(i * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), c + (lane >> 4)));
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              if constexpr (GROUPED && BITS == 4) weights(c + cc);
              const uint32_t x0 = BITS == 8 ? w[2 * cc] ^ codes.sign : w[2 * cc];
              const uint32_t x1 = BITS == 8 ? w[2 * cc + 1] ^ codes.sign : w[2 * cc + 1];
#pragma unroll
              for (int st = 0; st < C::kSteps; ++st) {
                const uint32_t a[4] = {BITS == 8 ? codes.from8(x0, 0x4240) : codes.from4(x0 >> (8 * st)),
                                       BITS == 8 ? codes.from8(x0, 0x4341) : codes.from4(x0 >> (8 * st + 4)),
                                       BITS == 8 ? codes.from8(x1, 0x4240) : codes.from4(x1 >> (8 * st)),
                                       BITS == 8 ? codes.from8(x1, 0x4341) : codes.from4(x1 >> (8 * st + 4))};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  float(&sum)[4] = o[(c + cc) * C::kSteps + st][n];
                  float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                  for (int j = 0; j < WPARTS; ++j) mma(PARTS == 2 ? part : sum, a, b[n][j][0], b[n][j][1]);
                  if constexpr (PARTS == 2) {  // as kApart: over 8192 keys 5e-7 of the output, 1.4e-6 without
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] += part[e];
                  }
                }
              }
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // Join the four warps. o's fragment: lane g holds channels 2 g, 2 g + 1 of a
    // chunk (8 bits), 4 g + 2 st, + 1 of a chunk's half st (4 bits).
    __syncthreads();
    float* const mo = reinterpret_cast<float*>(smem) + warp * C::kRows * C::kMergeRow;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[n][e];
        x += __shfl_xor_sync(~0u, x, 4);
        x += __shfl_xor_sync(~0u, x, 8);
        x += __shfl_xor_sync(~0u, x, 16);
        const int r = 8 * n + 2 * t + e;
        const float real = __uint_as_float((254 - unit[n][e]) << 23), part = x == 0.f ? 0.f : 1.f / x;
        if (g == 0) warp_ml[warp][r] = make_float2(ref[n][e], x);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const int at = BITS == 8 ? i * 16 + 2 * g : i / 2 * 32 + 4 * g + 2 * (i % 2);
          *reinterpret_cast<float2*>(mo + r * C::kMergeRow + at) =
              make_float2(o[i][n][e] * part * real, o[i][n][2 + e] * part * real);
        }
      }
    __syncthreads();
    const bool whole = n_quads == at.quads && !p.prefix_len;
    const long long segment = ((own ? (long long)at.b * w.units : 0) + at.unit + blockIdx.x) * C::kRows;
    if (threadIdx.x < C::kRows) {  // the warps' shares in a row
      const int r = threadIdx.x;
      float most = -INFINITY, total = 0.f, f[kWarps];
#pragma unroll
      for (int i = 0; i < kWarps; ++i) most = fmaxf(most, warp_ml[i][r].x);
      const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        f[i] = warp_ml[i][r].y == 0.f ? 0.f : warp_ml[i][r].y * exp2_fast(warp_ml[i][r].x - base);
        total += f[i];
      }
      const float part = total == 0.f ? 0.f : 1.f / total;
      row_part[r] = make_float4(f[0] * part, f[1] * part, f[2] * part, f[3] * part);
      if (!whole && row_y[r] >= 0) w.ml[segment + r] = make_float2(most, total);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < C::kRows * DP; x += kWarps * 32) {
      const int r = x / DP, c = x % DP;
      const long long row = row_y[r];
      if (row < 0 || c >= dim) continue;
      static_assert(kWarps == 4, "a share each");
      const float* const mean = reinterpret_cast<const float*>(smem) + r * C::kMergeRow + c;
      constexpr int kFar = C::kRows * C::kMergeRow;
      const float4 f = row_part[r];
      const float y = (mean[0] * f.x + mean[kFar] * f.y) + (mean[2 * kFar] * f.z + mean[3 * kFar] * f.w);
      if (whole)
        store_y(p, row * dim + c, y);
      else
        w.o[(segment + r) * dim + c] = y;
    }
    at_quad += n_quads;
    if (at_quad >= stop || !next_unit(p, own, w.units, at)) break;
    __syncthreads();
  }
  after_prefix(p, own);
}

template <typename K>
int launch_part(K kernel, const Args& p, bool own, int threads, int smem, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(own ? p.own.grid : p.prefix.grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = own && p.prefix_len && pdl_enabled() ? 1 : 0;  // see after_prefix
  return cuda_check(cudaLaunchKernelEx(&cfg, kernel, p, own), "attention launch");
}

template <int PARTS, int WPARTS, int BITS, bool GROUPED, int DP, bool EXACT, int NT>
int launch(const Args& p, bool own, cudaStream_t st) {
  using C = Cfg<PARTS, WPARTS, BITS, GROUPED, DP, EXACT, NT>;
  auto* kernel = attend_kernel<PARTS, WPARTS, BITS, GROUPED, DP, EXACT, NT>;
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may use its shared memory
  int device = 0;
  NNRCU_CUDA(cudaGetDevice(&device));
  if (!(ready.load(std::memory_order_relaxed) >> device & 1)) {
    NNRCU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    ready.fetch_or(1ull << device, std::memory_order_relaxed);
  }
  return launch_part(kernel, p, own, kWarps * 32, C::kSmem, st);
}

// Query rows of a block: as few blocks of up to 24 rows as there can be, since
// each reads the keys again, and of these the smallest. 7 x 3 rows over 20000
// 4-bit tokens: one block of 24 60 us in bf16 and 70 in fp16, two of 16 71 and
// 86. Past 128 channels 8 are what registers hold with two blocks on an SM: 12
// rows over 32 sequences of 4096, dimension 256, two blocks of 8 177 us, one of
// 16 256 us; 4-bit groups of 32, 16 rows, 103 and 156 us; fp32 38 and 46 us.
inline int rows_of_block(long long rows, int dim) {
  const long long most = dim > 128 ? 8 : 24, blocks = (rows + most - 1) / most;
  return (int)(((rows + blocks - 1) / blocks + 7) / 8 * 8);
}
// The kernel for blocks of 128 rows (kv_attention_many.cu).
int launch_many(const Args& p, int bits, bool own, cudaStream_t st);

template <int PARTS, int WPARTS, int BITS>
int launch_for(const Args& p, bool own, cudaStream_t st) {
  const int rows = own ? p.own.rows : p.prefix.rows;
  auto go = [&](auto grouped, auto tiles) {
    constexpr bool G = decltype(grouped)::value;
    constexpr int N = decltype(tiles)::value;
    if (p.dim == 64) return launch<PARTS, WPARTS, BITS, G, 64, true, N>(p, own, st);
    if (p.dim == 128) return launch<PARTS, WPARTS, BITS, G, 128, true, N>(p, own, st);
    if (p.dim < 64) return launch<PARTS, WPARTS, BITS, G, 64, false, N>(p, own, st);
    if (p.dim < 128) return launch<PARTS, WPARTS, BITS, G, 128, false, N>(p, own, st);
    return launch<PARTS, WPARTS, BITS, G, 256, false, 1>(p, own, st);  // rows_of_block gives no more
  };
  auto by_rows = [&](auto grouped) {
    if (rows == 8) return go(grouped, std::integral_constant<int, 1>());
    if (rows == 16) return go(grouped, std::integral_constant<int, 2>());
    return go(grouped, std::integral_constant<int, 3>());
  };
  return p.groups > 1 ? by_rows(std::true_type()) : by_rows(std::false_type());
}

// The instances of launch_for, each in a file of its own.
int launch_bf16_b8(const Args& p, bool own, cudaStream_t st);
int launch_bf16_b4(const Args& p, bool own, cudaStream_t st);
int launch_f16_b8(const Args& p, bool own, cudaStream_t st);
int launch_f16_b4(const Args& p, bool own, cudaStream_t st);
int launch_f32_b8(const Args& p, bool own, cudaStream_t st);
int launch_f32_b4(const Args& p, bool own, cudaStream_t st);

}  // namespace attn
}  // namespace nnrcu
