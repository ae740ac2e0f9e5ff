// Attention over a paged 8- or 4-bit cache: argument checks, the division of
// the work and the launch (kv_attention.cuh has the kernels).
#include <algorithm>
#include <climits>
#include <cmath>

#include "kv_attention.cuh"

namespace nnrcu {
namespace {

using attn::Args;

int check(const nnrcu_kv_cache* c, const nnrcu_kv_attention_desc* d, bool buffers) {
  const int rc = kv_cache_check(c, buffers);
  if (rc != NNRCU_OK) return rc;
  if (!d) return set_error(NNRCU_ERR_INVALID, "desc is NULL");
  if (!dtype_ok(d->dtype)) return set_error(NNRCU_ERR_INVALID, "dtype must be fp32, bf16 or fp16");
  if (d->batch < 0 || d->q_len < 1 || d->q_heads < 1 || d->q_heads % c->heads)
    return set_error(NNRCU_ERR_INVALID, "batch %d, q_len %d, q_heads %d over %d cache heads", d->batch, d->q_len,
                     d->q_heads, c->heads);
  if ((long long)d->batch * d->q_len * d->q_heads >= (1LL << 31))
    return set_error(NNRCU_ERR_INVALID, "too many query rows");
  if (d->max_len < 0 || d->table_pages < 0 || d->max_len > (long long)d->table_pages * c->page_size)
    return set_error(NNRCU_ERR_INVALID, "max_len %d does not fit %d pages of %d tokens", d->max_len, d->table_pages,
                     c->page_size);
  if (d->batch > 1 && d->table_stride < d->table_pages)
    return set_error(NNRCU_ERR_INVALID, "table_stride %lld is below table_pages %d", d->table_stride, d->table_pages);
  if (d->prefix_len < 0 || d->prefix_pages < 0 || d->prefix_len > (long long)d->prefix_pages * c->page_size)
    return set_error(NNRCU_ERR_INVALID, "prefix_len %d does not fit %d pages of %d tokens", d->prefix_len,
                     d->prefix_pages, c->page_size);
  if ((long long)d->prefix_len + d->max_len >= (1LL << 30))
    return set_error(NNRCU_ERR_INVALID, "prefix_len + max_len must be below 2^30");
  if (d->window < 0) return set_error(NNRCU_ERR_INVALID, "window must not be negative");
  if (!(d->scale > -INFINITY && d->scale < INFINITY)) return set_error(NNRCU_ERR_INVALID, "scale must be finite");
  return NNRCU_OK;
}

// Rows of a key/value head from which the blocks of 128 are worth their fixed
// cost, and as many as take the kernel for few rows two blocks, or three. A
// prefix of 16384 keys, 8 heads, few against many (us), bf16: 8 bits and
// dimension 128, 32 rows 40.8 and 41.1, 40 rows 50.5 and 41.4; 16 sequences of
// 8192, 32 rows 59 and 68, 40 rows 74 and 68. With less to do for a key the two
// meet later: 4 bits, 48 rows 39.7 and 40.9, 64 rows 47.1 and 41.0; dimension 64,
// 48 rows 30.7 and 34.7, 64 rows 35.0 and 34.8. fp16: 32 rows 43.2 and 46.8, 40
// rows 52.8 and 46.9; 4 bits 48 rows 43.0 and 46.8, 64 rows 51.4 and 47.1.
constexpr int many_rows(int bits, int dim) { return bits == 8 && dim == 128 ? 40 : 56; }

// How the work is divided (one sequence at least): what runs at once on the SMs,
// or a block for each quad of keys where those are fewer.
void divide(const nnrcu_kv_cache& c, const nnrcu_kv_attention_desc& d, Args* p) {
  const long long rows = (long long)d.q_len * (d.q_heads / c.heads);
  // Many rows go to the kernel for blocks of 128, which has its products on
  // tcgen05, for what it is made for: 16-bit tensors, one scale a row.
  const bool many = d.dtype != NNRCU_DT_F32 && (c.group == 0 || c.group == c.head_dim) &&
                    (c.head_dim == 64 || c.head_dim == 128);
  auto part = [&](long long rows, long long sequences, int keys) {
    Args::Part w{};
    w.rows = many && rows >= many_rows(c.bits, c.head_dim) ? 128 : attn::rows_of_block(rows, c.head_dim);
    w.blocks = (int)((rows + w.rows - 1) / w.rows);
    w.units = w.blocks * c.heads;
    const long long quads = std::max(1LL, ((long long)keys + attn::kQuad - 1) / attn::kQuad);
    const long long at_once =
        (long long)num_sms() * (w.rows == 128 ? 1 : attn::blocks_of_sm(c.head_dim, d.dtype == NNRCU_DT_F32, w.rows));
    w.grid = (int)std::min(at_once, sequences * w.units * quads);
    return w;
  };
  p->prefix = d.prefix_len ? part(rows * d.batch, 1, d.prefix_len) : Args::Part{};
  p->own = part(rows, d.batch, d.max_len);
}

// Whether the units may be cut, so that there is something to join.
bool joined(const nnrcu_kv_attention_desc& d) { return d.prefix_len || d.max_len > attn::kQuad; }

// Lays the parts' segments out in the workspace; returns its bytes.
size_t lay_out(const nnrcu_kv_cache& c, const nnrcu_kv_attention_desc& d, Args* p, void* workspace) {
  if (!joined(d)) return 0;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  auto take = [&](size_t bytes) {
    uint8_t* const mine = at;
    at += (bytes + 255) / 256 * 256;
    return mine;
  };
  for (Args::Part* w : {&p->own, &p->prefix}) {
    if (!w->grid) continue;
    const size_t segments = (size_t)w->units * (w == &p->own ? d.batch : 1) + w->grid;
    w->ml = reinterpret_cast<float2*>(take(segments * w->rows * sizeof(float2)));
    w->o = reinterpret_cast<float*>(take(segments * w->rows * c.head_dim * sizeof(float)));
  }
  return at - static_cast<uint8_t*>(workspace);
}

// Joins the segments of each row: WARPS warps a row, which share its segments
// out, four channels a lane. A lane
// holds one segment's share in the result, so that the segments' means are
// loaded without waiting for one another. Starts while the attention ends, and then takes 3 to
// 4 us, which is latency: lengths, shares, means, one after the other. The order
// of the sums depends on the segments alone.
template <int WARPS>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Args p) {
  static_assert(WARPS == 1 || WARPS == 4, "a warp or the block");
  __shared__ float refs[4], totals[4];
  __shared__ float4 sums[WARPS > 1 ? 4 : 1][2][32];
  const int row = (int)(blockIdx.x * (4 / WARPS)) + (WARPS == 1 ? threadIdx.x >> 5 : 0);
  const int lane = threadIdx.x & 31, warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
  if (row >= p.batch * p.q_len * p.q_heads) return attn::pdl_wait();
  const int h = row % p.q_heads, i = row / p.q_heads % p.q_len, b = row / p.q_heads / p.q_len;
  const int head = h / p.share, in = i * p.share + h % p.share;
  // Where its own part's segments and the prefix's begin in ml and o, how many
  // there are and how far apart they are.
  const float2* ml[2] = {};
  const float* o[2] = {};
  int count[2] = {}, step[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const bool own = k == 0;
    if (!own && !p.prefix_len) continue;
    const Args::Part w = own ? p.own : p.prefix;
    const int r = own ? in : b * p.q_len * p.share + in;
    const int unit = head * w.blocks + r / w.rows;
    const attn::Shares s = attn::shares_of(p, own, lane, own ? b : 0);
    const int quads = attn::quads_of(p, own, own ? b : 0), begin = s.before + unit * quads;
    const int id = (own ? b * w.units : 0) + unit;
    const int most = (own ? p.batch * w.units : w.units) + w.grid - 1;  // passed only if lengths change
    const int first = min(most, id + begin / s.share), last = min(most, id + (begin + quads - 1) / s.share);
    count[k] = last - first + 1;
    step[k] = w.rows;
    const long long at = (long long)first * w.rows + r % w.rows;
    ml[k] = w.ml + at;
    o[k] = w.o + at * p.dim;
  }
  attn::pdl_wait();  // in every thread: what follows on the stream relies on it
  if (!p.prefix_len && count[0] == 1) return;  // written already
  // The sum of p over the warp's segments, and what it is relative to.
  float2 held[2];  // this lane's first segment of its own part and of the prefix
  float ref = -INFINITY, total = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int s = warp + lane * WARPS;
    held[k] = s < count[k] ? ml[k][s * step[k]] : make_float2(-INFINITY, 0.f);
  }
  auto add = [&](const float2 x) {
    const float next = fmaxf(ref, x.y == 0.f ? -INFINITY : x.x), base = next == -INFINITY ? 0.f : next;
    total = total * attn::exp2_fast(ref - base) + (x.y == 0.f ? 0.f : x.y * attn::exp2_fast(x.x - base));
    ref = next;
  };
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    add(held[k]);
    for (int s = warp + (lane + 32) * WARPS; s < count[k]; s += 32 * WARPS) add(ml[k][s * step[k]]);
  }
  const float mine = ref;
  for (int w = 16; w; w >>= 1) ref = fmaxf(ref, __shfl_xor_sync(~0u, ref, w));
  total *= attn::exp2_fast(mine - (ref == -INFINITY ? 0.f : ref));
  for (int w = 16; w; w >>= 1) total += __shfl_xor_sync(~0u, total, w);
  const float base = ref == -INFINITY ? 0.f : ref, part = total == 0.f ? 0.f : 1.f / total;
  float4 sum[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int s0 = warp; s0 < count[k]; s0 += 32 * WARPS) {  // segments s0, s0 + WARPS, ...
      float f = 0.f;
      if (s0 + lane * WARPS < count[k]) {
        const float2 x = s0 == warp ? held[k] : ml[k][(s0 + lane * WARPS) * step[k]];
        if (x.y != 0.f) f = x.y * attn::exp2_fast(x.x - base) * part;
      }
      const int n = min(32, (count[k] - s0 + WARPS - 1) / WARPS);
      const float* from = o[k] + (long long)s0 * step[k] * p.dim + lane * 4;
      const long long far = (long long)step[k] * p.dim * WARPS;
#pragma unroll 8
      for (int s = 0; s < n; ++s, from += far) {
        const float g = __shfl_sync(~0u, f, s);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (e * 128 + lane * 4 < p.dim) {
            const float4 x = *reinterpret_cast<const float4*>(from + e * 128);
            sum[e].x += x.x * g, sum[e].y += x.y * g, sum[e].z += x.z * g, sum[e].w += x.w * g;
          }
      }
    }
  if constexpr (WARPS > 1) {  // the warps' means, as the segments'
    if (lane == 0) refs[warp] = ref, totals[warp] = total;
    sums[warp][0][lane] = sum[0], sums[warp][1][lane] = sum[1];
    __syncthreads();
    if (warp) return;
    const float top = fmaxf(fmaxf(refs[0], refs[1]), fmaxf(refs[2], refs[3]));
    float f[4], all = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = totals[w] == 0.f ? 0.f : totals[w] * attn::exp2_fast(refs[w] - (top == -INFINITY ? 0.f : top));
      all += f[w];
    }
    const float of_all = all == 0.f ? 0.f : 1.f / all;
    sum[0] = sum[1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float g = f[w] * of_all;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 x = sums[w][e][lane];
        sum[e].x += x.x * g, sum[e].y += x.y * g, sum[e].z += x.z * g, sum[e].w += x.w * g;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (e * 128 + lane * 4 < p.dim) {
      const long long at = (long long)row * p.dim + e * 128 + lane * 4;
      attn::store_y(p, at, sum[e].x), attn::store_y(p, at + 1, sum[e].y);
      attn::store_y(p, at + 2, sum[e].z), attn::store_y(p, at + 3, sum[e].w);
    }
}

int launch_join(const Args& p, cudaStream_t st) {
  const long long rows = (long long)p.batch * p.q_len * p.q_heads;
  cudaLaunchConfig_t cfg{};
  // A block a row while the SMs take those at once and its warps have a segment
  // each: one sequence of 30000, 8 rows of 115 segments, the whole call 23 us and
  // 54 with a warp a row; 37 sequences of 2000, 2 segments a row, 40 and 37 us.
  const long long own = p.own.grid / ((long long)p.batch * p.own.units);
  const long long segments = own + (p.prefix_len ? p.prefix.grid / p.prefix.units : 0);
  const bool block = rows <= 8LL * num_sms() && segments >= 4;
  cfg.gridDim = dim3((unsigned)(block ? rows : (rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr{};  // its look at the lengths overlaps the end of the attention kernel
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  return cuda_check(cudaLaunchKernelEx(&cfg, block ? join_kernel<4> : join_kernel<1>, p), "attention join launch");
}

}  // namespace
}  // namespace nnrcu

using namespace nnrcu;

extern "C" {

int nnrcu_kv_attention_workspace(const nnrcu_kv_cache* cache, const nnrcu_kv_attention_desc* desc, size_t* bytes) {
  const int rc = check(cache, desc, false);
  if (rc != NNRCU_OK) return rc;
  if (!bytes) return set_error(NNRCU_ERR_INVALID, "bytes is NULL");
  *bytes = 0;
  if (desc->batch == 0) return NNRCU_OK;  // there are no rows to divide
  Args p{};
  divide(*cache, *desc, &p);
  *bytes = lay_out(*cache, *desc, &p, nullptr);
  return NNRCU_OK;
}

int nnrcu_kv_attention_run(const nnrcu_kv_cache* cache, const nnrcu_kv_attention_desc* desc, const void* q,
                           const int32_t* page_table, const int32_t* lens, const int32_t* prefix_table, void* y,
                           void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check(cache, desc, true);
  if (rc != NNRCU_OK || desc->batch == 0) return rc;
  const nnrcu_kv_attention_desc& d = *desc;
  if (!q || !lens || !y || (d.max_len && !page_table) || (d.prefix_len && !prefix_table))
    return set_error(NNRCU_ERR_INVALID, "NULL argument");
  Args p{};
  p.status = status_ptr();
  if (!p.status) return NNRCU_ERR_CUDA;
  divide(*cache, d, &p);
  for (const Args::Part* w : {&p.own, &p.prefix}) {
    const long long quads = (w == &p.own ? (long long)d.batch * (d.max_len / attn::kQuad + 2) : d.prefix_len / attn::kQuad + 2);
    if (w->units > 0 && quads >= INT_MAX / w->units - w->grid)
      return set_error(NNRCU_ERR_INVALID, "too many query rows over too long sequences for one call");
  }
  const size_t need = lay_out(*cache, d, &p, workspace);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error(NNRCU_ERR_INVALID, "workspace of %zu bytes, 16-byte aligned, required", need);
  p.q = q;
  p.y = y;
  p.q_batch = d.q_batch_stride;
  p.q_token = d.q_token_stride;
  p.q_head = d.q_head_stride;
  p.batch = d.batch;
  p.q_len = d.q_len;
  p.q_heads = d.q_heads;
  p.heads = cache->heads;
  p.share = d.q_heads / cache->heads;
  p.dim = cache->head_dim;
  p.k = static_cast<const uint8_t*>(cache->k);
  p.v = static_cast<const uint8_t*>(cache->v);
  p.k_scale = cache->k_scale;
  p.v_scale = cache->v_scale;
  p.pages = cache->pages;
  p.groups = cache->group ? cache->head_dim / cache->group : 1;
  p.page = divisor(cache->page_size);
  p.table = page_table;
  p.table_stride = d.table_stride;
  p.lens = lens;
  p.prefix_table = prefix_table;
  p.max_len = d.max_len;
  p.prefix_len = d.prefix_len;
  p.window = d.window;
  p.scale_log2 = std::fabs(d.scale) * 1.44269504088896340736f;
  p.q_sign = d.scale < 0 ? -1.f : 1.f;
  p.run = cache->page_size % 32 == 0 ? 32 : (cache->page_size % 16 == 0 ? 16 : 1);
  p.dtype = d.dtype;
  const int wide = 128 / cache->bits / 4;  // channels that a lane reads at once
  const size_t align = std::min<size_t>(16, wide * dtype_size(d.dtype));
  p.q_wide16 = reinterpret_cast<uintptr_t>(q) % 16 == 0 && d.q_batch_stride % 8 == 0 && d.q_token_stride % 8 == 0 &&
               d.q_head_stride % 8 == 0;
  p.q_wide = reinterpret_cast<uintptr_t>(q) % align == 0 && d.q_batch_stride % wide == 0 &&
             d.q_token_stride % wide == 0 && d.q_head_stride % wide == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool eight = cache->bits == 8;
  const auto few = d.dtype == NNRCU_DT_F32   ? (eight ? attn::launch_f32_b8 : attn::launch_f32_b4)
                   : d.dtype == NNRCU_DT_F16 ? (eight ? attn::launch_f16_b8 : attn::launch_f16_b4)
                                             : (eight ? attn::launch_bf16_b8 : attn::launch_bf16_b4);
  auto launch = [&](const Args& a, bool own, cudaStream_t s) {
    return (own ? a.own : a.prefix).rows == 128 ? attn::launch_many(a, cache->bits, own, s) : few(a, own, s);
  };
  if (p.prefix.grid) {
    const int rc2 = launch(p, false, st);
    if (rc2 != NNRCU_OK) return rc2;
  }
  const int rc3 = launch(p, true, st);
  return rc3 != NNRCU_OK || !joined(d) ? rc3 : launch_join(p, st);
}

}  // extern "C"
