// The bookkeeping and the writes of one step of a paged cache:
//   dkv_plan_paged_step  block tables, slots and positions from device-resident lengths
//   dkv_append_paged     RoPE of the new q and k rows, K and V stored in their slots
// They extend the layouts of the paged scatter / gather (src/deltakv/paged.py:8-70); the
// rotation is the reference's rotate-half RoPE (src/deltakv/rope.py:9-63).
#include "paged_rows.cuh"

namespace dkv {
namespace step {

// ---------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kMaxSeqs = 16384;  // cu_new and the block offsets of all sequences in shared memory

// What one sequence asks for, with every input forced into its documented range.
struct Want {
  int len, fresh, held, extra;
};
__device__ __forceinline__ Want want_of(const dkv_step_plan_args &a, int b, int32_t *status) {
  Want w;
  const int raw = a.lengths[b];
  w.len = max(raw, 0);
  const int n = a.new_lengths ? a.new_lengths[b] : w.len;
  w.fresh = min(max(n, 0), w.len);
  const int held = a.table_lens ? a.table_lens[b] : a.table_width;
  w.held = min(max(held, 0), a.table_width);
  const int need = static_cast<int>((static_cast<int64_t>(w.len) + a.block_size - 1) / a.block_size);
  if (raw < 0 || n != w.fresh || held != w.held) record_error(status, DKV_ERR_INVALID_ARGUMENT);
  if (need > a.table_width) record_error(status, DKV_ERR_BLOCK_TABLE_SHORT);
  w.extra = max(min(need, a.table_width) - w.held, 0);
  return w;
}

// largest b in [0, n) with cu[b] <= x (cu non-decreasing, cu[0] = 0 <= x): the sequence of
// item x, skipping empty ones
__device__ __forceinline__ int owner(const int *cu, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int saturate(int64_t v) { return v > INT32_MAX ? INT32_MAX : static_cast<int>(v); }

// Latency: a plan reads and writes a few hundred bytes to a few hundred KB (0.04 us at the HBM
// rate), so what counts is one launch and a short chain of dependent loads (lengths, table entry).
// Measured on a B200: 8 sequences of one new token 3.9 us, 512 of one 5.4 us, 96 prefill chunks of
// up to 2048 tokens 5.9 us of device time.
//
// Every CTA scans all sequences itself (their lengths are a few KB, resident in L2) and then
// fills its share of the rows and of the new table entries, so the whole plan is one launch;
// CTA 0 also writes the per-sequence outputs.  A new entry comes from the free list by index,
// never from the table another CTA may be writing.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(dkv_step_plan_args a) {
  extern __shared__ int sm[];
  begin_overlapped();
  const int n = a.n_seqs;
  int *cu_new = sm, *cu_ext = sm + n + 1;
  __shared__ int64_t warp_sum[3][kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool first = blockIdx.x == 0;
  int32_t *status = first ? a.status : nullptr;
  int64_t carry[3] = {0, 0, 0};
  for (int base = 0; base < n; base += kPlanThreads) {
    const int b = base + tid;
    Want w = {0, 0, 0, 0};
    if (b < n) w = want_of(a, b, status);
    const int64_t own[3] = {w.len, w.fresh, w.extra};
    int64_t inc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int64_t v = own[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      inc[k] = v;
      if (lane == 31) warp_sum[k][warp] = v;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int64_t before = carry[k], total = carry[k];
      for (int i = 0; i < kPlanThreads / 32; ++i) {
        const int64_t s = warp_sum[k][i];
        if (i < warp) before += s;
        total += s;
      }
      inc[k] += before;  // inclusive prefix over the whole batch
      carry[k] = total;
    }
    __syncthreads();
    if (b < n) {
      cu_new[b] = saturate(inc[1] - own[1]);
      cu_ext[b] = saturate(inc[2] - own[2]);
      if (first) {
        a.cu_seqlens[b + 1] = saturate(inc[0]);
        a.cu_new[b + 1] = inc[1] < a.n_rows ? static_cast<int>(inc[1]) : a.n_rows;
        const int64_t left = a.n_free - (inc[2] - own[2]);
        const int64_t got = left < 0 ? 0 : (left < w.extra ? left : w.extra);
        a.table_lens_out[b] = w.held + static_cast<int>(got);
      }
    }
  }
  if (tid == 0) {
    cu_new[n] = saturate(carry[1]);
    cu_ext[n] = saturate(carry[2]);
    if (first) {
      a.cu_seqlens[0] = 0;
      a.cu_new[0] = 0;
      a.blocks_used[0] = saturate(carry[2] < a.n_free ? carry[2] : a.n_free);
      if (carry[2] > a.n_free) record_error(status, DKV_ERR_NO_BLOCKS);
      if (carry[0] > INT32_MAX || carry[1] > a.n_rows) record_error(status, DKV_ERR_INVALID_ARGUMENT);
    }
  }
  __syncthreads();

  const int rows = cu_new[n], taken = cu_ext[n];
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid;
  for (int64_t r = at; r < a.n_rows; r += stride) {
    int pos = 0;
    int64_t slot = -1;
    if (r < rows) {
      const int b = owner(cu_new, n, static_cast<int>(r));
      const Want w = want_of(a, b, nullptr);
      pos = w.len - w.fresh + (static_cast<int>(r) - cu_new[b]);
      const int blk = pos / a.block_size;
      int id = -1;
      if (blk < w.held) {
        id = a.block_tables[static_cast<int64_t>(b) * a.table_stride + blk];
      } else if (blk < w.held + w.extra) {
        const int64_t f = static_cast<int64_t>(cu_ext[b]) + (blk - w.held);
        if (f < a.n_free) id = a.free_blocks[f];
      }
      if (id >= 0) slot = static_cast<int64_t>(id) * a.block_size + pos % a.block_size;
    }
    a.positions[r] = pos;
    a.slots[r] = slot;
  }
  const int64_t entries = taken < a.n_free ? taken : a.n_free;
  for (int64_t e = at; e < entries; e += stride) {
    const int b = owner(cu_ext, n, static_cast<int>(e));
    const Want w = want_of(a, b, nullptr);
    a.block_tables[static_cast<int64_t>(b) * a.table_stride + w.held + (e - cu_ext[b])] = a.free_blocks[e];
  }
}

// ---------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------
// A thread has VEC columns i and their partners i + half of up to kHeads heads of a row, so that
// the row's slot, position and cos / sin are read once for all of them and 2 kHeads 16-byte loads
// are in flight; the heads of a thread are `groups` apart, so that neighbouring threads read
// neighbouring heads.  Bound by memory: every q, k and v element is read once and written once.  Measured
// on a B200: 16384 rows of 32 + 8 + 8 heads x 128, bf16 68-70 us = 5.9-6.0 TB/s, 0.90-0.92 of the measured HBM rate
// (an element pair a thread: 312 us; two heads a thread 75 us; a thread's heads adjacent 71 us); 64 rows 3.0 us.
// fp32, the same rows: 120 us, at the floor of 123.  Rows whose halves are not 16-byte pieces go an element pair a
// thread, with four heads' loads in flight still: head_dim 72 / 100, bf16, 120 / 166 us (floors 35 / 48), fp32 100 167 (96).
template <int SDT, int PDT, int VEC, bool kForms>
__global__ void __launch_bounds__(kAppThreads) append_kernel(const __grid_constant__ Append a) {
  begin_overlapped();
  append_rows<SDT, PDT, VEC, kForms>(a, static_cast<int64_t>(blockIdx.x) * kAppThreads + threadIdx.x);
}

bool float_dtype(int dt) { return dt == DKV_F32 || dt == DKV_F16 || dt == DKV_BF16; }

}  // namespace step
}  // namespace dkv

using namespace dkv;

extern "C" int dkv_plan_paged_step(const dkv_step_plan_args *args, dkv_stream_t stream) {
  if (args == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  const dkv_step_plan_args &a = *args;
  if (a.n_seqs < 0 || a.n_rows < 0 || a.block_size <= 0 || a.table_width < 0 || a.n_free < 0)
    return DKV_ERR_INVALID_ARGUMENT;
  if (a.n_seqs > step::kMaxSeqs) return DKV_ERR_UNSUPPORTED;
  if (a.cu_seqlens == nullptr || a.cu_new == nullptr || a.blocks_used == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (a.n_seqs > 0 && (a.lengths == nullptr || a.table_lens_out == nullptr)) return DKV_ERR_INVALID_ARGUMENT;
  if (a.n_seqs > 0 && a.table_width > 0 && a.block_tables == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (a.n_rows > 0 && (a.positions == nullptr || a.slots == nullptr)) return DKV_ERR_INVALID_ARGUMENT;
  if (a.n_free > 0 && a.free_blocks == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (a.n_free > INT32_MAX) return DKV_ERR_UNSUPPORTED;
  if (a.n_seqs > 0 && (a.table_lens_out == a.table_lens || a.table_lens_out == a.lengths))
    return DKV_ERR_INVALID_ARGUMENT;
  const int smem = 2 * (a.n_seqs + 1) * static_cast<int>(sizeof(int));
  // A launch without the opt-in has 48 KB, the kernel's own static arrays included (384 bytes now): opted in well
  // before that.  Always to the same limit: two threads' calls cannot lower each other's.
  if (smem > 40 * 1024)
    DKV_CUDA_CHECK(cudaFuncSetAttribute(step::plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        2 * (step::kMaxSeqs + 1) * static_cast<int>(sizeof(int))));
  const int64_t want = (static_cast<int64_t>(a.n_rows) + 2 * step::kPlanThreads - 1) / (2 * step::kPlanThreads);
  int grid = 1;
  if (want > 1) {
    const int rc = sm_count(&grid);
    if (rc != DKV_OK) return rc;
    if (want < grid) grid = static_cast<int>(want);
  }
  DKV_CUDA_CHECK(launch_overlapped(step::plan_kernel, dim3(grid), step::kPlanThreads, smem,
                                   reinterpret_cast<cudaStream_t>(stream), a));
  return DKV_OK;
}

extern "C" int dkv_append_paged(const dkv_append_args *args, dkv_stream_t stream) {
  return dkv_append_paged_rotary(args, nullptr, stream);
}

extern "C" int dkv_append_paged_rotary(const dkv_append_args *args, const dkv_rotary *rotary, dkv_stream_t stream) {
  if (args == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  const dkv_append_args &g = *args;
  const dkv_paged_cache &kp = g.k_pages, &vp = g.v_pages;
  if (!step::float_dtype(kp.dtype) || !step::float_dtype(g.in_dtype)) return DKV_ERR_UNSUPPORTED;
  if (g.in_dtype != kp.dtype && g.in_dtype != DKV_F32) return DKV_ERR_UNSUPPORTED;
  if (kp.dtype != vp.dtype || kp.block_size != vp.block_size || kp.n_heads != vp.n_heads || kp.head_dim != vp.head_dim ||
      kp.block_size <= 0 || kp.n_heads <= 0 || kp.head_dim <= 0 || kp.num_blocks < 0 || vp.num_blocks < 0)
    return DKV_ERR_LAYOUT;
  if (g.n_rows < 0 || (g.q != nullptr && g.n_q_heads <= 0)) return DKV_ERR_INVALID_ARGUMENT;
  if ((g.rope_cos == nullptr) != (g.rope_sin == nullptr)) return DKV_ERR_INVALID_ARGUMENT;
  step::Rotary rot;
  const int form = step::rotary_of(g.rope_cos != nullptr, rotary, kp.head_dim, &rot);
  if (form < 0) return DKV_ERR_UNSUPPORTED;
  if (g.n_rows == 0) return DKV_OK;
  if (g.k == nullptr || g.v == nullptr || g.slots == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (g.rope_cos != nullptr && g.positions == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (g.q != nullptr && g.q_out == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if ((kp.base == nullptr && kp.num_blocks > 0) || (vp.base == nullptr && vp.num_blocks > 0))
    return DKV_ERR_INVALID_ARGUMENT;
  step::Append a;
  step::describe(g, rot, &a);
  a.heads[1] = a.heads[2] = kp.n_heads;
  // 16-byte accesses where every half row of a head starts on 16 bytes 
  const int64_t ssz = g.in_dtype == DKV_F32 ? 4 : 2, psz = kp.dtype == DKV_F32 ? 4 : 2;
  const int vec = static_cast<int>(16 / psz);
  int64_t in_bits = 0, page_bits = 0;
  for (int w = g.q != nullptr ? 0 : 1; w < 3; ++w) {
    in_bits |= reinterpret_cast<intptr_t>(a.src[w]) | a.src_row[w] * ssz | a.src_head[w] * ssz;
    if (w == 0)
      in_bits |= reinterpret_cast<intptr_t>(a.dst[0]) | a.dst_row[0] * ssz | a.dst_head[0] * ssz;
    else
      page_bits |= reinterpret_cast<intptr_t>(a.dst[w]) | a.dst_row[w] * psz | a.dst_head[w] * psz | a.dst_block[w] * psz;
  }
  in_bits |= reinterpret_cast<intptr_t>(a.cos_t) | reinterpret_cast<intptr_t>(a.sin_t);
  const bool wide = step::whole_pieces(rot, kp.head_dim, vec) && (in_bits | page_bits) % 16 == 0;
  const int all = a.heads[0] + a.heads[1] + a.heads[2];
  const int64_t total = a.n_rows * ((all + step::kHeads - 1) / step::kHeads) *
                        (form ? step::pieces_of(rot, kp.head_dim, wide ? vec : 1) : a.half / (wide ? vec : 1));
  a.wide = total > UINT32_MAX;
  const int64_t ctas = (total + step::kAppThreads - 1) / step::kAppThreads;
  if (ctas > INT32_MAX) return DKV_ERR_UNSUPPORTED;
  const unsigned grid = static_cast<unsigned>(ctas);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define DKV_APPEND_CASE(S, P)                                                                              \
  if (g.in_dtype == S && kp.dtype == P) {                                                                  \
    constexpr int kVec = P == DKV_F32 ? 4 : 8;                                                             \
    const auto kernel = form ? (wide ? step::append_kernel<S, P, kVec, true> : step::append_kernel<S, P, 1, true>)     \
                             : (wide ? step::append_kernel<S, P, kVec, false> : step::append_kernel<S, P, 1, false>);  \
    DKV_CUDA_CHECK(launch_overlapped(kernel, dim3(grid), step::kAppThreads, 0, st, a));                    \
    return DKV_OK;                                                                                         \
  }
  DKV_APPEND_CASE(DKV_BF16, DKV_BF16)
  DKV_APPEND_CASE(DKV_F16, DKV_F16)
  DKV_APPEND_CASE(DKV_F32, DKV_F32)
  DKV_APPEND_CASE(DKV_F32, DKV_BF16)
  DKV_APPEND_CASE(DKV_F32, DKV_F16)
#undef DKV_APPEND_CASE
  return DKV_ERR_UNSUPPORTED;
}
