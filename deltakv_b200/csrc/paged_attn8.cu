// Attention of one new token per sequence over 8-bit pages: the entries, and the kernels for e4m3.
#include "paged_attn8.cuh"

namespace dkv {
namespace pattn {

int check8(const dkv_paged_decode_args *a, int q_dtype) {
  if (a == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if ((a->k_pages.dtype != DKV_E4M3 && a->k_pages.dtype != DKV_I8) || !float_dtype(q_dtype)) return DKV_ERR_UNSUPPORTED;
  return check_args(*a);
}

int shape8(const dkv_paged_decode_args *a, int q_dtype, Shape *s) {
  const int hd = a->k_pages.head_dim;
  s->hd_pad = hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
  const bool f32 = q_dtype == DKV_F32;
  s->g = heads8(f32, s->hd_pad, a->n_q_heads / a->k_pages.n_heads);
  return cut_up(*a, variant8(f32, s->hd_pad, s->g), kSeqCost8, kLeastLocal8, s);
}

}  // namespace pattn
}  // namespace dkv

using namespace dkv;

extern "C" int dkv_paged_decode_quant_workspace_bytes(const dkv_paged_decode_args *args, int32_t q_dtype, int64_t *bytes) {
  if (bytes == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  const int rc = pattn::check8(args, q_dtype);
  if (rc != DKV_OK) return rc;
  pattn::Shape s;
  const int rs = pattn::shape8(args, q_dtype, &s);
  if (rs != DKV_OK) return rs;
  *bytes = s.bytes;
  return DKV_OK;
}

extern "C" int dkv_paged_decode_attention_quant(const dkv_paged_decode_args *args, int32_t q_dtype,
                                                const dkv_page_scales *k_scales, const dkv_page_scales *v_scales,
                                                dkv_stream_t stream) {
  const int rc = pattn::check8(args, q_dtype);
  if (rc != DKV_OK) return rc;
  const dkv_paged_decode_args &a = *args;
  const dkv_paged_cache &k = a.k_pages, &v = a.v_pages;
  if (k_scales == nullptr || v_scales == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if (a.seqs.n_seqs == 0) return DKV_OK;
  if (a.q == nullptr || a.out == nullptr || a.seqs.cu_seqlens == nullptr) return DKV_ERR_INVALID_ARGUMENT;
  if ((k.num_blocks > 0 && (k.base == nullptr || k_scales->base == nullptr)) ||
      (v.num_blocks > 0 && (v.base == nullptr || v_scales->base == nullptr)))
    return DKV_ERR_INVALID_ARGUMENT;
  pattn::Shape s;
  const int rs = pattn::shape8(args, q_dtype, &s);
  if (rs != DKV_OK) return rs;
  if (s.bytes > 0 && (a.workspace == nullptr || a.workspace_bytes < s.bytes)) return DKV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a.workspace) % 16) return DKV_ERR_ALIGNMENT;
  pattn::Params p;
  pattn::fill_params(a, s, 1, q_dtype == DKV_F32 ? 4 : 2, &p);
  p.k_scale = k_scales->base, p.ks_block = k_scales->stride_block, p.ks_head = k_scales->stride_head;
  // a tile's halves are copied as pages where each lies in one block
  if (p.copy == pattn::kRows && k.block_size % pattn::kTile == 0) p.copy = pattn::kPages;
  // places in the pages are 32 bits of 16 bytes, strides of rows and of scales 32 bits
  auto reach = [](int64_t blocks, int64_t block, int64_t slots, int64_t slot) {
    return block >= 0 && slot >= 0 && slot <= INT32_MAX &&
           (blocks == 0 || (blocks - 1) * block + (slots - 1) * slot < (int64_t{1} << 36));
  };
  if (p.copy != pattn::kPlain && (!reach(p.num_blocks, p.k_block, k.block_size, p.k_slot) ||
                                  !reach(p.num_blocks, p.v_block, k.block_size, p.v_slot)))
    p.copy = pattn::kPlain;
  p.v_scale = v_scales->base, p.vs_block = v_scales->stride_block, p.vs_head = v_scales->stride_head;
  if (p.ks_block < 0 || p.vs_block < 0 || p.ks_block > UINT32_MAX || p.vs_block > UINT32_MAX) return DKV_ERR_UNSUPPORTED;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return k.dtype == DKV_I8 ? pattn::launch8_int8(q_dtype, p, s, st) : pattn::launch8<DKV_E4M3>(q_dtype, p, s, st);
}
