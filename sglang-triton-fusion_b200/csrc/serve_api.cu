// C ABI of the serving operators (declared in include/fp8gq.h): argument
// checks, kernel selection and launch.
#include <cuda_runtime.h>

#include <cmath>

#include "../../include/fp8gq.h"
#include "fp8gq_device.cuh"
#include "host_common.h"
#include "paged_decode.cuh"
#include "prompt_attention.cuh"
#include "rope_append.cuh"
#include "token_logprobs.cuh"

namespace fp8gq {

int serve_error_word(unsigned int* code, int clear) {
  if (cudaMemcpyFromSymbol(code, g_device_error, sizeof(*code)) != cudaSuccess) return FP8GQ_ERR_LAUNCH;
  if (clear && *code) {
    const unsigned int zero = 0;
    if (cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero)) != cudaSuccess) return FP8GQ_ERR_LAUNCH;
  }
  return FP8GQ_OK;
}

int serve_set_wait_limit(unsigned long long limit_ns) {
  return cudaMemcpyToSymbol(g_wait_limit_ns, &limit_ns, sizeof(limit_ns)) == cudaSuccess ? FP8GQ_OK : FP8GQ_ERR_LAUNCH;
}

}  // namespace fp8gq

using namespace fp8gq;

namespace {

int check_heads(int Hq, int Hkv, int D) {
  if (Hq < 1 || Hkv < 1 || Hq % Hkv) return FP8GQ_ERR_SHAPE;
  if (D != 64 && D != 128) return FP8GQ_ERR_UNSUPPORTED;
  return FP8GQ_OK;
}

// log2 of a power of two, -1 of any other number.
int log2_of(int x) {
  for (int i = 0; i < 31; ++i)
    if (x == 1 << i) return i;
  return -1;
}

// A cache's checks; strides are multiples of 16 bytes and (for a cache with
// several pages, slots or heads) positive.
int to_cache_view(const fp8gq_paged_cache* c, int Hkv, int D, CacheView* v) {
  if (!c || !c->k || !c->v) return FP8GQ_ERR_NULL_POINTER;
  if (c->num_pages < 1 || c->page_size < 1 || c->num_pages > INT32_MAX) return FP8GQ_ERR_SHAPE;
  if (c->dtype != FP8GQ_DTYPE_BF16 && c->dtype != FP8GQ_DTYPE_E4M3) return FP8GQ_ERR_UNSUPPORTED;
  const int64_t st[6] = {c->k_page_stride, c->k_slot_stride, c->k_head_stride,
                         c->v_page_stride, c->v_slot_stride, c->v_head_stride};
  const int64_t n[3] = {c->num_pages, c->page_size, Hkv};
  const int unit = c->dtype == FP8GQ_DTYPE_BF16 ? 8 : 16;
  for (int i = 0; i < 6; ++i) {
    if (n[i % 3] > 1 && st[i] < D) return FP8GQ_ERR_STRIDE;
    if (st[i] % unit) return FP8GQ_ERR_ALIGNMENT;
  }
  if (!aligned16(c->k) || !aligned16(c->v)) return FP8GQ_ERR_ALIGNMENT;
  if (c->dtype == FP8GQ_DTYPE_E4M3 && !(c->k_scale > 0.0f && c->v_scale > 0.0f)) return FP8GQ_ERR_UNSUPPORTED;
  v->k = c->k;
  v->v = c->v;
  v->k_page = st[0];
  v->k_slot = st[1];
  v->k_head = st[2];
  v->v_page = st[3];
  v->v_slot = st[4];
  v->v_head = st[5];
  v->num_pages = c->num_pages;
  v->page_size = c->page_size;
  v->k_scale = c->k_scale;
  v->v_scale = c->v_scale;
  return FP8GQ_OK;
}

// q, k, v or out [tokens, heads, D] bf16: strides of at least a head, 16-byte
// rows.
int check_rows(const void* p, int64_t token, int64_t head, int tokens, int heads, int D) {
  if (!p) return FP8GQ_ERR_NULL_POINTER;
  if ((tokens > 1 && token < D) || (heads > 1 && head < D)) return FP8GQ_ERR_STRIDE;
  if (!aligned16(p) || token % 8 || head % 8) return FP8GQ_ERR_ALIGNMENT;
  return FP8GQ_OK;
}

// ----------------------------------------------------------------- prompt --
constexpr int kPromptSplitSeqs = 32;         // (a lane of the item warp has a sequence)
constexpr int kPromptSplitGain = 1000;       // keys whose tiles take as long as pieces and their join cost

// Whole items off a counter, or equal ranges of key tiles whose pieces are
// joined: by the tiles that the busiest CTA computes when items are whole,
// against the mean, for sequences of the mean lengths.  Measured, whole items and
// ranges: 64 tokens behind 6000 (16 heads, 1 kv head) 93 and 25 us, 4 x 16 behind
// 4000 (32, 8, D = 64) 54 and 25, 4 x 1024 ragged behind 5003 (16, 4, D = 64) 90
// and 61, 2 x 700 behind 1000 (8, 8) 33 and 24; 1 x 2048 (32, 8) 42 and 54, 8 x 1
// behind 700 15.5 and 18.5, 4 x 500 (40, 8) 30 and 37.
bool prompt_split(int B, int Tq, int Tk, int Hkv, int span, int keys, bool causal, int sms) {
  if (B > kPromptSplitSeqs) return false;
  const int lq = (Tq + B - 1) / B;
  const double most = static_cast<double>(Tk) / B / keys, own = std::min(causal ? static_cast<double>(lq) / keys : 0.0, most);
  const double least = most - own;             // tiles of a sequence's last and of its first item
  const double share = static_cast<double>(B) * ((lq + span - 1) / span) * Hkv / sms;
  const double mean = share * (most - own / 2);
  const double busiest = std::max(most, mean + (std::ceil(share) - share) * least);
  return (busiest - mean) * keys >= kPromptSplitGain;
}

// Counters, and where a split call leaves its pieces.
static_assert(FP8GQ_PROMPT_COUNTER_BYTES == kDecCounterBytes, "");
size_t prompt_split_bytes(int D, int sm_count) {
  return kDecCounterBytes + sm_count * (sizeof(PrSplit) + 2 * sizeof(float) * (D == 128 ? PrCfg<128>::kPart : PrCfg<64>::kPart));
}
int prompt_keys(int D) { return D == 128 ? PrCfg<128>::kKeys : PrCfg<64>::kKeys; }

// [tokens, heads, D] bf16 as boxes of 64 values x `box_heads` heads x
// `box_tokens` tokens, 128-byte swizzle.  A stride that no coordinate above 0
// uses is replaced by a valid one.
bool make_heads_tmap(CUtensorMap* map, const void* p, int tokens, int heads, int D, int64_t token, int64_t head,
                     int box_heads, int box_tokens) {
  auto enc = tensor_map_encoder();
  if (!enc) return false;
  if (heads == 1) head = D;
  if (tokens == 1) token = static_cast<int64_t>(heads) * head;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head) * 2, static_cast<cuuint64_t>(token) * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ---------------------------------------------------------- log probabilities --
// CTAs per row: enough for two CTAs per SM, each with 4096 values at least, 16
// at most.  Measured at 151936 values: 37 fp32 rows 13.1 us with 8 (20.5 us with
// 16, four CTAs per SM: the joins outweigh the shorter stream), 1 bf16 row
// 8.0 us with 16 (8.3 with 8, 9.3 with 4).
int logprobs_cluster(int T, int V, int sm_count) {
  int c = 1;
  while (c < 16 && static_cast<int64_t>(T) * c < 2 * sm_count && V / (2 * c) >= 4096) c *= 2;
  return c;
}

// ----------------------------------------------------------------- decode --

size_t decode_workspace_bytes(int group, int D, int sm_count) {
  return kDecCounterBytes +
         static_cast<size_t>(kDecCtas) * sm_count * 2 * dec_slot_floats(D, group > 8 ? 2 : 1) * sizeof(float);
}

template <int D, bool kFp8, int kNT>
cudaError_t launch_decode(const DecodeParams& p, const DeviceInfo& di, fp8gq_stream_t stream) {
  using Cfg = DecCfg<D, kFp8, kNT>;
  auto fn = paged_decode_kernel<D, kFp8, kNT>;
  cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(fn), static_cast<int>(Cfg::kSmem));
  if (e != cudaSuccess) return e;
  // no more CTAs than tiles, were every sequence as long as its page table
  const int64_t tiles = (static_cast<int64_t>(p.max_pages) * p.cache.page_size + Cfg::kTile - 1) / Cfg::kTile;
  int64_t grid = kDecCtas * di.sm_count;
  if (grid * 4 > kDecCounterBytes) grid = kDecCounterBytes / 4;      // a counter per CTA
  const int64_t most = tiles > grid ? grid : tiles * p.Hkv * p.blocks * p.B;
  if (most < grid) grid = most < 1 ? 1 : most;
  return launch_with_pdl(fn, dim3(static_cast<unsigned>(grid)), dim3(kDecThreads), Cfg::kSmem,
                         static_cast<cudaStream_t>(stream), p);
}

}  // namespace

extern "C" {

int fp8gq_qk_norm_rope_append(const void* qkv, int64_t ldqkv, const int64_t* positions, const int64_t* slots,
                              const float* cos_sin, int64_t max_position, const void* q_weight, const void* k_weight,
                              float eps, void* q_out, int64_t ldq, void* k_out, int64_t ldk,
                              const fp8gq_paged_cache* cache, int T, int Hq, int Hkv, int D, fp8gq_stream_t stream) {
  if (T < 0) return FP8GQ_ERR_SHAPE;
  int st = check_heads(Hq, Hkv, D);
  if (st != FP8GQ_OK) return st;
  AppendParams p{};
  st = to_cache_view(cache, Hkv, D, &p.cache);
  if (st != FP8GQ_OK) return st;
  if (T == 0) return FP8GQ_OK;
  if (!qkv || !positions || !slots || !cos_sin || !q_out) return FP8GQ_ERR_NULL_POINTER;
  const int64_t heads = static_cast<int64_t>(Hq) + 2 * static_cast<int64_t>(Hkv);
  if (max_position < 1 || heads > INT32_MAX / D) return FP8GQ_ERR_SHAPE;
  if (T > 1 && (ldqkv < heads * D || ldq < static_cast<int64_t>(Hq) * D ||
                (k_out && ldk < static_cast<int64_t>(Hkv) * D)))
    return FP8GQ_ERR_STRIDE;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(cos_sin) || !aligned16(q_weight) ||
      !aligned16(k_weight) || ldqkv % 8 || ldq % 8 || (k_out && ldk % 8))
    return FP8GQ_ERR_ALIGNMENT;
  DeviceInfo di;
  st = device_info(&di, nullptr);
  if (st != FP8GQ_OK) return st;
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.ldqkv = ldqkv;
  p.positions = positions;
  p.slots = slots;
  p.cos_sin = cos_sin;
  p.max_position = max_position;
  p.qw = static_cast<const __nv_bfloat16*>(q_weight);
  p.kw = static_cast<const __nv_bfloat16*>(k_weight);
  p.eps = eps;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.ldq = ldq;
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.ldk = ldk;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.page_shift = log2_of(cache->page_size);
  const int64_t units = static_cast<int64_t>(T) * heads, per_block = kAppendThreads / (D / 16);
  const int64_t blocks = (units + per_block - 1) / per_block;
  if (units > INT32_MAX) return FP8GQ_ERR_UNSUPPORTED;
  p.units = static_cast<uint32_t>(units);
  const bool fp8 = cache->dtype == FP8GQ_DTYPE_E4M3;
  auto fn = D == 128 ? (fp8 ? rope_append_kernel<128, true> : rope_append_kernel<128, false>)
                     : (fp8 ? rope_append_kernel<64, true> : rope_append_kernel<64, false>);
  const cudaError_t e = launch_with_pdl(fn, dim3(static_cast<unsigned>(blocks)), dim3(kAppendThreads), 0,
                                        static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? launch_status() : cuda_fail(e, "fp8gq_qk_norm_rope_append");
}

size_t fp8gq_paged_decode_workspace_bytes(int Hq, int Hkv, int D) {
  DeviceInfo di;
  if (check_heads(Hq, Hkv, D) != FP8GQ_OK || device_info(&di, nullptr) != FP8GQ_OK) return 0;
  return decode_workspace_bytes(Hq / Hkv, D, di.sm_count);
}

int fp8gq_paged_decode_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                 const fp8gq_paged_cache* cache, const int32_t* page_table, int64_t ld_table,
                                 int max_pages, const int32_t* lens, void* out, int64_t o_token_stride,
                                 int64_t o_head_stride, float* lse, int B, int Hq, int Hkv, int D, float scale,
                                 void* workspace, size_t workspace_bytes, fp8gq_stream_t stream) {
  if (B < 0 || max_pages < 0) return FP8GQ_ERR_SHAPE;
  int st = check_heads(Hq, Hkv, D);
  if (st != FP8GQ_OK) return st;
  DecodeParams p{};
  st = to_cache_view(cache, Hkv, D, &p.cache);
  if (st != FP8GQ_OK) return st;
  if (B == 0) return FP8GQ_OK;
  if (!lens || (!page_table && max_pages > 0)) return FP8GQ_ERR_NULL_POINTER;
  st = check_rows(q, q_token_stride, q_head_stride, B, Hq, D);
  if (st != FP8GQ_OK) return st;
  st = check_rows(out, o_token_stride, o_head_stride, B, Hq, D);
  if (st != FP8GQ_OK) return st;
  if (B > 1 && ld_table < max_pages) return FP8GQ_ERR_STRIDE;
  DeviceInfo di;
  st = device_info(&di, nullptr);
  if (st != FP8GQ_OK) return st;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.table = page_table;
  p.ld_table = ld_table;
  p.max_pages = max_pages;
  p.lens = lens;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_token = o_token_stride;
  p.o_head = o_head_stride;
  p.lse = lse;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  const bool fp8 = cache->dtype == FP8GQ_DTYPE_E4M3;
  // rows are addressed by 32-bit offsets in units of 16 bytes
  for (int kv = 0; kv < 2; ++kv) {
    const int64_t span = (cache->num_pages - 1) * (kv ? cache->v_page_stride : cache->k_page_stride) +
                         (cache->page_size - 1) * (kv ? cache->v_slot_stride : cache->k_slot_stride) +
                         (Hkv - 1) * (kv ? cache->v_head_stride : cache->k_head_stride) + D;
    if (span / (fp8 ? 16 : 8) > UINT32_MAX) return FP8GQ_ERR_UNSUPPORTED;
  }
  p.page_shift = log2_of(cache->page_size);
  p.group = Hq / Hkv;
  const int nt = p.group > 8 ? 2 : 1;
  p.blocks = (p.group + 8 * nt - 1) / (8 * nt);
  p.scale_log2 = scale * 1.4426950408889634f * (fp8 ? cache->k_scale : 1.0f);
  p.out_scale = fp8 ? cache->v_scale : 1.0f;
  if (!workspace || workspace_bytes < decode_workspace_bytes(p.group, D, di.sm_count)) return FP8GQ_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FP8GQ_ERR_ALIGNMENT;
  p.counters = static_cast<int*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + kDecCounterBytes);
  cudaError_t e;
  if (D == 128)
    e = fp8 ? (nt == 2 ? launch_decode<128, true, 2>(p, di, stream) : launch_decode<128, true, 1>(p, di, stream))
            : (nt == 2 ? launch_decode<128, false, 2>(p, di, stream) : launch_decode<128, false, 1>(p, di, stream));
  else
    e = fp8 ? (nt == 2 ? launch_decode<64, true, 2>(p, di, stream) : launch_decode<64, true, 1>(p, di, stream))
            : (nt == 2 ? launch_decode<64, false, 2>(p, di, stream) : launch_decode<64, false, 1>(p, di, stream));
  return e == cudaSuccess ? launch_status() : cuda_fail(e, "fp8gq_paged_decode_attention");
}

size_t fp8gq_prompt_workspace_bytes(void) {
  DeviceInfo di;
  if (device_info(&di, nullptr) != FP8GQ_OK) return 0;
  return prompt_split_bytes(128, di.sm_count);
}

size_t fp8gq_prompt_split_bytes(int B, int Tq, int Tk, int Hq, int Hkv, int D, int causal) {
  DeviceInfo di;
  if (B < 1 || Tq < 1 || Tk < 0 || check_heads(Hq, Hkv, D) != FP8GQ_OK || Hq / Hkv > 128 ||
      device_info(&di, nullptr) != FP8GQ_OK ||
      !prompt_split(B, Tq, Tk, Hkv, 2 * (128 / (Hq / Hkv)), prompt_keys(D), causal != 0, di.sm_count))
    return 0;
  return prompt_split_bytes(D, di.sm_count);
}

int fp8gq_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                           int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                           int64_t v_head_stride, void* out, int64_t o_token_stride, int64_t o_head_stride, float* lse,
                           const int32_t* cu_q, const int32_t* cu_k, int B, int Tq, int Tk, int Hq, int Hkv, int D,
                           float scale, int causal, void* workspace, size_t workspace_bytes, fp8gq_stream_t stream) {
  if (B < 0 || Tq < 0 || Tk < 0) return FP8GQ_ERR_SHAPE;
  int st = check_heads(Hq, Hkv, D);
  if (st != FP8GQ_OK) return st;
  if (B == 0 || Tq == 0) return FP8GQ_OK;
  if (!cu_q || !cu_k) return FP8GQ_ERR_NULL_POINTER;
  st = check_rows(q, q_token_stride, q_head_stride, Tq, Hq, D);
  if (st == FP8GQ_OK) st = check_rows(out, o_token_stride, o_head_stride, Tq, Hq, D);
  if (st == FP8GQ_OK && Tk > 0) st = check_rows(k, k_token_stride, k_head_stride, Tk, Hkv, D);
  if (st == FP8GQ_OK && Tk > 0) st = check_rows(v, v_token_stride, v_head_stride, Tk, Hkv, D);
  if (st != FP8GQ_OK) return st;
  DeviceInfo di;
  st = device_info(&di, nullptr);
  if (st != FP8GQ_OK) return st;
  if (!std::isfinite(scale)) return FP8GQ_ERR_UNSUPPORTED;
  const int group = Hq / Hkv;
  if (group > 128) return FP8GQ_ERR_UNSUPPORTED;
  PromptParams p{};
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.o_token = o_token_stride;
  p.o_head = o_head_stride;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.B = B;
  p.Tq = Tq;
  p.Tk = Tk;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.group = group;
  p.rows = 128 / group;
  p.group_inv = (65536 + group - 1) / group;
  // a scale of 0 as one too small to tell scores apart, so that -inf stays -inf
  p.scale_log2 = scale == 0.0f ? 1e-30f : std::fabs(scale) * 1.4426950408889634f;
  p.negate = scale < 0.0f;
  p.causal = causal ? 1 : 0;
  const int keys = prompt_keys(D);
  CUtensorMap tq, tk, tv;
  if (!make_heads_tmap(&tq, q, Tq, Hq, D, q_token_stride, q_head_stride, group, p.rows) ||
      !make_heads_tmap(&tk, Tk ? k : q, Tk ? Tk : 1, Hkv, D, Tk ? k_token_stride : 0, Tk ? k_head_stride : D, 1, keys) ||
      !make_heads_tmap(&tv, Tk ? v : q, Tk ? Tk : 1, Hkv, D, Tk ? v_token_stride : 0, Tk ? v_head_stride : D, 1, keys))
    return FP8GQ_ERR_LAUNCH;
  // a row block more than the tokens fill for each sequence's odd end
  const int64_t items = (static_cast<int64_t>(Tq) / (2 * p.rows) + B) * Hkv;
  if (items > INT32_MAX / 2) return FP8GQ_ERR_UNSUPPORTED;
  p.split = prompt_split(B, Tq, Tk, Hkv, 2 * p.rows, keys, causal != 0, di.sm_count);
  const size_t need = p.split ? prompt_split_bytes(D, di.sm_count) : FP8GQ_PROMPT_COUNTER_BYTES;
  if (!workspace || workspace_bytes < need) return FP8GQ_ERR_WORKSPACE;
  if (!aligned16(workspace)) return FP8GQ_ERR_ALIGNMENT;
  p.counters = static_cast<int*>(workspace);
  p.splits = reinterpret_cast<PrSplit*>(static_cast<char*>(workspace) + kDecCounterBytes);
  p.parts = reinterpret_cast<float*>(p.splits + di.sm_count);
  const unsigned blocks = static_cast<unsigned>(p.split || items > di.sm_count ? di.sm_count : items);
  auto fn = D == 128 ? prompt_attention_kernel<128> : prompt_attention_kernel<64>;
  const size_t smem = D == 128 ? PrCfg<128>::kSmem : PrCfg<64>::kSmem;
  cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(fn), static_cast<int>(smem));
  if (e == cudaSuccess)
    e = launch_with_pdl(fn, dim3(blocks), dim3(kPrThreads), smem, static_cast<cudaStream_t>(stream), tq, tk, tv, p);
  if (e == cudaSuccess && p.split)
    e = launch_with_pdl(D == 128 ? prompt_join_kernel<128> : prompt_join_kernel<64>, dim3(blocks, D / 16), dim3(256), 0,
                        static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? launch_status() : cuda_fail(e, "fp8gq_prompt_attention");
}

int fp8gq_token_logprobs(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int T, int V,
                         float* logprobs, float* entropy, int64_t* top_ids, float* top_logprobs, int top_k,
                         fp8gq_stream_t stream) {
  if (T < 0 || V < 1 || top_k < 0 || top_k > V) return FP8GQ_ERR_SHAPE;
  if (top_k > kMaxTop || (dtype != FP8GQ_DTYPE_BF16 && dtype != FP8GQ_DTYPE_F32)) return FP8GQ_ERR_UNSUPPORTED;
  if (T == 0) return FP8GQ_OK;
  if (T > INT32_MAX / 16 || V > INT32_MAX - kLpThreads) return FP8GQ_ERR_UNSUPPORTED;     // (32-bit loops)
  if (!logits || (logprobs && !tokens) || (top_k > 0 && (!top_ids || !top_logprobs))) return FP8GQ_ERR_NULL_POINTER;
  if (T > 1 && ld < V) return FP8GQ_ERR_STRIDE;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == FP8GQ_DTYPE_BF16 ? 1u : 3u)) return FP8GQ_ERR_ALIGNMENT;
  DeviceInfo di;
  int st = device_info(&di, nullptr);
  if (st != FP8GQ_OK) return st;
  LogprobParams p{};
  p.logits = logits;
  p.ld = ld;
  p.tokens = tokens;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.top_ids = top_ids;
  p.top_logprobs = top_logprobs;
  p.T = T;
  p.V = V;
  p.K = top_k;
  auto fn = dtype == FP8GQ_DTYPE_BF16 ? token_logprobs_kernel<__nv_bfloat16> : token_logprobs_kernel<float>;
  p.cluster = logprobs_cluster(T, V, di.sm_count);
  const size_t smem = kLpStages * kLpStepBytes;
  cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(fn), static_cast<int>(smem));
  if (e == cudaSuccess && p.cluster > 8) e = ensure_nonportable_clusters(reinterpret_cast<const void*>(fn));
  if (e == cudaSuccess)
    e = launch_with_pdl_cluster(fn, dim3(static_cast<unsigned>(T) * p.cluster), dim3(kLpThreads), smem,
                                static_cast<cudaStream_t>(stream), p.cluster, p);
  return e == cudaSuccess ? launch_status() : cuda_fail(e, "fp8gq_token_logprobs");
}

}  // extern "C"
