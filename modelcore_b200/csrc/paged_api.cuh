// C-ABI entry points of the paged cache (declared in include/mcb200.h): host-side validation and
// launches.  Included by mcb200.cu, whose helpers it uses.
#pragma once

namespace {

// Runs a C entry's body: no C++ exception (a failed host allocation) leaves the library.
template <typename F>
int guarded(const char* what, F body) {
  try {
    return body();
  } catch (...) {
    try {
      return fail(MCB_ERR_CUDA, "%s: host allocation failed", what);
    } catch (...) {
      return MCB_ERR_CUDA;
    }
  }
}

int page_shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

int check_page_size(int page_size, const char* who) {
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
    return fail(MCB_ERR_UNSUPPORTED, "%s: page_size %d (a power of two from 16 to 1024)", who, page_size);
  return MCB_OK;
}

int check_pool(int n_pages, int page_size, int max_pages, const char* who) {
  if (n_pages <= 0 || max_pages <= 0)
    return fail(MCB_ERR_INVALID_ARG, "%s: n_pages %d and max_pages %d must be positive", who, n_pages, max_pages);
  if (static_cast<long long>(max_pages) * page_size > INT32_MAX)
    return fail(MCB_ERR_UNSUPPORTED, "%s: max_pages %d * page_size %d positions a request (at most 2^31 - 1)", who,
                max_pages, page_size);
  return check_page_size(page_size, who);
}

int page_plan(const mcb_page_plan_args* a, void* stream) {
  const char* who = "mcb_page_plan";
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->R < 0 || a->N < 0) return fail(MCB_ERR_INVALID_ARG, "%s: bad sizes R=%d N=%d", who, a->R, a->N);
  int rc = check_pool(a->n_pages, a->page_size, a->max_pages, who);
  if (rc != MCB_OK) return rc;
  if (a->cu_new == nullptr || a->free_state == nullptr || a->free_state_out == nullptr || a->free_pages == nullptr ||
      (a->R > 0 && (a->cache_seqlens == nullptr || a->new_lens == nullptr || a->block_table == nullptr)) ||
      a->counter == nullptr || (a->N > 0 && (a->positions == nullptr || a->slot_map == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  if (a->table_stride < a->max_pages)
    return fail(MCB_ERR_INVALID_ARG, "%s: table_stride %lld below max_pages %d", who,
                static_cast<long long>(a->table_stride), a->max_pages);
  mcb::PagePlanParams p = {};
  p.seqlens = a->cache_seqlens;
  p.new_lens = a->new_lens;
  p.block_table = a->block_table;
  p.table_stride = a->table_stride;
  p.free_pages = a->free_pages;
  p.free_state = reinterpret_cast<const long long*>(a->free_state);
  p.free_state_out = reinterpret_cast<long long*>(a->free_state_out);
  p.cu_new = a->cu_new;
  p.positions = a->positions;
  p.slot_map = reinterpret_cast<long long*>(a->slot_map);
  p.R = a->R;
  p.N = a->N;
  p.n_pages = a->n_pages;
  p.max_pages = a->max_pages;
  p.page_shift = page_shift_of(a->page_size);
  p.counter = a->counter;
  // a thread a row up to 1,024, and about two tokens a thread before another CTA joins
  const int threads = a->R <= 256 && a->N <= 512 ? 256 : mcb::kPlanMaxThreads;
  const int ctas = static_cast<int>(std::clamp<long long>((a->N + 2ll * threads - 1) / (2 * threads), 1,
                                                          device_sm_count()));
  cudaError_t e = launch_pdl(mcb::page_plan_kernel, dim3(static_cast<unsigned>(ctas)),
                             dim3(static_cast<unsigned>(threads)), 0, static_cast<cudaStream_t>(stream), p);
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "page_plan launch");
  return MCB_OK;
}

int page_release(const mcb_page_release_args* a, const int32_t* keep_lens, const char* who, void* stream) {
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->R < 0) return fail(MCB_ERR_INVALID_ARG, "%s: bad size R=%d", who, a->R);
  int rc = check_pool(a->n_pages, a->page_size, a->max_pages, who);
  if (rc != MCB_OK) return rc;
  if (a->free_state == nullptr || a->free_state_out == nullptr || a->free_pages == nullptr || a->counter == nullptr ||
      (a->R > 0 && (a->done == nullptr || a->cache_seqlens == nullptr || a->block_table == nullptr ||
                    a->seqlens_out == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  if (a->table_stride < a->max_pages)
    return fail(MCB_ERR_INVALID_ARG, "%s: table_stride %lld below max_pages %d", who,
                static_cast<long long>(a->table_stride), a->max_pages);
  mcb::PageReleaseParams p = {};
  p.done = a->done;
  p.seqlens = a->cache_seqlens;
  p.block_table = a->block_table;
  p.table_stride = a->table_stride;
  p.free_pages = a->free_pages;
  p.free_state = reinterpret_cast<const long long*>(a->free_state);
  p.free_state_out = reinterpret_cast<long long*>(a->free_state_out);
  p.seqlens_out = a->seqlens_out;
  p.keep_lens = keep_lens;
  p.R = a->R;
  p.n_pages = a->n_pages;
  p.max_pages = a->max_pages;
  p.page_shift = page_shift_of(a->page_size);
  p.counter = a->counter;
  // at most a table's worth of pages comes back, eight a thread
  const int threads = a->R <= 256 ? 256 : mcb::kPlanMaxThreads;
  const long long most = static_cast<long long>(a->R) * a->max_pages;
  const int ctas = static_cast<int>(std::clamp<long long>(most / (8 * threads), 1, device_sm_count()));
  cudaError_t e = launch_pdl(mcb::page_release_kernel, dim3(static_cast<unsigned>(ctas)),
                             dim3(static_cast<unsigned>(threads)), 0, static_cast<cudaStream_t>(stream), p);
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "page_release launch");
  return MCB_OK;
}

// (token, head) strides of packed head vectors; the stride of a dimension of one is arbitrary and not used.
struct PackedStrides {
  int64_t s[2];
  PackedStrides(const int64_t (&given)[2], int tokens, int heads, int D)
      : s{tokens > 1 ? given[0] : static_cast<int64_t>(heads) * D, heads > 1 ? given[1] : D} {}
};

bool rows16(const void* p, const int64_t (&strides)[2]) {
  return aligned(p, 16) && strides[0] % 8 == 0 && strides[1] % 8 == 0;
}

int check_paged_heads(int D, const char* who) {
  if (D != 64 && D != 128) return fail(MCB_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", who, D);
  return MCB_OK;
}

int paged_append(const mcb_paged_append_args* a, void* stream) {
  const char* who = "mcb_paged_append_rope";
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->N < 0 || a->Hq <= 0 || a->Hkv <= 0)
    return fail(MCB_ERR_INVALID_ARG, "%s: bad sizes N=%d Hq=%d Hkv=%d", who, a->N, a->Hq, a->Hkv);
  int rc = check_paged_heads(a->D, who);
  if (rc != MCB_OK) return rc;
  const bool kv = a->k != nullptr;
  if (kv != (a->v != nullptr)) return fail(MCB_ERR_INVALID_ARG, "%s: k and v come together", who);
  if (a->N == 0) return MCB_OK;
  if (a->q == nullptr || a->q_out == nullptr || a->positions == nullptr || a->cos == nullptr || a->sin == nullptr ||
      (kv && (a->k_pages == nullptr || a->v_pages == nullptr || a->slot_map == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  if (a->rot_len <= 0) return fail(MCB_ERR_INVALID_ARG, "%s: rot_len %d", who, a->rot_len);
  if (kv) {
    rc = check_page_size(a->page_size, who);
    if (rc != MCB_OK) return rc;
    if (a->n_pages <= 0) return fail(MCB_ERR_INVALID_ARG, "%s: n_pages %d", who, a->n_pages);
  }
  const PackedStrides qs(a->q_stride, a->N, a->Hq, a->D), ks(a->k_stride, a->N, a->Hkv, a->D),
      vs(a->v_stride, a->N, a->Hkv, a->D);
  for (int i = 0; i < 2; ++i)
    if (qs.s[i] < 0 || (kv && (ks.s[i] < 0 || vs.s[i] < 0)))
      return fail(MCB_ERR_INVALID_ARG, "%s: negative stride", who);
  if (!rows16(a->q, qs.s) || !aligned(a->q_out, 16) || !aligned(a->cos, 16) || !aligned(a->sin, 16) ||
      (kv && (!rows16(a->k, ks.s) || !rows16(a->v, vs.s) || !aligned(a->k_pages, 16) ||
              !aligned(a->v_pages, 16))))
    return fail(MCB_ERR_ALIGNMENT, "%s: head vectors, tables and pages must start on 16-byte boundaries", who);
  mcb::PagedAppendParams p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = qs.s[i];
    p.ks[i] = ks.s[i];
    p.vs[i] = vs.s[i];
  }
  p.q_out = static_cast<uint16_t*>(a->q_out);
  p.k_pages = static_cast<uint16_t*>(a->k_pages);
  p.v_pages = static_cast<uint16_t*>(a->v_pages);
  p.positions = a->positions;
  p.slot_map = reinterpret_cast<const long long*>(a->slot_map);
  p.cos = static_cast<const uint16_t*>(a->cos);
  p.sin = static_cast<const uint16_t*>(a->sin);
  p.N = a->N;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.page_shift = kv ? page_shift_of(a->page_size) : 0;
  p.n_slots = static_cast<long long>(a->n_pages) * a->page_size;
  p.rot_len = a->rot_len;
  p.eps = a->eps;
  p.scale = a->scale;
  p.nk = kv ? a->Hkv : 0;
  p.rotate_k = a->rotate_k != 0;
  const long long heads = p.Hq + 2ll * p.nk, vpw = 32 / (a->D / 16), steps = (heads + vpw - 1) / vpw;
  if (static_cast<long long>(a->N) * heads > INT32_MAX)
    return fail(MCB_ERR_UNSUPPORTED, "%s: %lld vectors in one call (at most 2^31 - 1)", who,
                static_cast<long long>(a->N) * heads);
  // a warp a token once tokens fill the resident warps; before that its heads over several
  const long long wpb = mcb::kAppendVecThreads / 32;
  const long long resident = static_cast<long long>(kAppendVecCtasPerSm) * device_sm_count();
  p.parts = static_cast<int>(std::clamp<long long>(resident * wpb / a->N, 1, steps));
  const long long blocks = std::min<long long>((static_cast<long long>(a->N) * p.parts + wpb - 1) / wpb, resident);
  const dim3 grid(static_cast<unsigned>(blocks)), block(mcb::kAppendVecThreads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->D == 64)
    e = a->round_each ? launch_pdl(mcb::paged_append_kernel<64, true>, grid, block, 0, st, p)
                      : launch_pdl(mcb::paged_append_kernel<64, false>, grid, block, 0, st, p);
  else
    e = a->round_each ? launch_pdl(mcb::paged_append_kernel<128, true>, grid, block, 0, st, p)
                      : launch_pdl(mcb::paged_append_kernel<128, false>, grid, block, 0, st, p);
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paged_append launch");
  return MCB_OK;
}

// Shape checks of mcb_paged_attn: what its size queries need as well.
int check_paged_attn(const mcb_paged_attn_args* a, const char* who) {
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->R < 0 || a->N < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->max_new < 0)
    return fail(MCB_ERR_INVALID_ARG, "%s: bad sizes R=%d N=%d Hq=%d Hkv=%d max_new=%d", who, a->R, a->N, a->Hq,
                a->Hkv, a->max_new);
  if (a->Hq % a->Hkv != 0)
    return fail(MCB_ERR_INVALID_ARG, "%s: Hq %d must be divisible by Hkv %d", who, a->Hq, a->Hkv);
  if (a->Hq / a->Hkv > 128)
    return fail(MCB_ERR_UNSUPPORTED, "%s: %d query heads a kv head (at most 128)", who, a->Hq / a->Hkv);
  int rc = check_paged_heads(a->D, who);
  if (rc != MCB_OK) return rc;
  rc = check_pool(a->n_pages, a->page_size, a->max_pages, who);
  if (rc != MCB_OK) return rc;
  if (!(a->softmax_scale > 0.f) || a->softmax_scale > 3e38f)
    return fail(MCB_ERR_INVALID_ARG, "%s: softmax_scale %g must be positive and finite", who, a->softmax_scale);
  if (static_cast<long long>(a->N) * a->Hq > INT32_MAX)
    return fail(MCB_ERR_UNSUPPORTED, "%s: N %d * Hq %d above 2^31 - 1", who, a->N, a->Hq);
  if ((a->n_pages + 1ll) * a->Hkv > INT32_MAX)
    return fail(MCB_ERR_UNSUPPORTED, "%s: n_pages %d * Hkv %d above 2^31 - 1", who, a->n_pages, a->Hkv);
  return MCB_OK;
}

// The pages as a 4-D map {64 columns, position, D / 64 panels, page * Hkv + head}: a box of `box`
// positions of one head's page is one contiguous block, landing as D / 64 swizzled panels.
int encode_page_map(CUtensorMap* map, const void* base, const mcb_paged_attn_args* a, int box, int panels) {
  auto fn = encode_fn();
  if (fn == nullptr) return fail(MCB_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t D = static_cast<cuuint64_t>(a->D), page = static_cast<cuuint64_t>(a->page_size);
  cuuint64_t dims[4] = {64, page, D / 64, static_cast<cuuint64_t>(a->n_pages) * static_cast<cuuint64_t>(a->Hkv)};
  cuuint64_t strides[3] = {D * 2, 128, page * D * 2};
  cuuint32_t boxes[4] = {64u, static_cast<cuuint32_t>(box), static_cast<cuuint32_t>(panels), 1u};
  cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, boxes, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MCB_ERR_CUDA, "cuTensorMapEncodeTiled(pages) failed (CUresult %d)", (int)r);
  return MCB_OK;
}

template <int D, int NQT>
struct PagedDecodeVariant {
  // 128-KB and 48-KB rings: one CTA an SM at head size 128, three (two with 16 query rows) at 64.  Two
  // groups of consumer warps where they fit: batch 128 of 16/4 heads of 128, 198 -> 191 us.
  static constexpr int STAGES = D == 64 ? 3 : 4;
  static constexpr int GROUPS = D == 128 && NQT == 1 ? 2 : 1;
  using Cfg = mcb::PagedDecodeConfig<D, NQT, STAGES, GROUPS>;
  static constexpr auto kernel = mcb::paged_decode_kernel<D, NQT, STAGES, GROUPS>;

  // CTAs resident on the device (the shared-memory limit raised once); one an SM without a device.
  static int grid() {
    static std::atomic<uint64_t> done{0};
    static std::mutex mu;
    static int cache[64] = {0};
    const int per_sm = per_device(cache, mu, [] {
      int n = 0;
      if (ensure_smem(kernel, Cfg::SMEM_BYTES, done) != cudaSuccess ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, Cfg::THREADS, Cfg::SMEM_BYTES) != cudaSuccess)
        cudaGetLastError();
      return n;
    });
    return std::min(device_sm_count() * std::max(per_sm, 1), 1024);  // (share_begin's bound)
  }

  static int launch(const mcb_paged_attn_args* a, const mcb::PagedAttnParams& p, cudaStream_t st) {
    CUtensorMap km, vm;
    const int box = std::min(a->page_size, mcb::kPdTile);
    int rc = encode_page_map(&km, a->k_pages, a, box, D / 64);
    if (rc == MCB_OK) rc = encode_page_map(&vm, a->v_pages, a, box, D / 64);
    if (rc != MCB_OK) return rc;
    cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(grid())), dim3(Cfg::THREADS),
                               static_cast<size_t>(Cfg::SMEM_BYTES), st, km, vm, p);
    g_launches++;
    note_attn_kernel("paged_decode_kernel", D, NQT, STAGES, false);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "paged_decode launch");
    return MCB_OK;
  }
};

// Packed queries as a 3-D map {D, Hq, N}; a box is 64 columns x the G heads of a kv head x the tokens
// of a query tile, rows in (token, head) order.
int encode_packed_q_map(CUtensorMap* map, const mcb_paged_attn_args* a, const int64_t (&stride)[2], int tpb) {
  auto fn = encode_fn();
  if (fn == nullptr) return fail(MCB_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(a->D), static_cast<cuuint64_t>(a->Hq), static_cast<cuuint64_t>(a->N)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride[1]) * 2, static_cast<cuuint64_t>(stride[0]) * 2};
  cuuint32_t box[3] = {64u, static_cast<cuuint32_t>(a->Hq / a->Hkv), static_cast<cuuint32_t>(tpb)};
  cuuint32_t estr[3] = {1u, 1u, 1u};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a->q), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MCB_ERR_CUDA, "cuTensorMapEncodeTiled(packed q) failed (CUresult %d)", (int)r);
  return MCB_OK;
}

template <int D>
int launch_paged_chunk(const mcb_paged_attn_args* a, const mcb::PagedChunkParams& p, const int64_t (&q_stride)[2],
                       int grid, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  constexpr int smem = mcb::PagedChunkConfig<D>::kSmem;
  CUtensorMap qm, km, vm;
  const int box = std::min(a->page_size, mcb::kPcTile);
  int rc = encode_packed_q_map(&qm, a, q_stride, p.a.tpb);
  if (rc == MCB_OK) rc = encode_page_map(&km, a->k_pages, a, box, 1);
  if (rc == MCB_OK) rc = encode_page_map(&vm, a->v_pages, a, box, 1);
  if (rc != MCB_OK) return rc;
  cudaError_t e = ensure_smem(mcb::paged_chunk_kernel<D>, smem, done);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_chunk)");
  e = launch_pdl(mcb::paged_chunk_kernel<D>, dim3(static_cast<unsigned>(grid)), dim3(mcb::kPcThreads),
                 static_cast<size_t>(smem), st, qm, km, vm, p);
  g_launches++;
  note_attn_kernel("paged_chunk_kernel", D, 0, 0, false);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paged_chunk launch");
  e = launch_pdl(mcb::paged_combine_kernel<D>, dim3(static_cast<unsigned>(grid), 8), dim3(256), 0, st, p);
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paged_combine launch");
  return MCB_OK;
}

// How a call runs, from its shapes alone: which kernels, their grids, and the workspace's parts
// (the decode kernel's partials, then the chunk kernel's partials and its cut units).
struct PagedAttnPlan {
  bool decode, chunk;
  int nqt, decode_grid, chunk_grid;
  size_t d_o, d_lse, c_o, c_lse, c_cuts, ws_bytes, counters;
};

template <typename F>
auto with_decode_variant(int D, int nqt, F f) {
  if (D == 64) return nqt == 1 ? f(PagedDecodeVariant<64, 1>{}) : f(PagedDecodeVariant<64, 2>{});
  return nqt == 1 ? f(PagedDecodeVariant<128, 1>{}) : f(PagedDecodeVariant<128, 2>{});
}

PagedAttnPlan plan_paged_attn(const mcb_paged_attn_args* a) {
  PagedAttnPlan pl = {};
  const long long G = a->Hq / a->Hkv;
  const long long most = a->max_new > 0 ? a->max_new * G : 1ll << 40;  // query rows a kv head of a request
  pl.decode = G <= 16;
  pl.chunk = most > 16;  // (always when G > 16)
  // 8 query rows a unit where every request has no more, and beside the chunk kernel (whose share is
  // then the requests of 9 to 16 rows too): the variant of 8 reads half as fast again an SM
  pl.nqt = most <= 8 || (pl.chunk && G <= 8) ? 1 : 2;
  if (pl.decode) {
    pl.decode_grid = with_decode_variant(a->D, pl.nqt, [](auto v) { return decltype(v)::grid(); });
    const size_t rows = static_cast<size_t>(pl.decode_grid) * 2 * 8 * pl.nqt;
    pl.d_o = round256(rows * a->D * 4);
    pl.d_lse = round256(rows * 4);
    pl.counters = static_cast<size_t>(pl.decode_grid);
  }
  if (pl.chunk) {
    pl.chunk_grid = device_sm_count();
    const size_t rows = static_cast<size_t>(pl.chunk_grid) * 2 * 256;
    pl.c_o = round256(rows * a->D * 4);
    pl.c_lse = round256(rows * 4);
    pl.c_cuts = round256(pl.chunk_grid * sizeof(mcb::PagedCut));
  }
  pl.ws_bytes = pl.d_o + pl.d_lse + pl.c_o + pl.c_lse + pl.c_cuts;
  return pl;
}

int paged_attn(const mcb_paged_attn_args* a, void* stream) {
  const char* who = "mcb_paged_attn";
  int rc = check_paged_attn(a, who);
  if (rc != MCB_OK) return rc;
  if (a->N == 0) return MCB_OK;
  if (a->q == nullptr || a->out == nullptr || a->k_pages == nullptr || a->v_pages == nullptr ||
      a->cu_new == nullptr || (a->R > 0 && (a->block_table == nullptr || a->cache_seqlens == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  const PackedStrides qs(a->q_stride, a->N, a->Hq, a->D);
  const auto& q_stride = qs.s;
  if (q_stride[0] < 0 || q_stride[1] < 0 || a->table_stride < a->max_pages)
    return fail(MCB_ERR_INVALID_ARG, "%s: negative q stride or table_stride below max_pages", who);
  if (!rows16(a->q, q_stride) || !aligned(a->out, 16) || !aligned(a->k_pages, 16) || !aligned(a->v_pages, 16))
    return fail(MCB_ERR_ALIGNMENT, "%s: q rows, out and pages must start on 16-byte boundaries", who);
  const PagedAttnPlan pl = plan_paged_attn(a);
  if (a->workspace == nullptr || a->workspace_bytes < pl.ws_bytes || !aligned(a->workspace, 256))
    return fail(MCB_ERR_WORKSPACE, "%s: a 256-byte aligned workspace of %zu bytes is needed, got %zu", who, pl.ws_bytes,
                a->workspace_bytes);
  if (pl.counters > 0 && (a->counters == nullptr || a->counter_count < pl.counters))
    return fail(MCB_ERR_WORKSPACE, "%s: %zu counters are needed, got %zu", who, pl.counters, a->counter_count);
  mcb::PagedAttnParams p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.qs[0] = q_stride[0];
  p.qs[1] = q_stride[1];
  p.block_table = a->block_table;
  p.table_stride = a->table_stride;
  p.seqlens = a->cache_seqlens;
  p.cu_new = a->cu_new;
  p.out = static_cast<uint16_t*>(a->out);
  p.counters = a->counters;
  p.R = a->R;
  p.N = a->N;
  p.Hq = a->Hq;
  p.Hkv = a->Hkv;
  p.G = a->Hq / a->Hkv;
  p.n_pages = a->n_pages;
  p.max_pages = a->max_pages;
  p.page_shift = page_shift_of(a->page_size);
  p.window = a->window;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.few_rows = pl.decode ? 8 * pl.nqt : 0;
  p.tpb = mcb::kPcTile / p.G;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  if (pl.decode) {
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_lse = reinterpret_cast<float*>(ws + pl.d_o);
    p.all = !pl.chunk;
    p.fill = !pl.chunk;
    rc = with_decode_variant(a->D, pl.nqt, [&](auto v) { return decltype(v)::launch(a, p, st); });
    if (rc != MCB_OK || !pl.chunk) return rc;
  }
  ws += pl.d_o + pl.d_lse;
  mcb::PagedChunkParams c = {};
  c.a = p;
  c.a.part_o = reinterpret_cast<float*>(ws);
  c.a.part_lse = reinterpret_cast<float*>(ws + pl.c_o);
  c.a.all = 0;
  c.a.fill = 1;
  c.cuts = reinterpret_cast<mcb::PagedCut*>(ws + pl.c_o + pl.c_lse);
  c.wait_last = pl.decode;
  return a->D == 64 ? launch_paged_chunk<64>(a, c, q_stride, pl.chunk_grid, st)
                    : launch_paged_chunk<128>(a, c, q_stride, pl.chunk_grid, st);
}

}  // namespace

extern "C" {

int mcb_page_plan(const mcb_page_plan_args* a, void* stream) {
  return guarded("mcb_page_plan", [&] { return page_plan(a, stream); });
}
int mcb_page_release(const mcb_page_release_args* a, void* stream) {
  return guarded("mcb_page_release", [&] { return page_release(a, nullptr, "mcb_page_release", stream); });
}
int mcb_page_release_to(const mcb_page_release_args* a, const int32_t* keep_lens, void* stream) {
  return guarded("mcb_page_release_to", [&] { return page_release(a, keep_lens, "mcb_page_release_to", stream); });
}
int mcb_paged_append_rope(const mcb_paged_append_args* a, void* stream) {
  return guarded("mcb_paged_append_rope", [&] { return paged_append(a, stream); });
}
size_t mcb_paged_attn_workspace_size(const mcb_paged_attn_args* a) {
  size_t n = 0;
  guarded("mcb_paged_attn_workspace_size", [&] {
    const int rc = check_paged_attn(a, "mcb_paged_attn_workspace_size");
    if (rc == MCB_OK) n = plan_paged_attn(a).ws_bytes;
    return rc;
  });
  return n;
}
size_t mcb_paged_attn_counter_count(const mcb_paged_attn_args* a) {
  size_t n = 0;
  guarded("mcb_paged_attn_counter_count", [&] {
    const int rc = check_paged_attn(a, "mcb_paged_attn_counter_count");
    if (rc == MCB_OK) n = plan_paged_attn(a).counters;
    return rc;
  });
  return n;
}
int mcb_paged_attn(const mcb_paged_attn_args* a, void* stream) {
  return guarded("mcb_paged_attn", [&] { return paged_attn(a, stream); });
}

}  // extern "C"
