// C-ABI entry points of speculative decoding and of shared pages (declared in include/mcb200.h):
// host-side validation and launches.  Included by mcb200.cu after paged_api.cuh, whose helpers it uses.
#pragma once

namespace {

int check_words(int words, const char* who) {
  if (words < 1 || words > mcb::kTreeMaxWords)
    return fail(MCB_ERR_UNSUPPORTED, "%s: words %d (1 to %d: 32 to %d new tokens with a mask)", who, words,
                mcb::kTreeMaxWords, 32 * mcb::kTreeMaxWords);
  return MCB_OK;
}

template <int W>
cudaError_t launch_draft_tree(const mcb::DraftTreeParams& p, int words, cudaStream_t st) {
  if constexpr (W < mcb::kTreeMaxWords)
    if (words > W) return launch_draft_tree<W + 1>(p, words, st);
  // a CTA a request, at least the padding tokens' one
  return launch_pdl(mcb::draft_tree_kernel<W>, dim3(static_cast<unsigned>(std::clamp(p.R, 1, 1 << 20))), dim3(32 * W), 0,
                    st, p);
}

int draft_tree(const mcb_draft_tree_args* a, void* stream) {
  const char* who = "mcb_draft_tree";
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->R < 0 || a->N < 0) return fail(MCB_ERR_INVALID_ARG, "%s: bad sizes R=%d N=%d", who, a->R, a->N);
  const int rc = check_words(a->words, who);
  if (rc != MCB_OK) return rc;
  if (a->N == 0) return MCB_OK;
  if (a->parents == nullptr || a->cu_new == nullptr || a->positions == nullptr || a->mask == nullptr ||
      (a->R > 0 && a->cache_seqlens == nullptr))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  mcb::DraftTreeParams p = {};
  p.parents = a->parents;
  p.cu = a->cu_new;
  p.seqlens = a->cache_seqlens;
  p.positions = a->positions;
  p.mask = reinterpret_cast<uint32_t*>(a->mask);
  p.R = a->R;
  p.N = a->N;
  cudaError_t e = launch_draft_tree<1>(p, a->words, static_cast<cudaStream_t>(stream));
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "draft_tree launch");
  return MCB_OK;
}

int check_paged_tree(const mcb_paged_tree_attn_args* a, const char* who) {
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  const int rc = check_paged_attn(&a->attn, who);
  return rc != MCB_OK ? rc : check_words(a->words, who);
}

// How a call runs, from its shapes alone: the workspace's parts are the tree kernel's partials and cut units, then
// the chunk kernel's.
struct PagedTreePlan {
  bool chunk;  // some request may be a chunk of a prompt
  int rows;    // query rows a unit: 16 or 32 with the keys on the M side, 256 the other kernel
  int grid;
  size_t o, lse, cuts, chunk_o, chunk_lse, ws_bytes, counters;
};

PagedTreePlan plan_paged_tree(const mcb_paged_tree_attn_args* t) {
  PagedTreePlan pl = {};
  const long long G = t->attn.Hq / t->attn.Hkv;
  // Chunks of up to 1,024 tokens share the tree kernel's launch, which saves two kernels; longer ones get the chunk
  // kernel, whose products are faster.  Two chunks beside 22 trees of 41 tokens, one launch against two, us by events:
  //   16/4 heads of 128 at 4,000 cached: chunks of 300 95, 125; of 1,000 148, 166; of 2,000 232, 237
  //                     at 16,000:       300 278, 300; 1,000 474, 451; 2,000 761, 682;  window 1,024: 42, 83; 71, 92; 93, 115
  //   12/12 of 64       at 500:          300 46, 63; 1,000 60, 72; 2,000 87, 98
  //                     at 4,000:        300 157, 129; 1,000 191, 150; 2,000 249, 197;  window 1,024: 67, 76; 83, 86; 97, 98
  // So with long cached lengths and no window two would be faster from some 300 to 1,000 tokens on; the lengths are not
  // known here.
  pl.chunk = t->attn.max_new == 0 || t->attn.max_new > std::max(32 * t->words, 1024);
  pl.grid = std::min(device_sm_count(), mcb::kTreeMostCuts);
  // trees of at most max_new tokens, where that is known: as few rows as hold them
  const long long most = (t->attn.max_new == 0 || pl.chunk ? 32 * t->words : t->attn.max_new) * G;
  pl.rows = most <= 16 ? 16 : most <= 32 ? 32 : 256;
  const size_t rows = static_cast<size_t>(pl.grid) * 2 * pl.rows, chunk_rows = static_cast<size_t>(pl.grid) * 2 * 256;
  pl.counters = pl.rows < 256 ? static_cast<size_t>(pl.grid) : 0;
  pl.o = round256(rows * t->attn.D * 4);
  pl.lse = round256(rows * 4);
  pl.cuts = round256(pl.grid * sizeof(mcb::PagedCut));
  pl.ws_bytes = pl.o + pl.lse + pl.cuts;
  if (pl.chunk) {
    pl.chunk_o = round256(chunk_rows * t->attn.D * 4);
    pl.chunk_lse = round256(chunk_rows * 4);
    pl.ws_bytes += pl.chunk_o + pl.chunk_lse + pl.cuts;
  }
  return pl;
}

template <int D, int R>
int launch_tree_few(const mcb_paged_attn_args* a, const mcb::PagedTreeParams& p, const int64_t (&q_stride)[2], int grid,
                    cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  constexpr int smem = mcb::TreeFewConfig<D, R>::kBytes;
  CUtensorMap qm, km, vm;
  const int box = std::min(a->page_size, mcb::kPtTile);
  int rc = encode_packed_q_map(&qm, a, q_stride, p.a.tpb);
  if (rc == MCB_OK) rc = encode_page_map(&km, a->k_pages, a, box, 1);
  if (rc == MCB_OK) rc = encode_page_map(&vm, a->v_pages, a, box, 1);
  if (rc != MCB_OK) return rc;
  cudaError_t e = ensure_smem(mcb::paged_tree_few_kernel<D, R>, smem, done);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_tree_few)");
  e = launch_pdl(mcb::paged_tree_few_kernel<D, R>, dim3(static_cast<unsigned>(grid)), dim3(mcb::kPtThreads),
                 static_cast<size_t>(smem), st, qm, km, vm, p);
  g_launches++;
  note_attn_kernel("paged_tree_few_kernel", D, 0, R, false);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paged_tree_few launch");
  return MCB_OK;
}

template <int D>
int launch_paged_tree(const mcb_paged_attn_args* a, const mcb::PagedTreeParams& p, const int64_t (&q_stride)[2], int grid,
                      cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  constexpr int smem = mcb::PagedTreeConfig<D>::kBytes;
  CUtensorMap qm, km, vm;
  const int box = std::min(a->page_size, mcb::kPtTile);
  int rc = encode_packed_q_map(&qm, a, q_stride, p.a.tpb);
  if (rc == MCB_OK) rc = encode_page_map(&km, a->k_pages, a, box, 1);
  if (rc == MCB_OK) rc = encode_page_map(&vm, a->v_pages, a, box, 1);
  if (rc != MCB_OK) return rc;
  cudaError_t e = ensure_smem(mcb::paged_tree_kernel<D>, smem, done);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(paged_tree)");
  e = launch_pdl(mcb::paged_tree_kernel<D>, dim3(static_cast<unsigned>(grid)), dim3(mcb::kPtThreads),
                 static_cast<size_t>(smem), st, qm, km, vm, p);
  g_launches++;
  note_attn_kernel("paged_tree_kernel", D, 0, 0, false);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paged_tree launch");
  e = launch_pdl(mcb::tree_combine_kernel<D>, dim3(static_cast<unsigned>(grid), 8), dim3(256), 0, st, p);
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "tree_combine launch");
  return MCB_OK;
}

int paged_tree_attn(const mcb_paged_tree_attn_args* t, void* stream) {
  const char* who = "mcb_paged_tree_attn";
  int rc = check_paged_tree(t, who);
  if (rc != MCB_OK) return rc;
  const mcb_paged_attn_args* a = &t->attn;
  if (a->N == 0) return MCB_OK;
  if (a->q == nullptr || a->out == nullptr || a->k_pages == nullptr || a->v_pages == nullptr ||
      a->cu_new == nullptr || t->positions == nullptr || t->mask == nullptr ||
      (a->R > 0 && (a->block_table == nullptr || a->cache_seqlens == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  const PackedStrides qs(a->q_stride, a->N, a->Hq, a->D);
  if (qs.s[0] < 0 || qs.s[1] < 0 || a->table_stride < a->max_pages)
    return fail(MCB_ERR_INVALID_ARG, "%s: negative q stride or table_stride below max_pages", who);
  if (!rows16(a->q, qs.s) || !aligned(a->out, 16) || !aligned(a->k_pages, 16) || !aligned(a->v_pages, 16))
    return fail(MCB_ERR_ALIGNMENT, "%s: q rows, out and pages must start on 16-byte boundaries", who);
  const PagedTreePlan pl = plan_paged_tree(t);
  if (a->workspace == nullptr || a->workspace_bytes < pl.ws_bytes || !aligned(a->workspace, 256))
    return fail(MCB_ERR_WORKSPACE, "%s: a 256-byte aligned workspace of %zu bytes is needed, got %zu", who, pl.ws_bytes,
                a->workspace_bytes);
  if (pl.counters > 0 && (a->counters == nullptr || a->counter_count < pl.counters))
    return fail(MCB_ERR_WORKSPACE, "%s: %zu counters are needed, got %zu", who, pl.counters, a->counter_count);
  mcb::PagedTreeParams p = {};
  p.a.q = static_cast<const uint16_t*>(a->q);
  p.a.qs[0] = qs.s[0];
  p.a.qs[1] = qs.s[1];
  p.a.block_table = a->block_table;
  p.a.table_stride = a->table_stride;
  p.a.seqlens = a->cache_seqlens;
  p.a.cu_new = a->cu_new;
  p.a.counters = a->counters;
  p.a.out = static_cast<uint16_t*>(a->out);
  p.a.R = a->R;
  p.a.N = a->N;
  p.a.Hq = a->Hq;
  p.a.Hkv = a->Hkv;
  p.a.G = a->Hq / a->Hkv;
  p.a.n_pages = a->n_pages;
  p.a.max_pages = a->max_pages;
  p.a.page_shift = page_shift_of(a->page_size);
  p.a.window = a->window;
  p.a.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.a.few_rows = 32 * t->words * p.a.G;  // the chunk kernel's share begins above
  p.a.tpb = std::min(pl.rows, mcb::kPtTile) / p.a.G;
  p.unit_tok = pl.rows == 256 ? 2 * p.a.tpb : p.a.tpb;
  p.a.all = !pl.chunk;
  p.a.fill = 1;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.a.part_o = reinterpret_cast<float*>(ws);
  p.a.part_lse = reinterpret_cast<float*>(ws + pl.o);
  p.cuts = reinterpret_cast<mcb::PagedCut*>(ws + pl.o + pl.lse);
  p.positions = t->positions;
  p.mask = reinterpret_cast<const uint32_t*>(t->mask);
  p.words = t->words;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = [&](auto d) {
    constexpr int D = decltype(d)::value;
    switch (pl.rows) {
      case 16: return launch_tree_few<D, 16>(a, p, qs.s, pl.grid, st);
      case 32: return launch_tree_few<D, 32>(a, p, qs.s, pl.grid, st);
      default: return launch_paged_tree<D>(a, p, qs.s, pl.grid, st);
    }
  };
  rc = a->D == 64 ? launch(std::integral_constant<int, 64>()) : launch(std::integral_constant<int, 128>());
  if (rc != MCB_OK || !pl.chunk) return rc;
  mcb::PagedChunkParams c = {};
  c.a = p.a;
  c.a.all = 0;
  c.a.fill = 0;
  c.a.tpb = mcb::kPcTile / p.a.G;
  ws += pl.o + pl.lse + pl.cuts;
  c.a.part_o = reinterpret_cast<float*>(ws);
  c.a.part_lse = reinterpret_cast<float*>(ws + pl.chunk_o);
  c.cuts = reinterpret_cast<mcb::PagedCut*>(ws + pl.chunk_o + pl.chunk_lse);
  c.wait_last = 1;
  return a->D == 64 ? launch_paged_chunk<64>(a, c, qs.s, pl.grid, st) : launch_paged_chunk<128>(a, c, qs.s, pl.grid, st);
}

int verify_drafts(const mcb_verify_drafts_args* a, void* stream) {
  const char* who = "mcb_verify_drafts";
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  if (a->R < 0 || a->N < 0 || a->V <= 0 || a->max_path <= 0)
    return fail(MCB_ERR_INVALID_ARG, "%s: bad sizes R=%d N=%d V=%d max_path=%d", who, a->R, a->N, a->V, a->max_path);
  if (a->V > 1 << 30) return fail(MCB_ERR_UNSUPPORTED, "%s: V %d (at most 2^30)", who, a->V);
  if (!(a->temperature >= 0.f) || a->temperature > 3e38f)
    return fail(MCB_ERR_INVALID_ARG, "%s: temperature %g must be finite and not negative", who, a->temperature);
  // (outside, a logit of -infinity or 0 as the kernel widens it, 2^128 and 2^-127, would count beside the others)
  if (a->temperature != 0.f && (a->temperature < 1e-20f || a->temperature > 1e20f))
    return fail(MCB_ERR_UNSUPPORTED, "%s: temperature %g (0, or from 1e-20 to 1e20)", who, a->temperature);
  if (a->R == 0) return MCB_OK;
  if (a->cu_new == nullptr || a->draws == nullptr || a->accepted == nullptr || a->path == nullptr ||
      a->next_token == nullptr ||
      (a->N > 0 && (a->logits == nullptr || a->tokens == nullptr || a->parents == nullptr || a->accept == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  if ((a->N > 1 && a->logits_stride < a->V) || (a->draft_probs != nullptr && a->N > 1 && a->draft_stride < a->V))
    return fail(MCB_ERR_INVALID_ARG, "%s: rows closer together than V %d", who, a->V);
  mcb::VerifyParams p = {};
  p.logits = a->logits;
  p.logits_stride = a->logits_stride;
  p.tokens = reinterpret_cast<const long long*>(a->tokens);
  p.parents = a->parents;
  p.cu = a->cu_new;
  p.accept = a->accept;
  p.draws = a->draws;
  p.draft = a->draft_probs;
  p.draft_stride = a->draft_stride;
  p.accepted = a->accepted;
  p.path = a->path;
  p.next = reinterpret_cast<long long*>(a->next_token);
  p.R = a->R;
  p.N = a->N;
  p.V = a->V;
  p.max_path = a->max_path;
  p.temperature = a->temperature;
  // CTAs a request: as many as the GPU holds at two an SM, up to the portable cluster, none with less than 2,048
  // tokens
  int c = 1;
  while (c < 8 && 2ll * c * a->R <= 2ll * device_sm_count() && a->V / (2 * c) >= 2048) c *= 2;
  if (static_cast<long long>(a->R) * c > INT32_MAX)
    return fail(MCB_ERR_UNSUPPORTED, "%s: R %d requests", who, a->R);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a->R * c));
  cfg.blockDim = dim3(mcb::kVerifyThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(c);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = a->logits_bf16 ? cudaLaunchKernelEx(&cfg, mcb::verify_kernel<uint16_t>, p)
                                 : cudaLaunchKernelEx(&cfg, mcb::verify_kernel<float>, p);
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "verify_drafts launch");
  return MCB_OK;
}

// The pool of all slots, as page_fork and paged_keep take it.
template <typename Args>
int check_slots(const Args* a, const char* who) {
  if (a->R < 0 || a->slots <= 0 || a->Hkv <= 0)
    return fail(MCB_ERR_INVALID_ARG, "%s: bad sizes R=%d slots=%d Hkv=%d", who, a->R, a->slots, a->Hkv);
  int rc = check_paged_heads(a->D, who);
  if (rc != MCB_OK) return rc;
  rc = check_pool(a->n_pages, a->page_size, a->max_pages, who);
  if (rc != MCB_OK) return rc;
  if ((a->n_pages + 1ll) * a->Hkv > INT32_MAX)
    return fail(MCB_ERR_UNSUPPORTED, "%s: n_pages %d * Hkv %d above 2^31 - 1", who, a->n_pages, a->Hkv);
  return MCB_OK;
}

int paged_keep(const mcb_paged_keep_args* a, void* stream) {
  const char* who = "mcb_paged_keep";
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  const int rc = check_slots(a, who);
  if (rc != MCB_OK) return rc;
  if (a->P < 0) return fail(MCB_ERR_INVALID_ARG, "%s: bad size P=%d", who, a->P);
  if (a->R >= 65535) return fail(MCB_ERR_UNSUPPORTED, "%s: R %d requests (at most 65,534)", who, a->R);
  if (a->free_state == nullptr || a->free_state_out == nullptr || a->free_pages == nullptr || a->counter == nullptr ||
      a->k_pages == nullptr || a->v_pages == nullptr ||
      (a->R > 0 && ((a->P > 0 && a->path == nullptr) || a->accepted == nullptr || a->cache_seqlens == nullptr ||
                    a->new_lens == nullptr || a->block_table == nullptr || a->seqlens_out == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  if (a->table_stride < a->max_pages || (a->R > 1 && a->path_stride < a->P))
    return fail(MCB_ERR_INVALID_ARG, "%s: table_stride below max_pages or path_stride below P", who);
  if (!aligned(a->k_pages, 16) || !aligned(a->v_pages, 16))
    return fail(MCB_ERR_ALIGNMENT, "%s: pages must start on 16-byte boundaries", who);
  mcb::PagedKeepParams p = {};
  p.path = a->path;
  p.kept = a->accepted;
  p.seqlens = a->cache_seqlens;
  p.new_lens = a->new_lens;
  p.table = a->block_table;
  p.queue = a->free_pages;
  p.state = reinterpret_cast<const long long*>(a->free_state);
  p.k_pages = static_cast<uint16_t*>(a->k_pages);
  p.v_pages = static_cast<uint16_t*>(a->v_pages);
  p.state_out = reinterpret_cast<long long*>(a->free_state_out);
  p.seqlens_out = a->seqlens_out;
  p.counter = a->counter;
  p.table_stride = a->table_stride;
  p.path_stride = a->path_stride;
  p.R = a->R;
  p.P = a->P;
  p.n_pages = a->n_pages;
  p.max_pages = a->max_pages;
  p.page_shift = page_shift_of(a->page_size);
  p.slots = a->slots;
  p.Hkv = a->Hkv;
  p.D = a->D;
  p.in_place = a->seqlens_out == a->cache_seqlens;
  const long long columns = 2ll * a->slots * a->Hkv * (a->D / 8);
  const long long ctas = (columns + mcb::kKeepThreads - 1) / mcb::kKeepThreads;
  if (ctas * (a->R + 1ll) > INT32_MAX)
    return fail(MCB_ERR_UNSUPPORTED, "%s: slots %d * Hkv %d * D %d of %d requests above 2^41", who, a->slots, a->Hkv, a->D,
                a->R);
  cudaError_t e = launch_pdl(mcb::paged_keep_kernel,
                             dim3(static_cast<unsigned>(ctas), static_cast<unsigned>(p.in_place ? std::max(a->R, 1) : a->R + 1)),
                             dim3(mcb::kKeepThreads), 0, static_cast<cudaStream_t>(stream), p);
  g_launches++;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paged_keep launch");
  return MCB_OK;
}

struct PageForkLayout {
  size_t meta, rows, counts, change, table, bytes;
  bool table_in_place;
};

PageForkLayout fork_layout(const mcb_page_fork_args* a) {
  PageForkLayout l = {};
  const size_t R = static_cast<size_t>(a->R), n = static_cast<size_t>(a->n_pages);
  l.table_in_place = a->block_table_out == a->block_table;
  l.rows = 256;
  l.counts = l.rows + 5 * round256(R * 4);
  l.change = l.counts + round256((n + mcb::kForkBlock - 1) / mcb::kForkBlock * 4);
  l.table = l.change + round256(n * 4);
  l.bytes = l.table + (l.table_in_place ? round256(R * static_cast<size_t>(a->max_pages) * 4) : 0);
  return l;
}

int page_fork(const mcb_page_fork_args* a, void* stream) {
  const char* who = "mcb_page_fork";
  if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "%s: args is NULL", who);
  const int rc = check_slots(a, who);
  if (rc != MCB_OK) return rc;
  if (a->free_state == nullptr || a->free_state_out == nullptr || a->free_pages == nullptr || a->shares == nullptr ||
      a->shares_out == nullptr || a->k_pages == nullptr || a->v_pages == nullptr ||
      (a->R > 0 && (a->source == nullptr || a->cache_seqlens == nullptr || a->block_table == nullptr ||
                    a->block_table_out == nullptr || a->seqlens_out == nullptr)))
    return fail(MCB_ERR_INVALID_ARG, "%s: NULL pointer argument", who);
  if (a->table_stride < a->max_pages || a->table_out_stride < a->max_pages)
    return fail(MCB_ERR_INVALID_ARG, "%s: table strides below max_pages %d", who, a->max_pages);
  if (!aligned(a->k_pages, 16) || !aligned(a->v_pages, 16))
    return fail(MCB_ERR_ALIGNMENT, "%s: pages must start on 16-byte boundaries", who);
  const PageForkLayout l = fork_layout(a);
  if (a->workspace == nullptr || a->workspace_bytes < l.bytes || !aligned(a->workspace, 256))
    return fail(MCB_ERR_WORKSPACE, "%s: a 256-byte aligned workspace of %zu bytes is needed, got %zu", who, l.bytes,
                a->workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  const size_t row = round256(static_cast<size_t>(a->R) * 4);
  auto ints = [&](size_t at) { return reinterpret_cast<int32_t*>(ws + at); };
  mcb::PageForkParams p = {};
  p.source = a->source;
  p.seqlens = a->cache_seqlens;
  p.table = a->block_table;
  p.shares = a->shares;
  p.queue = a->free_pages;
  p.state = reinterpret_cast<const long long*>(a->free_state);
  p.k_pages = static_cast<uint16_t*>(a->k_pages);
  p.v_pages = static_cast<uint16_t*>(a->v_pages);
  p.table_out = a->block_table_out;
  p.shares_out = a->shares_out;
  p.seqlens_out = a->seqlens_out;
  p.state_out = reinterpret_cast<long long*>(a->free_state_out);
  p.table_stride = a->table_stride;
  p.out_stride = a->table_out_stride;
  p.R = a->R;
  p.n_pages = a->n_pages;
  p.max_pages = a->max_pages;
  p.page_shift = page_shift_of(a->page_size);
  p.slots = a->slots;
  p.Hkv = a->Hkv;
  p.D = a->D;
  p.table_in_place = l.table_in_place;
  p.meta = reinterpret_cast<long long*>(ws);
  p.heirs = ints(l.rows);
  p.first = ints(l.rows + row);
  p.new_len = ints(l.rows + 2 * row);
  p.fresh = ints(l.rows + 3 * row);
  p.jobs = ints(l.rows + 4 * row);
  p.counts = ints(l.counts);
  p.change = ints(l.change);
  p.table_tmp = ints(l.table);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = device_sm_count();
  const unsigned blocks = static_cast<unsigned>((a->n_pages + mcb::kForkBlock - 1) / mcb::kForkBlock);
  cudaError_t e = launch_pdl(mcb::page_fork_plan_kernel,
                             dim3(1 + std::min(blocks, static_cast<unsigned>(sms))), dim3(1024), 0, st, p);
  if (e == cudaSuccess) e = launch_pdl(mcb::page_fork_apply_kernel, dim3(static_cast<unsigned>(8 * sms)), dim3(256), 0, st, p);
  // one CTA counts a pool of up to 32 blocks as it places the pages, a launch (3 us) for some 0.3 us a block
  const bool one = blocks <= 32;
  if (e == cudaSuccess && !one) e = launch_pdl(mcb::page_fork_count_kernel, dim3(blocks), dim3(mcb::kForkBlock), 0, st, p);
  if (e == cudaSuccess)
    e = launch_pdl(mcb::page_fork_place_kernel, dim3(one ? 1u : blocks), dim3(mcb::kForkBlock), 0, st, p);
  g_launches += one ? 3 : 4;
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "page_fork launch");
  return MCB_OK;
}

}  // namespace

extern "C" {

int mcb_draft_tree(const mcb_draft_tree_args* a, void* stream) {
  return guarded("mcb_draft_tree", [&] { return draft_tree(a, stream); });
}
size_t mcb_paged_tree_attn_workspace_size(const mcb_paged_tree_attn_args* a) {
  size_t n = 0;
  guarded("mcb_paged_tree_attn_workspace_size", [&] {
    const int rc = check_paged_tree(a, "mcb_paged_tree_attn_workspace_size");
    if (rc == MCB_OK) n = plan_paged_tree(a).ws_bytes;
    return rc;
  });
  return n;
}
size_t mcb_paged_tree_attn_counter_count(const mcb_paged_tree_attn_args* a) {
  size_t n = 0;
  guarded("mcb_paged_tree_attn_counter_count", [&] {
    const int rc = check_paged_tree(a, "mcb_paged_tree_attn_counter_count");
    if (rc == MCB_OK) n = plan_paged_tree(a).counters;
    return rc;
  });
  return n;
}
int mcb_paged_tree_attn(const mcb_paged_tree_attn_args* a, void* stream) {
  return guarded("mcb_paged_tree_attn", [&] { return paged_tree_attn(a, stream); });
}
int mcb_verify_drafts(const mcb_verify_drafts_args* a, void* stream) {
  return guarded("mcb_verify_drafts", [&] { return verify_drafts(a, stream); });
}
int mcb_paged_keep(const mcb_paged_keep_args* a, void* stream) {
  return guarded("mcb_paged_keep", [&] { return paged_keep(a, stream); });
}
size_t mcb_page_fork_workspace_size(const mcb_page_fork_args* a) {
  size_t n = 0;
  guarded("mcb_page_fork_workspace_size", [&] {
    if (a == nullptr) return fail(MCB_ERR_INVALID_ARG, "mcb_page_fork_workspace_size: args is NULL");
    const int rc = check_slots(a, "mcb_page_fork_workspace_size");
    if (rc == MCB_OK) n = fork_layout(a).bytes;
    return rc;
  });
  return n;
}
int mcb_page_fork(const mcb_page_fork_args* a, void* stream) {
  return guarded("mcb_page_fork", [&] { return page_fork(a, stream); });
}

}  // extern "C"
