// The plan of a pa_decode_tree call, without a GPU: the entry point's own source over launches that only say what they were given, a JSON object a line.
//   tree_plan N_HEADS N_KV_HEADS HEAD_DIM F16 MAX_COLS RECORDS ROWS.TOKENS ...
// F16: activations and queries; RECORDS: of the partial buffers (0: as many as the context has).
#include "../pooled_b200/csrc/pa_tree_api.cu"

#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

namespace pa {
int fail(pa_ctx*, int code, const char* fmt, ...) {
  va_list a;
  va_start(a, fmt);
  vfprintf(stderr, fmt, a);
  va_end(a);
  return code;
}
cudaError_t launch_tree(const TreeParams& p, bool wide, const CUtensorMap&, const CUtensorMap&, uint32_t, uint32_t, int, cudaStream_t) {
  printf("{\"wide\": %d, \"items\": %u, \"units\": %u, \"tiles\": %u, \"run\": %u, \"fold\": %u}\n", wide, p.n_items, p.units, p.tps, p.seg, p.fold);
  return cudaSuccess;
}
cudaError_t launch_tree_finish(const TreeFinishParams&, uint32_t, cudaStream_t) { return cudaSuccess; }
}  // namespace pa

int main(int argc, char** argv) {
  if (argc < 7) return 2;
  pa_ctx ctx;
  pa_layer layer;
  ctx.cfg.n_heads = atoi(argv[1]); ctx.cfg.n_kv_heads = atoi(argv[2]); ctx.cfg.head_dim = atoi(argv[3]);
  ctx.cfg.act_dtype = atoi(argv[4]) ? PA_F16 : PA_F32; ctx.cfg.max_cols = atoi(argv[5]);
  ctx.G = ctx.cfg.n_heads / ctx.cfg.n_kv_heads; ctx.q_dim = ctx.cfg.n_heads * ctx.cfg.head_dim; ctx.kv_dim = ctx.cfg.n_kv_heads * ctx.cfg.head_dim;
  size_records(&ctx);
  printf("{\"part\": %zu, \"prefill\": %zu, \"tree\": %zu}\n", ctx.part_slots, ctx.pf_slots, ctx.tree_slots);
  if (atoi(argv[6])) ctx.tree_slots = atoi(argv[6]);
  pa_item items[kMaxTrees] = {};
  uint32_t n = 0, most = 0;
  for (int i = 7; i < argc && n < (uint32_t)kMaxTrees; ++i, ++n) {
    if (sscanf(argv[i], "%u.%u", &items[n].pos, &items[n].n_cols) != 2) return 2;
    items[n].seq = n;
    most = std::max(most, items[n].pos + items[n].n_cols);
  }
  layer.ctx = &ctx; layer.n_seqs = n; layer.max_seq = most;
  void* some = &ctx;
  return n ? -pa_decode_tree(&layer, items, n, nullptr, (void*)((uintptr_t)some & ~(uintptr_t)15), ctx.cfg.act_dtype, ctx.q_dim, ctx.cfg.head_dim, nullptr, 0, 0, some,
                             ctx.q_dim, nullptr) : 0;
}
