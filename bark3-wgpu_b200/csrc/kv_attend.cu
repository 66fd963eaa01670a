// kv_attend.cu — b3_kv_attend: checks, and the choice between the kernel for
// few query rows (kv_attend_rows.cu, bound by memory) and the one for many
// (kv_attend_tiles.cu, bound by arithmetic).
#include "kv_attend.cuh"

using namespace b3;

namespace {

int check(const b3_kv_cache* cache, const b3_kv_batch* batch, const b3_kv_attend_args* args) {
    if (int rc = kv_check(cache, batch)) return rc;
    if (!args) return set_error(B3_EINVAL, "null arguments");
    const b3_kv_attend_args& a = *args;
    if (a.dtype != B3_DTYPE_F16 && a.dtype != B3_DTYPE_BF16) return set_error(B3_EINVAL, "dtype %d (f16 or bf16)", a.dtype);
    if (a.q_heads <= 0 || a.q_heads % cache->kv_heads)
        return set_error(B3_EINVAL, "q_heads %d is no multiple of kv_heads %d", a.q_heads, cache->kv_heads);
    if (a.max_q <= 0) return set_error(B3_EINVAL, "max_q %d", a.max_q);
    if (a.window < 0 || (a.window && !a.causal)) return set_error(B3_EINVAL, "window %d (needs causal)", a.window);
    if (static_cast<int64_t>(batch->tokens) * a.q_heads > 0x7fffffffll)
        return set_error(B3_EINVAL, "%d tokens x %d heads are too many for one call", batch->tokens, a.q_heads);
    return 0;
}

// New tokens x heads of a group that share a key head's cached codes: one tile
// of the memory-bound kernel holds 16 (128 sequences of 16 to 7504 tokens, 8
// heads a group: 2 new tokens each 95 us there, 4 each 276 us in the other's
// tiles of 256 rows).  The longest sequence's new tokens decide for the call:
// 127 sequences of one token take 63 us and a prompt of 512 alone 35, both in
// one call 357; a program that mixes them makes two calls.
bool few_rows(const AttendParams& p) { return static_cast<int64_t>(p.a.max_q) * (p.a.q_heads / p.c.kv_heads) <= 16; }

int64_t workspace_of(const AttendParams& p) { return few_rows(p) ? attend_rows_workspace(p) : attend_tiles_workspace(p); }

}  // namespace

extern "C" int64_t b3_kv_attend_workspace(const b3_kv_cache* cache, const b3_kv_batch* batch,
                                          const b3_kv_attend_args* args) {
    if (int rc = check(cache, batch, args)) return rc;
    return workspace_of(AttendParams{*cache, *batch, *args});
}

extern "C" int b3_kv_attend(const b3_kv_cache* cache, const b3_kv_batch* batch, const b3_kv_attend_args* args,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check(cache, batch, args)) return rc;
    if (batch->tokens == 0) return 0;
    if (!args->q || !args->out) return set_error(B3_EINVAL, "null q or out");
    if (reinterpret_cast<uintptr_t>(args->out) & 15) return set_error(B3_EINVAL, "out must be 16-byte aligned");
    const AttendParams p{*cache, *batch, *args};
    const int64_t need = workspace_of(p);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return set_error(B3_EINVAL, "a workspace of %lld bytes, 16-byte aligned, is needed (got %lld)",
                         static_cast<long long>(need), static_cast<long long>(workspace_bytes));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return few_rows(p) ? launch_attend_rows(p, workspace, st) : launch_attend_tiles(p, workspace, st);
}
