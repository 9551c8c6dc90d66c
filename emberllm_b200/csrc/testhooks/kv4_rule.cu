// kv4_rule.cu — TEST HOOK, built into libember_testhooks.so only: the attention's choice
// of a kernel, so that tests can check which one their sizes reach.
#include "cuda/kv4_rule.h"
#include "ember_testhooks.h"

extern "C" int ember_testhook_kv4_kernel(int elem_bytes, int head_dim, int n_tokens, int max_q, int group, int n_kv,
                                         int n_seqs) {
    return emb::kv4_kernel(elem_bytes, head_dim, n_tokens, max_q, group, n_kv, n_seqs);
}
