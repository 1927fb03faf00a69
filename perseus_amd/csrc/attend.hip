// pcx_attention: keys and values packed or in caches, a run of rows for each sequence (the kernels: attend.h).
#include "attend.h"

using namespace pch;
using namespace pch::clear;

extern "C" uint64_t pcx_attention_workspace(const AttentionArgs* args) {
    AttentionArgs a;
    if (checked(args, &a) || !a.tokens || !a.seqs || !a.heads) return 0;
    return work_bytes(a, choose(a));
}

extern "C" int pcx_attention(const AttentionArgs* args, pc_stream_t s) {
    AttentionArgs a;
    if (int e = checked(args, &a)) return e;
    if ((uintptr_t)a.work % 16) return -2;
    if (!a.tokens || !a.seqs || !a.heads) return 0;
    return a.type == PCX_BF16 ? run<bf16, false>(a, {}, (hipStream_t)s) : run<f16, false>(a, {}, (hipStream_t)s);
}
