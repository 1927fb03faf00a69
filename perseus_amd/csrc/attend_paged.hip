// pcx_attention_paged: keys and values in pages of a pool (the kernels: attend.h).
#include "attend.h"

using namespace pch;
using namespace pch::clear;

// 0, the arguments with their strides settled and the pages, or the error
static int checked_paged(const AttentionPagedArgs* given, AttentionArgs* a, PagesRef* p) {
    if (!given) return -1;
    if (int e = checked(&given->attention, a, true)) return e;
    if (given->cache.start) return -1;
    if (int e = pages_of(given->cache, a->seqs, a->kv_rows, p)) return e;
    return (a->k.token << p->log) > PAGE_MAX || (a->v.token << p->log) > PAGE_MAX ? -2 : 0;
}

extern "C" uint64_t pcx_attention_paged_workspace(const AttentionPagedArgs* args) {
    AttentionArgs a;
    PagesRef p;
    if (checked_paged(args, &a, &p) || !a.tokens || !a.seqs || !a.heads) return 0;
    return work_bytes(a, choose(a));
}

extern "C" int pcx_attention_paged(const AttentionPagedArgs* args, pc_stream_t s) {
    AttentionArgs a;
    PagesRef p;
    if (int e = checked_paged(args, &a, &p)) return e;
    if ((uintptr_t)a.work % 16) return -2;
    if (!a.tokens || !a.seqs || !a.heads) return 0;
    return a.type == PCX_BF16 ? run<bf16, true>(a, p, (hipStream_t)s) : run<f16, true>(a, p, (hipStream_t)s);
}
