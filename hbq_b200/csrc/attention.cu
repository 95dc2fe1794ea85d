// Entry point of the attention over a cache: checks, the choice of kernel and the workspace.
#include "attention_dev.cuh"
#include <math.h>

namespace hbq {

namespace {

int check(const hbq_attention* p)
{
    if (!p || p->B < 0 || p->L < 0 || p->H < 0 || p->S < 0 || p->P < 0 || p->D <= 0 || p->Hkv <= 0 || p->sinks < 0) return HBQ_ERR_ARG;
    if (p->dtype != HBQ_DTYPE_F16 && p->dtype != HBQ_DTYPE_BF16) return HBQ_ERR_ARG;
    if (p->H % p->Hkv || !(p->scale > 0.f) || !isfinite(p->scale * 1.4426950408889634f)) return HBQ_ERR_ARG;
    if (p->B == 0 || p->L == 0 || p->H == 0) return HBQ_OK;
    if (!p->q || !p->out || (p->S > 0 && (!p->k || !p->v)) || (p->P > 0 && (!p->prefix_k || !p->prefix_v))) return HBQ_ERR_ARG;
    // (key positions are ints in the kernels, and a tile may end up to 127 behind the last key)
    if (p->D > 128 || (p->D % 8) || p->S > 0x7FFFFF00ll || p->P > 0x7FFFFF00ll || p->L > 0x7FFFFFFFll || p->B > 65535 || p->H > 65535 ||
        p->B * p->H > (1ll << 40) / p->L)
        return HBQ_ERR_UNSUPPORTED;
    int64_t s = 0;
    for (int i = 0; i < 3; ++i) s |= p->q_stride[i] | (p->S > 0 ? p->k_stride[i] | p->v_stride[i] : 0);
    for (int i = 0; i < 2 && p->P > 0; ++i) s |= p->pk_stride[i] | p->pv_stride[i];
    uintptr_t u = reinterpret_cast<uintptr_t>(p->q);
    if (p->S > 0) u |= reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v);
    if (p->P > 0) u |= reinterpret_cast<uintptr_t>(p->prefix_k) | reinterpret_cast<uintptr_t>(p->prefix_v);
    const bool same_keys = (p->S > 1 && (p->k_stride[2] <= 0 || p->v_stride[2] <= 0)) || (p->P > 1 && (p->pk_stride[1] <= 0 || p->pv_stride[1] <= 0));
    // (the copies' maps take an axis without a positive stride for one element repeated, of a cache, or a dense one, of the output)
    bool down = false;
    for (int i = 0; i < 2; ++i) {
        down |= p->S > 0 && (i ? p->Hkv : p->B) > 1 && (p->k_stride[i] < 0 || p->v_stride[i] < 0);
        down |= p->P > 0 && (i ? p->P : p->Hkv) > 1 && (p->pk_stride[i] < 0 || p->pv_stride[i] < 0);
    }
    const int64_t outs[3] = {p->B, p->L, p->H};
    for (int i = 0; i < 3; ++i) down |= outs[i] > 1 && p->out_stride[i] <= 0;
    return (s % 8) || (u & 15) || same_keys || down ? HBQ_ERR_ALIGN : HBQ_OK;
}

bool nothing(const hbq_attention* p) { return p->B == 0 || p->L == 0 || p->H == 0; }

// Which kernels a call takes.  The few-row kernel, on the warp-level MMA, reads a token's keys for that token alone; the
// tensor-core kernel reads them once for 256 rows, but takes 7 us and more whatever it does.
//  * One token a sequence: the few-row kernel.  More tokens: the tensor-core kernel, unless all row groups are resident in the
//    few-row kernel at once with few keys each ("small" there).  us, few-row and tensor-core, 32 / 8 heads of 128:
//    1 x 4 tokens of 2048 keys 12.5 and 15.6, 1 x 16 30 and 16, 8 x 2 of 8192 97 and 64, 32 x 2 of 1024 50 and 39.
//  * A prefix: the tensor-core kernel for all sequences at once and a kernel for their own keys, unless the call is small, or there
//    is one token to share it: then the prefix is the beginning of the few-row kernel's lists.  us, in the lists and by itself: prefix of
//    1024, 4 sequences 10.5 and 24, 8 12 and 19, 16 23 and 19; of 16384, 2 sequences 27.5 and 29, 4 39 and 31.
struct Plan {
    bool own_tc, prefix_tc;            // prefix_tc: the prefix has a launch of its own, else it is part of the rows' list
    int prefix, own;                   // the tensor-core kernel's pieces
    int blocks, shared, cluster;       // the few-row kernel's blocks (0: not launched)
    int parts;                         // entries of a row's list of parts; 0: every row is written by one block
    int64_t part_bytes, table_bytes, slot_bytes;
    int64_t bytes() const { return part_bytes + table_bytes + slot_bytes; }
    bool join() const { return parts > 0 || shared; }
};
Plan plan_of(const hbq_attention* p)
{
    Plan c = {};
    bool small;
    const int together = attention_rows_blocks(p, true, &c.shared, &c.cluster, &small);
    c.prefix_tc = p->P > 0 && !small && p->B * p->L > 1;
    if (p->P > 0 && !c.prefix_tc) c.blocks = together;
    else if (p->S > 0 || !c.prefix_tc) {
        c.blocks = attention_rows_blocks(p, false, &c.shared, &c.cluster, &small);
        c.own_tc = p->L > 1 && p->S > 0 && !small;
    }
    if (c.own_tc || (c.prefix_tc && p->S == 0)) c.blocks = c.shared = 0;
    if (c.prefix_tc) c.prefix = attention_tc_parts(p, true);
    if (c.own_tc) c.own = attention_tc_parts(p, false);
    c.parts = c.prefix + c.own + (c.prefix_tc && c.blocks ? 1 : 0);
    if (c.parts == 1) c.parts = 0;
    const auto up = [](int64_t n) { return (n + 31) / 32 * 32; };
    c.part_bytes = up(p->B * p->L * p->H * c.parts * (p->D + 2) * 4);
    if (c.shared) {
        c.table_bytes = up(p->B * p->L * p->Hkv * ((p->H / p->Hkv + 15) / 16) * 8);
        c.slot_bytes = up((int64_t)c.blocks * 2 * 16 * (p->D + 2) * 4);
    }
    return c;
}

// Windows and first tokens beyond the cache mean the whole of it (and their sums stay far from 64 bits' end).
hbq_attention bounded(const hbq_attention* p)
{
    hbq_attention c = *p;
    if (c.window >= c.S || c.window < 0) c.window = 0;
    if (c.sinks > c.S) c.sinks = c.S;
    return c;
}

}  // namespace

int64_t attention_workspace_bytes(const hbq_attention* call)
{
    if (check(call) || nothing(call)) return 0;
    const hbq_attention c = bounded(call);
    return plan_of(&c).bytes();
}

int attention_run(const hbq_attention* call, void* workspace, int64_t workspace_bytes, cudaStream_t stream)
{
    { const int rc = check(call); if (rc || nothing(call)) return rc; }
    const hbq_attention bound = bounded(call), *p = &bound;
    AttnArgs a = {};
    a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.pk = p->prefix_k; a.pv = p->prefix_v;
    a.lengths = p->lengths; a.starts = p->starts;
    for (int i = 0; i < 3; ++i) { a.qs[i] = p->q_stride[i]; a.ks[i] = p->k_stride[i]; a.vs[i] = p->v_stride[i]; a.os[i] = p->out_stride[i]; }
    for (int i = 0; i < 2; ++i) { a.pks[i] = p->pk_stride[i]; a.pvs[i] = p->pv_stride[i]; }
    a.S = p->S; a.P = p->P; a.window = p->window; a.sinks = p->sinks;
    a.B = (uint32_t)p->B; a.L = (uint32_t)p->L; a.H = (uint32_t)p->H; a.Hkv = (uint32_t)p->Hkv; a.G = (uint32_t)(p->H / p->Hkv); a.D = (uint32_t)p->D;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    const Plan c = plan_of(p);
    if (c.blocks < 0) return HBQ_ERR_UNSUPPORTED;
    const int64_t need = c.bytes();
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 31))) return HBQ_ERR_WORKSPACE;
    a.parts = c.parts; a.blocks = c.blocks; a.shared = c.shared; a.cluster = c.cluster;
    char* ws = static_cast<char*>(workspace);
    a.part = reinterpret_cast<float*>(ws);
    a.table = reinterpret_cast<int2*>(ws + c.part_bytes);
    a.slots = reinterpret_cast<float*>(ws + c.part_bytes + c.table_bytes);
    if (c.prefix_tc) {
        a.nsplit = c.prefix;
        { const int rc = attention_tc_launch(a, p->dtype, true, stream); if (rc) return rc; }
        a.P = 0;
        a.part0 = c.prefix;
        a.beside = 1;
    }
    if (c.own_tc) {
        a.nsplit = c.own;
        const int rc = attention_tc_launch(a, p->dtype, false, stream);
        if (rc) return rc;
    } else if (c.blocks) {
        const int rc = attention_rows_launch(a, p->dtype, stream);
        if (rc) return rc;
    }
    return c.join() ? attention_join_launch(a, p->dtype, stream) : HBQ_OK;
}

}  // namespace hbq
