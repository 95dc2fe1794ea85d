// Entry point of the attention over a cache: checks, the choice of kernel and the workspace.
#include "attention_dev.cuh"
#include <math.h>

namespace hbq {

namespace {

int check(const hbq_attention* p)
{
    if (!p || p->B < 0 || p->L < 0 || p->H < 0 || p->S < 0 || p->P < 0 || p->D <= 0 || p->Hkv <= 0 || p->sinks < 0) return HBQ_ERR_ARG;
    if (p->dtype != HBQ_DTYPE_F16 && p->dtype != HBQ_DTYPE_BF16) return HBQ_ERR_ARG;
    if (p->H % p->Hkv || !(p->scale > 0.f) || !isfinite(p->scale)) return HBQ_ERR_ARG;
    if (p->B == 0 || p->L == 0 || p->H == 0) return HBQ_OK;
    if (!p->q || !p->out || (p->S > 0 && (!p->k || !p->v)) || (p->P > 0 && (!p->prefix_k || !p->prefix_v))) return HBQ_ERR_ARG;
    if (p->D > 128 || (p->D % 8) || p->S > 0x7FFFFFFFll || p->P > 0x7FFFFFFFll || p->L > 0x7FFFFFFFll || p->B > 65535 || p->H > 65535 ||
        p->B * p->H > (1ll << 40) / p->L)
        return HBQ_ERR_UNSUPPORTED;
    int64_t s = 0;
    for (int i = 0; i < 3; ++i) s |= p->q_stride[i] | (p->S > 0 ? p->k_stride[i] | p->v_stride[i] : 0);
    for (int i = 0; i < 2 && p->P > 0; ++i) s |= p->pk_stride[i] | p->pv_stride[i];
    uintptr_t u = reinterpret_cast<uintptr_t>(p->q);
    if (p->S > 0) u |= reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v);
    if (p->P > 0) u |= reinterpret_cast<uintptr_t>(p->prefix_k) | reinterpret_cast<uintptr_t>(p->prefix_v);
    return (s % 8) || (u & 15) ? HBQ_ERR_ALIGN : HBQ_OK;
}

bool nothing(const hbq_attention* p) { return p->B == 0 || p->L == 0 || p->H == 0; }

int64_t part_bytes(const hbq_attention* p, int64_t parts) { return parts > 1 ? p->B * p->L * p->H * parts * (p->D + 2) * 4 : 0; }

}  // namespace

int64_t attention_workspace_bytes(const hbq_attention* p)
{
    if (check(p) || nothing(p)) return 0;
    int nsplit;
    return part_bytes(p, attention_rows_parts(p, &nsplit));
}

int attention_run(const hbq_attention* p, void* workspace, int64_t workspace_bytes, cudaStream_t stream)
{
    { const int rc = check(p); if (rc || nothing(p)) return rc; }
    AttnArgs a = {};
    a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out; a.pk = p->prefix_k; a.pv = p->prefix_v;
    a.lengths = p->lengths; a.starts = p->starts;
    for (int i = 0; i < 3; ++i) { a.qs[i] = p->q_stride[i]; a.ks[i] = p->k_stride[i]; a.vs[i] = p->v_stride[i]; a.os[i] = p->out_stride[i]; }
    for (int i = 0; i < 2; ++i) { a.pks[i] = p->pk_stride[i]; a.pvs[i] = p->pv_stride[i]; }
    a.S = p->S; a.P = p->P; a.window = p->window; a.sinks = p->sinks;
    a.B = (uint32_t)p->B; a.L = (uint32_t)p->L; a.H = (uint32_t)p->H; a.Hkv = (uint32_t)p->Hkv; a.G = (uint32_t)(p->H / p->Hkv); a.D = (uint32_t)p->D;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.parts = (int)attention_rows_parts(p, &a.nsplit);
    const int64_t need = part_bytes(p, a.parts);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))) return HBQ_ERR_WORKSPACE;
    a.part = static_cast<float*>(workspace);
    { const int rc = attention_rows_launch(a, p->dtype, stream); if (rc) return rc; }
    return a.parts > 1 ? attention_join_launch(a, p->dtype, stream) : HBQ_OK;
}

}  // namespace hbq
