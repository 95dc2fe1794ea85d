// Attention of few rows against a cache: the query heads that share a key head, for one token, on the warp-level MMA.
//
// For a row at position p the visible keys are the prefix, the first `sinks` ones and those behind p - window: a list
// u = 0 .. U - 1 whose entries map to rows of the cache.  Every lane loads list entries, so nothing that the mask hides is
// read at all, and entries behind the list's end are zeros.  Bound by memory: keys and values are read once for up to 16
// heads; one MMA tile is 16 rows by 8 keys, most of them empty for four heads, at a cost far below the memory's.
//
// Each warp has a ring of its own (16 keys and values a stage, asynchronous copies), a maximum, a weight and a sum of its
// own; no barrier until the warps' sums are joined at the end.  With few sequences the list is cut over several blocks,
// whose parts (sum, maximum, weight) a second kernel joins.
#include "attention_dev.cuh"

namespace hbq {

namespace {

constexpr int RW = 4, STAGES = 3, GROUP = 16;      // warps, stages a warp, keys a stage

template <class E> struct Mma;
template <> struct Mma<__half> {
    static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) { return h2_bits(__floats2half2_rn(x, y)); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(bits_h2(u)); }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) { static_cast<__half*>(p)[i] = __float2half_rn(v); }
};
template <> struct Mma<__nv_bfloat16> {
    static __device__ __forceinline__ void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y)
    {
        __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
    static __device__ __forceinline__ void store(void* p, int64_t i, float v) { static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v); }
};

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <int NK> struct RowsShape {
    static constexpr int DP = NK * 16;                       // head length, rounded up
    static constexpr int ROW = DP * 2 + 16;                  // bytes of a staged row: an odd number of 16-byte pieces, so that
                                                             // the eight rows of an 8 x 8 matrix lie in different banks
    static constexpr int STAGE = 2 * GROUP * ROW;
    static constexpr int RING = RW * STAGES * STAGE;
    static constexpr int JOIN = RW * 16 * (DP + 2) * 4;
    static constexpr int BYTES = RING > JOIN ? RING : JOIN;
};

template <class E, int NK>
__global__ void __launch_bounds__(RW * 32) attention_rows_kernel(const __grid_constant__ AttnArgs a, uint32_t tiles)
{
    using Sh = RowsShape<NK>;
    extern __shared__ __align__(16) uint8_t smem[];
    grid_dependency_wait();
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t id = blockIdx.x;
    const uint32_t split = id % (uint32_t)a.nsplit; id /= (uint32_t)a.nsplit;
    const uint32_t tile = id % tiles; id /= tiles;
    const uint32_t hk = id % a.Hkv; id /= a.Hkv;
    const uint32_t i = id % a.L, b = id / a.L;
    const uint32_t g0 = tile * 16, rows = min(16u, a.G - g0), h0 = hk * a.G + g0;

    // the list of visible keys, and this block's piece of it
    int64_t n, p;
    sequence_of(a, b, &n, &p);
    p += i;
    int64_t lo = 0, ns = 0, U = 0;
    if (p < n) {
        U = a.P;
        if (p >= 0) {
            lo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
            ns = a.sinks < lo ? a.sinks : lo;
            U += ns + (p + 1 - lo);
        }
    }
    const int64_t piece = ((U + a.nsplit - 1) / a.nsplit + RW * GROUP - 1) / (RW * GROUP) * (RW * GROUP);
    const int64_t u0 = (int64_t)split * piece, u1 = U < u0 + piece ? U : u0 + piece;

    const E* kb = static_cast<const E*>(a.k) + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[1];
    const E* vb = static_cast<const E*>(a.v) + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[1];
    const E* pk = static_cast<const E*>(a.pk) + (int64_t)hk * a.pks[0];
    const E* pv = static_cast<const E*>(a.pv) + (int64_t)hk * a.pvs[0];
    const uint32_t ring = smem_of(smem) + warp * (STAGES * Sh::STAGE);

    // queries as the left operand's fragments: rows lane / 4 and lane / 4 + 8
    uint32_t qf[NK][4];
    #pragma unroll
    for (int kk = 0; kk < NK; ++kk)
        #pragma unroll
        for (int f = 0; f < 4; ++f) {
            const uint32_t r = lane / 4 + 8 * (f & 1), d = kk * 16 + (lane & 3) * 2 + 8 * (f >> 1);
            qf[kk][f] = r < rows && d < a.D
                ? *reinterpret_cast<const uint32_t*>(static_cast<const E*>(a.q) + (int64_t)b * a.qs[0] + (int64_t)i * a.qs[1] + (int64_t)(h0 + r) * a.qs[2] + d) : 0u;
        }

    auto load = [&](int64_t u, int stage) {
        // a row of 2 NK pieces of 16 bytes, neighbouring lanes along a row: whole lines from memory
        const uint32_t dst = ring + stage * Sh::STAGE;
        #pragma unroll
        for (int c = 0; c < NK; ++c) {
            const int x = lane + 32 * c, key = x / (2 * NK), d = (x - key * (2 * NK)) * 8;
            const int64_t y = u + key;
            const E *kp = kb, *vp = vb;
            const bool live = y < u1 && (uint32_t)d < a.D;
            if (live) {
                if (y < a.P) { kp = pk + y * a.pks[1] + d; vp = pv + y * a.pvs[1] + d; }
                else {
                    const int64_t z = y - a.P, j = z < ns ? z : lo + (z - ns);
                    kp = kb + j * a.ks[2] + d; vp = vb + j * a.vs[2] + d;
                }
            }
            copy16(dst + key * Sh::ROW + d * 2, kp, live);
            copy16(dst + (GROUP + key) * Sh::ROW + d * 2, vp, live);
        }
    };

    float o[NK * 2][4];
    #pragma unroll
    for (int t = 0; t < NK * 2; ++t)
        #pragma unroll
        for (int f = 0; f < 4; ++f) o[t][f] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    constexpr int64_t STEP = RW * GROUP;
    const int64_t first = u0 + warp * GROUP;
    #pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        if (first + s * STEP < u1) load(first + s * STEP, s);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int stage = 0;
    for (int64_t u = first; u < u1; u += STEP) {
        {
            const int64_t next = u + (STAGES - 1) * STEP;
            int s = stage + STAGES - 1;
            if (s >= STAGES) s -= STAGES;
            if (next < u1) load(next, s);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        const uint32_t kt = ring + stage * Sh::STAGE, vt = kt + GROUP * Sh::ROW;
        float s[2][4] = {};
        #pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
            uint32_t f[4];
            ldsm4(f, kt + ((lane & 7) + 8 * (lane >> 4)) * Sh::ROW + kk * 32 + ((lane >> 3) & 1) * 16);
            Mma<E>::run(s[0], qf[kk], f[0], f[1]);
            Mma<E>::run(s[1], qf[kk], f[2], f[3]);
        }
        uint32_t hi[4], rest[4];
        #pragma unroll
        for (int r = 0; r < 2; ++r) {                  // row lane / 4 + 8 r
            float x[4], top = -INFINITY;
            #pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t key = u + (e >> 1) * 8 + (lane & 3) * 2 + (e & 1);
                x[e] = key < u1 ? s[e >> 1][2 * r + (e & 1)] * a.scale_log2 : -INFINITY;
                top = fmaxf(top, x[e]);
            }
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const float now = fmaxf(m[r], top), ref = now == -INFINITY ? 0.f : now, old = exp2_fast(m[r] - ref);
            m[r] = now;
            float w[4], sum = 0.f;
            #pragma unroll
            for (int e = 0; e < 4; ++e) { w[e] = exp2_fast(x[e] - ref); sum += w[e]; }
            l[r] = l[r] * old + sum;
            #pragma unroll
            for (int t = 0; t < NK * 2; ++t) { o[t][2 * r] *= old; o[t][2 * r + 1] *= old; }
            // the weights as two numbers of the values' type, so that their rounding does not reach the result
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t top2 = Mma<E>::pack(w[2 * e], w[2 * e + 1]);
                const float2 back = Mma<E>::unpack(top2);
                hi[2 * e + r] = top2;
                rest[2 * e + r] = Mma<E>::pack(w[2 * e] - back.x, w[2 * e + 1] - back.y);
            }
        }
        #pragma unroll
        for (int t = 0; t < NK; ++t) {
            uint32_t f[4];
            ldsm4t(f, vt + ((lane & 7) + 8 * ((lane >> 3) & 1)) * Sh::ROW + t * 32 + (lane >> 4) * 16);
            Mma<E>::run(o[2 * t], hi, f[0], f[1]);
            Mma<E>::run(o[2 * t], rest, f[0], f[1]);
            Mma<E>::run(o[2 * t + 1], hi, f[2], f[3]);
            Mma<E>::run(o[2 * t + 1], rest, f[2], f[3]);
        }
        __syncwarp();                                  // the stage is refilled by the copies of the next round
        if (++stage == STAGES) stage = 0;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    #pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
        l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
    }

    // join the warps: [warp][16][DP] sums, then [warp][16] maxima and weights
    __syncthreads();
    float* js = reinterpret_cast<float*>(smem);
    float* jm = js + RW * 16 * Sh::DP;
    #pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = lane / 4 + 8 * r;
        #pragma unroll
        for (int t = 0; t < NK * 2; ++t)
            *reinterpret_cast<float2*>(js + (warp * 16 + row) * Sh::DP + t * 8 + (lane & 3) * 2) = make_float2(o[t][2 * r], o[t][2 * r + 1]);
        if ((lane & 3) == 0) { jm[(warp * 16 + row) * 2] = m[r]; jm[(warp * 16 + row) * 2 + 1] = l[r]; }
    }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < rows * a.D; x += RW * 32) {
        const uint32_t row = x / a.D, d = x - row * a.D;
        float top = -INFINITY, sum = 0.f, weight = 0.f;
        #pragma unroll
        for (int w = 0; w < RW; ++w) top = fmaxf(top, jm[(w * 16 + row) * 2]);
        const float ref = top == -INFINITY ? 0.f : top;
        #pragma unroll
        for (int w = 0; w < RW; ++w) {
            const float f = exp2_fast(jm[(w * 16 + row) * 2] - ref);
            sum = fmaf(js[(w * 16 + row) * Sh::DP + d], f, sum);
            weight = fmaf(jm[(w * 16 + row) * 2 + 1], f, weight);
        }
        if (a.parts > 1) {
            const int64_t at = ((int64_t)b * a.L + i) * a.H + h0 + row;
            part_sum(a, at, a.part0 + split)[d] = sum;
            if (d == 0) *part_weight(a, at, a.part0 + split) = make_float2(top, weight);
        } else {
            Mma<E>::store(a.out, (int64_t)b * a.os[0] + (int64_t)i * a.os[1] + (int64_t)(h0 + row) * a.os[2] + d, weight == 0.f ? 0.f : sum / weight);
        }
    }
}

// One warp joins a row's parts: maxima, then weights and sums relative to the largest.
template <class E>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ AttnArgs a)
{
    grid_dependency_wait();
    dependents_may_start();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.B * a.L * a.H) return;
    const float2* w = part_weight(a, row, 0);
    float top = -INFINITY;
    for (int s = lane; s < a.parts; s += 32) top = fmaxf(top, w[s].x);
    #pragma unroll
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
    const float ref = top == -INFINITY ? 0.f : top;
    float weight = 0.f, sum[4] = {};
    for (int s = 0; s < a.parts; ++s) {
        const float2 ml = w[s];
        if (ml.y == 0.f) continue;                       // an empty part's sums are not looked at
        const float f = exp2_fast(ml.x - ref);
        weight = fmaf(ml.y, f, weight);
        const float* x = part_sum(a, row, s);
        #pragma unroll
        for (int e = 0; e < 4; ++e)
            if (lane + 32 * e < (int)a.D) sum[e] = fmaf(x[lane + 32 * e], f, sum[e]);
    }
    const int64_t h = row % a.H, bl = row / a.H, i = bl % a.L, b = bl / a.L;
    #pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < (int)a.D)
            Mma<E>::store(a.out, b * a.os[0] + i * a.os[1] + h * a.os[2] + lane + 32 * e, weight == 0.f ? 0.f : sum[e] / weight);
}

template <class E, int NK>
int rows_launch(const AttnArgs& a, cudaStream_t stream)
{
    const uint32_t tiles = (a.G + 15) / 16;
    const int64_t blocks = (int64_t)a.B * a.L * a.Hkv * tiles * a.nsplit;
    if (blocks > 0x7FFFFFFFll) return HBQ_ERR_UNSUPPORTED;
    { const int rc = ensure_dynamic_smem(attention_rows_kernel<E, NK>, RowsShape<NK>::BYTES); if (rc) return rc; }
    HBQ_CUDA_TRY(launch_dependent(attention_rows_kernel<E, NK>, (unsigned)blocks, RW * 32, (size_t)RowsShape<NK>::BYTES, stream, a, tiles));
    HBQ_LAUNCH_CHECK("attention_rows_kernel");
    return HBQ_OK;
}

template <class E>
int rows_type(const AttnArgs& a, cudaStream_t stream)
{
    switch ((a.D + 15) / 16) {
        case 1: case 2: case 3: case 4: return rows_launch<E, 4>(a, stream);
        case 5: return rows_launch<E, 5>(a, stream);
        case 6: return rows_launch<E, 6>(a, stream);
        case 7: return rows_launch<E, 7>(a, stream);
        default: return rows_launch<E, 8>(a, stream);
    }
}

}  // namespace

// Into how many pieces a row's list of keys is cut; prefix: the list begins with it.
int attention_rows_parts(const hbq_attention* p, bool prefix)
{
    int sms = 148;
    device_sms(&sms);
    const int64_t blocks = p->B * p->L * p->Hkv * ((p->H / p->Hkv + 15) / 16);
    int64_t keys = p->S;
    if (p->window > 0 && p->window + p->sinks < keys) keys = p->window + p->sinks;
    if (prefix) keys += p->P;
    // two blocks an SM are resident; twice as many pieces as that even out sequences of different lengths, as far as a
    // piece keeps 128 keys
    int64_t n = ((int64_t)sms * 4 + blocks - 1) / blocks;
    if (n > (keys + 127) / 128) n = (keys + 127) / 128;
    return (int)(n < 1 ? 1 : n > 256 ? 256 : n);
}

int attention_rows_launch(AttnArgs& a, int dtype, cudaStream_t stream)
{
    return dtype == HBQ_DTYPE_F16 ? rows_type<__half>(a, stream) : rows_type<__nv_bfloat16>(a, stream);
}

int attention_join_launch(const AttnArgs& a, int dtype, cudaStream_t stream)
{
    const int64_t blocks = ((int64_t)a.B * a.L * a.H + 7) / 8;
    if (blocks > 0x7FFFFFFFll) return HBQ_ERR_UNSUPPORTED;
    if (dtype == HBQ_DTYPE_F16) HBQ_CUDA_TRY(launch_dependent(attention_join_kernel<__half>, (unsigned)blocks, 256, 0, stream, a));
    else HBQ_CUDA_TRY(launch_dependent(attention_join_kernel<__nv_bfloat16>, (unsigned)blocks, 256, 0, stream, a));
    HBQ_LAUNCH_CHECK("attention_join_kernel");
    return HBQ_OK;
}

}  // namespace hbq
