// Attention of few rows against a cache: the query heads that share a key head, for one token, on the warp-level MMA.
//
// For a row at position p the visible keys are the prefix, the first `sinks` ones and those behind p - window: a list
// u = 0 .. U - 1 whose entries map to rows of the cache.  Every lane loads list entries, so nothing that the mask hides is
// read at all, and entries behind the list's end are zeros.  Bound by memory: keys and values are read once for up to 16
// heads; one MMA tile is 16 rows by 8 keys, most of them empty for four heads, at a cost far below the memory's.
//
// Each warp has a ring of its own (16 keys and values a stage, asynchronous copies), a maximum, a weight and a sum of its
// own; no barrier until the warps' sums are joined at the end of a row group.
//
// The lengths are known on the device alone and may be as different as one key and a hundred thousand.  So the groups'
// units of 64 keys form one list over all sequences, of which every block (two an SM) takes an equal share; where a share
// begins or ends inside a group, its part (sum, maximum, weight) goes to a slot of the block and a second kernel joins.
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

// The keys of row (b, i): U entries -- the prefix, `ns` first keys, then those from lo on.
struct KeyList { int64_t U, lo, ns; };
__device__ __forceinline__ KeyList keys_of(const AttnArgs& a, uint32_t b, uint32_t i)
{
    int64_t n, p;
    sequence_of(a, b, &n, &p);
    p += i;
    KeyList k = {0, 0, 0};
    if (p < n) {
        k.U = a.P;
        if (p >= 0) {
            k.lo = a.window > 0 && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
            k.ns = a.sinks < k.lo ? a.sinks : k.lo;
            k.U += k.ns + (p + 1 - k.lo);
        }
    }
    return k;
}
// A group's units; one that sees nothing has one, in which its zeros are written.
__device__ __forceinline__ int64_t units_of(const KeyList& k) { return k.U > ROWS_UNIT ? (k.U + ROWS_UNIT - 1) / ROWS_UNIT : 1; }

// Units before each token, [0 .. tokens], by the whole block (tokens at most two a thread).
__device__ void count_units(const AttnArgs& a, int64_t* table)
{
    __shared__ int64_t warps[RW];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t tokens = a.B * a.L, r = 2 * threadIdx.x;
    int64_t c0 = 0, c1 = 0;
    if (r < tokens) c0 = units_of(keys_of(a, r / a.L, r % a.L));
    if (r + 1 < tokens) c1 = units_of(keys_of(a, (r + 1) / a.L, (r + 1) % a.L));
    int64_t sum = c0 + c1;
    #pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const int64_t below = __shfl_up_sync(0xFFFFFFFFu, sum, d);
        if (lane >= d) sum += below;
    }
    if (lane == 31) warps[warp] = sum;
    __syncthreads();
    int64_t before = sum - c0 - c1;
    for (int w = 0; w < warp; ++w) before += warps[w];
    if (r < tokens) { table[r] = before; table[r + 1] = before + c0; }
    if (r + 1 < tokens) table[r + 2] = before + c0 + c1;
    __syncthreads();
}

template <class E, int NK>
__global__ void __launch_bounds__(RW * 32) attention_rows_kernel(const __grid_constant__ AttnArgs a, uint32_t tiles)
{
    using Sh = RowsShape<NK>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int64_t table[RW * 64 + 1];
    grid_dependency_wait();
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t groups = a.Hkv * tiles, tokens = a.B * a.L;       // row groups of a token
    int64_t w0, w1;                                                  // this block's share of the units
    uint32_t token;
    if (a.shared) {
        count_units(a, table);
        if (blockIdx.x == 0)
            for (uint32_t r = threadIdx.x; r <= tokens; r += RW * 32) a.table[r] = table[r];
        const int64_t total = table[tokens] * groups;
        const int64_t takers = rows_takers(a, total);
        if (blockIdx.x >= takers) return;
        w0 = total * blockIdx.x / takers; w1 = total * (blockIdx.x + 1) / takers;
        uint32_t low = 0, high = tokens;                             // the last token that begins at or before w0
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if (table[mid] * groups <= w0) low = mid; else high = mid;
        }
        token = low;
    } else {
        token = blockIdx.x / groups;
        w0 = 0; w1 = 1;
    }
    while (w0 < w1) {
    const uint32_t b = token / a.L, i = token - b * a.L;
    const KeyList list = keys_of(a, b, i);
    const int64_t lo = list.lo, ns = list.ns, U = list.U;
    int64_t u0 = 0, u1 = U, take = 1;
    uint32_t g;
    int slot = -1;                                                   // -1: the whole group
    if (a.shared) {
        const int64_t units = table[token + 1] - table[token], in = w0 - table[token] * groups;
        g = (uint32_t)(in / units);
        const int64_t off = in - g * units;
        take = min(units - off, w1 - w0);
        u0 = off * ROWS_UNIT;
        if ((off + take) * ROWS_UNIT < U) u1 = (off + take) * ROWS_UNIT;
        slot = take == units ? -1 : off > 0 ? 0 : 1;
    } else g = blockIdx.x - token * groups;
    const uint32_t hk = g / tiles, g0 = (g - hk * tiles) * 16, rows = min(16u, a.G - g0), h0 = hk * a.G + g0;

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
        if (slot >= 0) {
            slot_sum(a, blockIdx.x, slot, row)[d] = sum;
            if (d == 0) *slot_weight(a, blockIdx.x, slot, row) = make_float2(top, weight);
        } else if (a.parts > 0) {
            const int64_t at = ((int64_t)b * a.L + i) * a.H + h0 + row;
            part_sum(a, at, a.part0)[d] = sum;
            if (d == 0) *part_weight(a, at, a.part0) = make_float2(top, weight);
        } else {
            Mma<E>::store(a.out, (int64_t)b * a.os[0] + (int64_t)i * a.os[1] + (int64_t)(h0 + row) * a.os[2] + d, weight == 0.f ? 0.f : sum / weight);
        }
    }
    w0 += take;
    if (a.shared && w0 < w1) {
        if (w0 >= table[token + 1] * groups) ++token;
        __syncthreads();                                             // the join's memory becomes the ring again
    }
    }
}

// One warp joins a row's parts: the tensor-core kernel's, and the few-row kernel's part or slots.  Maxima, then weights and
// sums relative to the largest.
template <class E>
__global__ void __launch_bounds__(64) attention_join_kernel(const __grid_constant__ AttnArgs a, uint32_t tiles)
{
    grid_dependency_wait();
    dependents_may_start();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 2 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.B * a.L * a.H) return;
    const int64_t token = row / a.H;
    const uint32_t h = (uint32_t)(row - token * a.H);
    int first = 0, count = a.parts, listed = a.parts, gr = 0;       // parts 0 .. listed - 1 lie in the row's list, the rest in slots
    if (a.shared) {
        const uint32_t hk = h / a.G, gg = h - hk * a.G, groups = a.Hkv * tiles;
        gr = (int)(gg & 15);
        const int64_t* table = behind_wait(a.table);
        const int64_t begin = table[token], units = table[token + 1] - begin, total = table[(int64_t)a.B * a.L] * groups;
        const int64_t s0 = begin * groups + (int64_t)(hk * tiles + gg / 16) * units;
        const int64_t takers = rows_takers(a, total);
        first = rows_owner(s0, total, takers);
        const int last = rows_owner(s0 + units - 1, total, takers);
        if (first < last) {
            if (listed > 0) --listed;                                // (the entry for an undivided group is not in use)
            count = listed + last - first + 1;
        } else if (a.parts == 0) return;                             // undivided: written already
    }
    const auto weight_of = [&](int s) { return s < listed ? *part_weight(a, row, s) : *slot_weight(a, first + s - listed, s == listed, gr); };
    const auto sum_of = [&](int s) { return (s < listed ? part_sum(a, row, s) : slot_sum(a, first + s - listed, s == listed, gr)); };
    float top = -INFINITY;
    for (int s = lane; s < count; s += 32) {
        const float2 ml = weight_of(s);
        if (ml.y != 0.f) top = fmaxf(top, ml.x);
    }
    #pragma unroll
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, k));
    const float ref = top == -INFINITY ? 0.f : top;
    float weight = 0.f, sum[4] = {};
    const bool in = lane * 4 < (int)a.D;
    for (int s0 = 0; s0 < count; s0 += 32) {
        float f = 0.f;
        if (s0 + lane < count) {
            const float2 ml = weight_of(s0 + lane);
            if (ml.y != 0.f) { f = exp2_fast(ml.x - ref); weight = fmaf(ml.y, f, weight); }
        }
        const int end = min(32, count - s0);
        #pragma unroll 4
        for (int s = 0; s < end; ++s) {
            const float g = __shfl_sync(0xFFFFFFFFu, f, s);
            if (g != 0.f && in) {                                    // an empty part's sums are not looked at (a NaN is no zero)
                const float4 x = *reinterpret_cast<const float4*>(sum_of(s0 + s) + lane * 4);
                sum[0] = fmaf(x.x, g, sum[0]); sum[1] = fmaf(x.y, g, sum[1]); sum[2] = fmaf(x.z, g, sum[2]); sum[3] = fmaf(x.w, g, sum[3]);
            }
        }
    }
    #pragma unroll
    for (int k = 16; k; k >>= 1) weight += __shfl_xor_sync(0xFFFFFFFFu, weight, k);
    const int64_t b = token / a.L, i = token - b * a.L;
    if (in) {
        #pragma unroll
        for (int e = 0; e < 4; ++e)
            Mma<E>::store(a.out, b * a.os[0] + i * a.os[1] + h * a.os[2] + lane * 4 + e, weight == 0.f ? 0.f : sum[e] / weight);
    }
}

template <class E, int NK>
int rows_launch(const AttnArgs& a, cudaStream_t stream)
{
    { const int rc = ensure_dynamic_smem(attention_rows_kernel<E, NK>, RowsShape<NK>::BYTES); if (rc) return rc; }
    HBQ_CUDA_TRY(launch_dependent(attention_rows_kernel<E, NK>, (unsigned)a.blocks, RW * 32, (size_t)RowsShape<NK>::BYTES, stream, a, (a.G + 15) / 16));
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

// Blocks of the few-row kernel; prefix: a row's list begins with it.  Shares of equal size over two blocks an SM; a block a
// row group where there are too many tokens for the table, or where every group is a unit or two by its bounds alone.
int attention_rows_blocks(const hbq_attention* p, bool prefix, int* shared)
{
    int sms = 148;
    device_sms(&sms);
    const int64_t groups = p->Hkv * ((p->H / p->Hkv + 15) / 16), tokens = p->B * p->L;
    int64_t keys = p->S;
    if (p->window > 0 && p->window + p->sinks < keys) keys = p->window + p->sinks;
    if (prefix) keys += p->P;
    const int64_t units = (keys + ROWS_UNIT - 1) / ROWS_UNIT;
    if (tokens > RW * 64 || units <= 1) {
        *shared = 0;
        return groups * tokens > 0x7FFFFFFF ? -1 : (int)(groups * tokens);
    }
    *shared = 1;
    const int64_t most = units * groups * tokens;
    return (int)(most < 2 * sms ? most : 2 * sms);
}

int attention_rows_launch(const AttnArgs& a, int dtype, cudaStream_t stream)
{
    return dtype == HBQ_DTYPE_F16 ? rows_type<__half>(a, stream) : rows_type<__nv_bfloat16>(a, stream);
}

int attention_join_launch(const AttnArgs& a, int dtype, cudaStream_t stream)
{
    const int64_t blocks = ((int64_t)a.B * a.L * a.H + 1) / 2;
    if (blocks > 0x7FFFFFFFll) return HBQ_ERR_UNSUPPORTED;
    const uint32_t tiles = (a.G + 15) / 16;
    if (dtype == HBQ_DTYPE_F16) HBQ_CUDA_TRY(launch_dependent(attention_join_kernel<__half>, (unsigned)blocks, 64, 0, stream, a, tiles));
    else HBQ_CUDA_TRY(launch_dependent(attention_join_kernel<__nv_bfloat16>, (unsigned)blocks, 64, 0, stream, a, tiles));
    HBQ_LAUNCH_CHECK("attention_join_kernel");
    return HBQ_OK;
}

}  // namespace hbq
