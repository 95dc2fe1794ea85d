// Rotary positions of projected heads, with 64-bit angles, after an RMS norm of every head where there is one.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (norm only)
//   (u, v) -> factor * (u cos a - v sin a, v cos a + u sin a),   a = position * inv_freq[i], for each pair i
//
// Bound by memory: each value is read once and written once.  A position's angles are the same for all of its heads, so a
// warp computes them once for many: the product and its reduction to a part of a turn in 64 bits (at position
// 10^6 an angle in 32 bits is off by 0.06), cosine and sine of that part in 32 bits.  A table of them would be read
// from memory in their place and has to be kept for every position.
#include "common.cuh"

namespace hbq {

namespace {

struct HeadsArg {
    const void* data;
    void* out;
    const void* weight;
    int64_t sb, st, sh, ob, ot, oh;
};
struct RotaryArgs {
    HeadsArg x[2];                 // queries and keys; the second is empty for one tensor
    const double* inv_freq;
    const void* positions;
    int64_t pb, pt, tokens;        // tokens = B * T
    uint32_t T, heads0, heads, D, rot;
    int interleaved, positions_64;
    float factor, eps, inv_D;
    int many;                      // a warp per token
};

constexpr int WARPS = 4;

template <class E> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ float2 up(uint32_t u) { return __half22float2(bits_h2(u)); }
    static __device__ __forceinline__ uint32_t down(float a, float b) { return h2_bits(__floats2half2_rn(a, b)); }
    static __device__ __forceinline__ float up1(const void* p, int64_t i) { return __half2float(static_cast<const __half*>(p)[i]); }
    static __device__ __forceinline__ void down1(void* p, int64_t i, float v) { static_cast<__half*>(p)[i] = __float2half_rn(v); }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 up(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t down(float a, float b)
    {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float up1(const void* p, int64_t i) { return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]); }
    static __device__ __forceinline__ void down1(void* p, int64_t i, float v) { static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v); }
};

// Cosine and sine of position * inv_freq: in turns, so that the reduction is a subtraction of the nearest whole number.
__device__ __forceinline__ float2 turn(int64_t position, double inv_freq, float factor)
{
    const double t = (double)position * (inv_freq * 0.15915494309189535);       // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    return make_float2(c * factor, s * factor);
}
__device__ __forceinline__ void rotate(float& u, float& v, float2 cs)
{
    const float r = fmaf(u, cs.x, -(v * cs.y));
    v = fmaf(v, cs.x, u * cs.y);
    u = r;
}
__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t b, int64_t t)
{
    const int64_t i = b * a.pb + t * a.pt;
    return a.positions_64 ? static_cast<const int64_t*>(a.positions)[i] : static_cast<const int32_t*>(a.positions)[i];
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{ .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 z, x, y, z;\n mov.b64 {%0, %1}, z; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("{ .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// A lane's two runs as first and second values of its eight pairs, two pairs to a register pair (the packed 32-bit operations
// halve the instructions, which bound the norm: 302 a group of heads before)
template <class E>
__device__ __forceinline__ void unpack(uint4 r0, uint4 r1, bool apart, float2 (&u)[4], float2 (&v)[4])
{
    const uint32_t x[4] = {r0.x, r0.y, r0.z, r0.w}, y[4] = {r1.x, r1.y, r1.z, r1.w};
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (apart) { u[i] = Pair<E>::up(x[i]); v[i] = Pair<E>::up(y[i]); }
        else {
            const float2 p = Pair<E>::up(i < 2 ? x[2 * i] : y[2 * i - 4]), q = Pair<E>::up(i < 2 ? x[2 * i + 1] : y[2 * i - 3]);
            u[i] = make_float2(p.x, q.x);
            v[i] = make_float2(p.y, q.y);
        }
    }
}

// Heads whose length and turning part are multiples of 16: a lane holds two runs of 8 values, which the rotation pairs
// with one another (runs c and c + rot / 16 of the half layout, neighbours of the interleaved one), so that a pair never
// leaves its lane; LANES lanes share a head and 32 / LANES heads a warp.  Each lane needs the 8 angles from 8 c on.
// A warp has one token, whose angles it computes for itself; with many tokens it walks over all of the token's heads, with
// few a token's heads are spread over the warps of its blocks (blockIdx.y).
//
// Bytes in flight are what it needs: a warp's next heads are loaded before it works on the present ones, and its first ones
// before the block's angles are known (16384 tokens of 32 heads of 128: 48 us, 5.6 TB/s; 32 + 8 heads with
// the norm: 68 us, 4.9 TB/s).
template <class E, int LANES, bool NORM>
__global__ void __launch_bounds__(WARPS * 32, 6) rotary_kernel(const __grid_constant__ RotaryArgs a)
{
    __shared__ float2 block_angles[WARPS][128];    // [warp][rot / 2]
    grid_dependency_wait();
    dependents_may_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & (LANES - 1), sub = lane / LANES;
    const uint32_t half = a.rot / 2;
    const bool in_head = (uint32_t)c * 16 < a.D, turns = (uint32_t)c * 16 < a.rot;
    // `apart`: pair i of the lane is (first run's i, second run's i); else its values are neighbours
    const bool apart = !a.interleaved;
    uint32_t d0, d1;                               // where the lane's two runs begin
    if (a.interleaved || !turns) { d0 = 16 * c; d1 = d0 + 8; }
    else { d0 = 8 * c; d1 = d0 + half; }

    // this warp's token, and its groups of heads: first the queries', then the keys'
    constexpr uint32_t PER = 32 / LANES;
    const uint32_t token = a.many ? blockIdx.x * WARPS + warp : blockIdx.x, step = a.many ? 1 : WARPS * gridDim.y;
    const bool any = token < (uint32_t)a.tokens;
    const uint32_t b = token / a.T, t = token - b * a.T;
    uint32_t g = a.many ? 0 : blockIdx.y * WARPS + warp;

    struct Item { uint4 u0, u1; E* out; };         // out: null for lanes without a head
    const auto load = [&](const HeadsArg& x, const E* from, E* to, uint32_t heads, uint32_t group) {
        Item v = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0), nullptr};
        const uint32_t h = group * PER + sub;
        if (h < heads && in_head) {
            const E* p = from + (int64_t)(int)h * (int)x.sh;
            v.u0 = *reinterpret_cast<const uint4*>(p + d0);
            v.u1 = *reinterpret_cast<const uint4*>(p + d1);
            v.out = to + (int64_t)(int)h * (int)x.oh;
        }
        return v;
    };
    const double* freq = behind_wait(a.inv_freq);
    // the lane's pairs, two and two: (u, v) -> (u uu + v vu, v vv + u uv), cosines and sines times the weights where there is a norm
    float2 uu[4], vu[4], vv[4], uv[4];
    bool ready = false;
    #pragma unroll 1
    for (int j = 0; j < 2; ++j) {
        const HeadsArg& x = a.x[j];
        const uint32_t heads = j ? a.heads - a.heads0 : a.heads0, groups = (heads + PER - 1) / PER;
        const E* from = static_cast<const E*>(x.data) + (int64_t)b * x.sb + (int64_t)t * x.st;
        E* to = static_cast<E*>(x.out) + (int64_t)b * x.ob + (int64_t)t * x.ot;
        Item next = load(x, from, to, any ? heads : 0, g);
        uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
        if (NORM && in_head && g < groups) {
            w0 = *reinterpret_cast<const uint4*>(static_cast<const E*>(x.weight) + d0);
            w1 = *reinterpret_cast<const uint4*>(static_cast<const E*>(x.weight) + d1);
        }
        if (!ready) {                              // (the first loads are on their way)
            ready = true;
            float2* angles = block_angles[warp];
            if (any) {
                const int64_t position = position_of(a, b, t);
                for (uint32_t i = lane; i < half; i += 32) angles[i] = turn(position, freq[i], a.factor);
            }
            __syncwarp();
            if (!NORM && turns && any) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 p = angles[8 * c + 2 * i], q = angles[8 * c + 2 * i + 1];
                    uu[i] = make_float2(p.x, q.x);
                    vu[i] = make_float2(-p.y, -q.y);
                }
            }
        }
        if (NORM) {
            float2 wu[4], wv[4];
            unpack<E>(w0, w1, apart, wu, wv);
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                float2 p = make_float2(1.f, 0.f), q = p;
                if (turns && any) { p = block_angles[warp][8 * c + 2 * i]; q = block_angles[warp][8 * c + 2 * i + 1]; }
                uu[i] = mul2(make_float2(p.x, q.x), wu[i]);
                uv[i] = mul2(make_float2(p.y, q.y), wu[i]);
                vv[i] = mul2(make_float2(p.x, q.x), wv[i]);
                vu[i] = mul2(make_float2(-p.y, -q.y), wv[i]);
            }
        }
        for (; g < groups && any; g += step) {
            const Item cur = next;
            next = load(x, from, to, heads, g + step);
            float2 u[4], v[4];
            unpack<E>(cur.u0, cur.u1, apart, u, v);
            float2 ss = make_float2(1.f, 1.f);
            if (NORM) {
                float2 q = make_float2(0.f, 0.f);
                #pragma unroll
                for (int i = 0; i < 4; ++i) { q = fma2(u[i], u[i], q); q = fma2(v[i], v[i], q); }
                float s = q.x + q.y;
                #pragma unroll
                for (int m = LANES / 2; m; m >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, m);
                s = rsqrtf(fmaf(s, a.inv_D, a.eps));
                ss = make_float2(s, s);
            }
            if (turns) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 r = fma2(u[i], uu[i], mul2(v[i], vu[i]));
                    v[i] = fma2(v[i], NORM ? vv[i] : uu[i], mul2(u[i], NORM ? uv[i] : make_float2(-vu[i].x, -vu[i].y)));
                    u[i] = r;
                }
            } else if (NORM) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) { u[i] = mul2(u[i], uu[i]); v[i] = mul2(v[i], vv[i]); }
            }
            if (NORM) {
                #pragma unroll
                for (int i = 0; i < 4; ++i) { u[i] = mul2(u[i], ss); v[i] = mul2(v[i], ss); }
            }
            if (cur.out) {
                if (apart) {
                    *reinterpret_cast<uint4*>(cur.out + d0) = make_uint4(Pair<E>::down(u[0].x, u[0].y), Pair<E>::down(u[1].x, u[1].y), Pair<E>::down(u[2].x, u[2].y), Pair<E>::down(u[3].x, u[3].y));
                    *reinterpret_cast<uint4*>(cur.out + d1) = make_uint4(Pair<E>::down(v[0].x, v[0].y), Pair<E>::down(v[1].x, v[1].y), Pair<E>::down(v[2].x, v[2].y), Pair<E>::down(v[3].x, v[3].y));
                } else {
                    *reinterpret_cast<uint4*>(cur.out + d0) = make_uint4(Pair<E>::down(u[0].x, v[0].x), Pair<E>::down(u[0].y, v[0].y), Pair<E>::down(u[1].x, v[1].x), Pair<E>::down(u[1].y, v[1].y));
                    *reinterpret_cast<uint4*>(cur.out + d1) = make_uint4(Pair<E>::down(u[2].x, v[2].x), Pair<E>::down(u[2].y, v[2].y), Pair<E>::down(u[3].x, v[3].x), Pair<E>::down(u[3].y, v[3].y));
                }
            }
        }
        g = g > groups ? g - groups : 0;           // among the keys' groups
        if (a.many) g = 0;
    }
}

// Every other head length, turning part, stride and alignment: a warp per head, value by value.  A lane reads both values
// of a pair before it writes either, and the norm's sum is complete before any is written, so `out` may be the input.
template <class E, bool NORM>
__global__ void __launch_bounds__(WARPS * 32) rotary_any_kernel(const __grid_constant__ RotaryArgs a)
{
    grid_dependency_wait();
    dependents_may_start();
    const double* freq = behind_wait(a.inv_freq);
    const uint32_t lane = threadIdx.x & 31, half = a.rot / 2;
    const int64_t total = a.tokens * a.heads;
    for (int64_t i = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * WARPS) {
        const int64_t token = i / a.heads, b = token / a.T, t = token - b * a.T;
        uint32_t h = (uint32_t)(i - token * a.heads);
        const bool second = h >= a.heads0;
        const HeadsArg& x = a.x[second ? 1 : 0];
        if (second) h -= a.heads0;
        const int64_t in = b * x.sb + t * x.st + h * x.sh, on = b * x.ob + t * x.ot + h * x.oh;
        float s = 1.f;
        if (NORM) {
            s = 0.f;
            for (uint32_t d = lane; d < a.D; d += 32) { const float v = Pair<E>::up1(x.data, in + d); s = fmaf(v, v, s); }
            #pragma unroll
            for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, m);
            s = rsqrtf(s / (float)a.D + a.eps);
        }
        const int64_t position = position_of(a, b, t);
        for (uint32_t p = lane; p < half; p += 32) {
            const uint32_t d0 = a.interleaved ? 2 * p : p, d1 = a.interleaved ? d0 + 1 : p + half;
            float u = Pair<E>::up1(x.data, in + d0), v = Pair<E>::up1(x.data, in + d1);
            if (NORM) { u *= s * Pair<E>::up1(x.weight, d0); v *= s * Pair<E>::up1(x.weight, d1); }
            const float2 cs = turn(position, freq[p], a.factor);
            rotate(u, v, cs);
            Pair<E>::down1(x.out, on + d0, u);
            Pair<E>::down1(x.out, on + d1, v);
        }
        for (uint32_t d = a.rot + lane; d < a.D; d += 32) {
            float v = Pair<E>::up1(x.data, in + d);
            if (NORM) v *= s * Pair<E>::up1(x.weight, d);
            Pair<E>::down1(x.out, on + d, v);
        }
    }
}

template <class E, int LANES, bool NORM>
int launch_lanes(RotaryArgs& a, int sms, cudaStream_t stream)
{
    constexpr int PER = 32 / LANES;
    const uint32_t groups = (a.heads0 + PER - 1) / PER + (a.heads - a.heads0 + PER - 1) / PER;
    // (600 tokens of 32 heads: a warp a token 4.5 us, heads spread 4.9; 1200: 5.5 and 7.0; 300: 3.5 either way)
    a.many = a.tokens >= (int64_t)sms * 4;
    const int64_t blocks = a.many ? (a.tokens + WARPS - 1) / WARPS : a.tokens;
    const unsigned spread = (groups + WARPS - 1) / WARPS, split = a.many ? 1u : spread < 65535u ? spread : 65535u;
    HBQ_CUDA_TRY(launch_dependent(rotary_kernel<E, LANES, NORM>, dim3((unsigned)blocks, split), WARPS * 32, 0, stream, a));
    HBQ_LAUNCH_CHECK("rotary_kernel");
    return HBQ_OK;
}

template <class E, bool NORM>
int launch_type(RotaryArgs& a, bool runs, cudaStream_t stream)
{
    int sms = 0;
    { const int rc = device_sms(&sms); if (rc) return rc; }
    if (runs) {
        const uint32_t lanes = a.D / 16;
        if (lanes <= 4) return launch_lanes<E, 4, NORM>(a, sms, stream);
        if (lanes <= 8) return launch_lanes<E, 8, NORM>(a, sms, stream);
        return launch_lanes<E, 16, NORM>(a, sms, stream);
    }
    const int64_t need = (a.tokens * a.heads + WARPS - 1) / WARPS, cap = (int64_t)sms * 8;
    HBQ_CUDA_TRY(launch_dependent(rotary_any_kernel<E, NORM>, (unsigned)(need < cap ? need : cap), WARPS * 32, 0, stream, a));
    HBQ_LAUNCH_CHECK("rotary_any_kernel");
    return HBQ_OK;
}

// The vector kernel's terms for one tensor: 16-byte runs everywhere, neighbouring heads less than 2^31 values apart.
bool in_runs(const hbq_heads* x)
{
    int64_t s = 0;
    if (x->stride[2] > 0x7FFFFFFF || x->out_stride[2] > 0x7FFFFFFF || x->stride[2] < 0 || x->out_stride[2] < 0) return false;
    for (int i = 0; i < 3; ++i) s |= x->stride[i] | x->out_stride[i];
    return (s % 8) == 0 && ((reinterpret_cast<uintptr_t>(x->data) | reinterpret_cast<uintptr_t>(x->out) | reinterpret_cast<uintptr_t>(x->weight)) & 15) == 0;
}

}  // namespace

int rotary_launch(const hbq_heads* q, const hbq_heads* k, const hbq_rotary* r, int dtype, int64_t B, int64_t T, int64_t D,
                  bool norm, float eps, cudaStream_t stream)
{
    if (!q || !r || B < 0 || T < 0 || D <= 0 || q->heads < 0 || (k && k->heads < 0)) return HBQ_ERR_ARG;
    if (dtype != HBQ_DTYPE_F16 && dtype != HBQ_DTYPE_BF16) return HBQ_ERR_ARG;
    if (r->rot < 2 || (r->rot & 1) || r->rot > D) return HBQ_ERR_ARG;
    const int64_t heads = q->heads + (k ? k->heads : 0);
    if (B == 0 || T == 0 || heads == 0) return HBQ_OK;
    if (!r->inv_freq || !r->positions) return HBQ_ERR_ARG;
    if (D > (1 << 20) || heads > (1 << 20) || T > 0x7FFFFFFFll || B > 0x7FFFFFFFll) return HBQ_ERR_UNSUPPORTED;
    RotaryArgs a = {};
    const hbq_heads* x[2] = {q, k};
    bool runs = (D % 16) == 0 && D <= 256 && (r->rot % 16) == 0 && B * T <= 0x7FFFFFFFll;
    for (int i = 0; i < 2; ++i) {
        if (!x[i] || x[i]->heads == 0) continue;
        if (!x[i]->data || !x[i]->out || (norm && !x[i]->weight)) return HBQ_ERR_ARG;
        a.x[i] = {x[i]->data, x[i]->out, x[i]->weight, x[i]->stride[0], x[i]->stride[1], x[i]->stride[2],
                  x[i]->out_stride[0], x[i]->out_stride[1], x[i]->out_stride[2]};
        runs = runs && in_runs(x[i]);
    }
    a.inv_freq = r->inv_freq; a.positions = r->positions; a.pb = r->pos_stride[0]; a.pt = r->pos_stride[1];
    a.tokens = B * T; a.T = (uint32_t)T; a.heads0 = (uint32_t)q->heads; a.heads = (uint32_t)heads;
    a.D = (uint32_t)D; a.rot = (uint32_t)r->rot; a.interleaved = r->interleaved != 0; a.positions_64 = r->positions_64 != 0;
    a.factor = r->factor; a.eps = eps; a.inv_D = 1.f / (float)D;
    if (dtype == HBQ_DTYPE_F16) return norm ? launch_type<__half, true>(a, runs, stream) : launch_type<__half, false>(a, runs, stream);
    return norm ? launch_type<__nv_bfloat16, true>(a, runs, stream) : launch_type<__nv_bfloat16, false>(a, runs, stream);
}

}  // namespace hbq
