// What runs between the q|k|v projection and the attention: RMS norm of every query and key head and the position rotation in
// one pass over the projection's rows, the keys and values quantised into the paged cache as they are made, and the cache
// read back.
//
//   y = x · rsqrt(mean(x²) + eps) · w          (no weight: y = x)
//   pair p of the first rope_dim elements, (a, b) -> (a·c - b·s, b·c + a·s), c + i·s = scale · e^(i · pos · inv_freq[p])
//
// A pair is (p, p + rope_dim / 2) or, `neighbours`, (2p, 2p + 1); the elements past rope_dim keep their values.
// The angle is a product in 64 bits (a position of 10^5 times a frequency near 1 has no fraction left to speak of in 32).
// Bound by memory at many tokens: 4096 of 64 + 8 heads of 64 34 us (4.4 TB/s, a large copy's 4.76). Into a cache it is bound by latency: no
// load of a row is issued before the angles are made and the barrier passed, and a key in 64 bits takes 101 to 107 registers (140 for
// rows that are not 16-byte aligned) where the rotation alone takes 42, so 4 (3) waves a SIMD hide it instead of 8: 2048 tokens of
// 32 + 8 + 8 heads of 128 into Q4_0 28 us with their rows in the last-level cache, 33 without (3.1 and 2.6 TB/s), 333 of 16 + 2 + 2 of 256 into F16 9.
// One token is the launch, 4 us from Python.
// What is only returned is computed in 32 bits; a key that is rounded to a code is computed in 64 up to the f32 value that
// the code is taken from, so that its code does not depend on the order of the norm's sum.
#include "kvcache.h"
#include "launch.h"

namespace jamhip {

namespace {

constexpr int QK_THREADS = 256;

// sin and cos of an angle of any size a position gives: the quadrant n = round(x · 2/π), the rest in [-π/4, π/4] by two
// fused steps over π/2 in two parts (106 bits, so exact to 2^-60 for |x| < 2^31), then the Taylor series, whose first
// omitted terms are (π/4)^17 / 17! and (π/4)^18 / 18!, below 5e-17.
JAMHIP_DEV void sin_cos(double x, double* sn, double* cs) {
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.5707963267948965580, x);
    r = fma(-n, 6.1232339957367658861e-17, r);
    const double z = r * r;
    double s = -1.0 / 1307674368000.0;                 // -1 / 15!
    s = fma(s, z, 1.0 / 6227020800.0);
    s = fma(s, z, -1.0 / 39916800.0);
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, r, r);
    double c = 1.0 / 20922789888000.0;                 // 1 / 16!
    c = fma(c, z, -1.0 / 87178291200.0);
    c = fma(c, z, 1.0 / 479001600.0);
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const int q = (int) (long long) n & 3;
    const double a = q & 1 ? c : s, b = q & 1 ? s : c;
    *sn = q & 2 ? -a : a;
    *cs = (q + 1) & 2 ? -b : b;
}

// Sum over LPH (a power of two up to 64) neighbouring lanes, the same in each.
template <int LPH> JAMHIP_DEV float head_sum(float v) {
    if constexpr (LPH > 1) v += dpp<0xB1>(v);
    if constexpr (LPH > 2) v += dpp<0x4E>(v);
    if constexpr (LPH > 4) v += dpp<0x141>(v);
    if constexpr (LPH > 8) v += dpp<0x140>(v);
    if constexpr (LPH > 16) v += __shfl_xor(v, 16);
    if constexpr (LPH > 32) v += __shfl_xor(v, 32);
    return v;
}
template <int LPH> JAMHIP_DEV double head_sum(double v) {
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// 1 / sqrt(v). In 32 bits with one rounding, as the definition has it (a root and a division have two): the instruction's value r, off
// by an ulp at most, corrected by half of what v · r² leaves of 1, the product v · r in two parts.
JAMHIP_DEV double inv_sqrt(double v) { return 1.0 / sqrt(v); }
JAMHIP_DEV float inv_sqrt(float v) {
    const float r = rsqrtf(v);
    if (!(r > 0.0f && r < __builtin_inff())) return r;   // of 0, Inf and NaN
    const float h = v * r, rest = fmaf(-r, fmaf(v, r, -h), fmaf(-r, h, 1.0f));
    return fmaf(0.5f * r, rest, r);
}

// 8 consecutive elements of a row, from element 8·j on, into the cache. Four neighbouring lanes hold one block of 32.
template <int TYPE> JAMHIP_DEV void cache_store8(const KvView& c, uint8_t* buf, int64_t row, int j, const float* x) {
    if constexpr (TYPE == F16) {
        half8_t h;
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = (_Float16) x[i];
        *reinterpret_cast<half8_t*>(buf + (row * c.dim + 8 * j) * 2) = h;
        return;
    }
    const int nb = c.dim / 32, t = j & 3;
    _Float16* sc = reinterpret_cast<_Float16*>(buf + c.scale_off) + row * nb + j / 4;
    if constexpr (TYPE == Q8_0) {   // d = max|x| / 127, code = round to nearest even of x · (1 / d)
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[i]));
        top = fmaxf(top, dpp<0xB1>(top));
        top = fmaxf(top, dpp<0x4E>(top));
        const float d = __fdiv_rn(top, 127.0f), inv = d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int code = (int) fminf(fmaxf(rintf(x[i] * inv), -127.0f), 127.0f);
            w[i / 4] |= (uint32_t) (code & 255) << (8 * (i % 4));
        }
        *reinterpret_cast<uint2_t*>(buf + row * c.dim + 8 * j) = uint2_t{w[0], w[1]};
        if (t == 0) *sc = (_Float16) d;
    } else {   // d = (the element of largest magnitude, the first of equals) / -8, code = floor(x · (1 / d) + 8.5), at most 15
        float top = 0.0f, at = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (fabsf(x[i]) > top) top = fabsf(x[i]), at = x[i];
        auto join = [&](float ot, float oa, bool lower) {
            if (ot > top || (ot == top && lower)) top = ot, at = oa;
        };
        join(dpp<0xB1>(top), dpp<0xB1>(at), t & 1);
        join(dpp<0x4E>(top), dpp<0x4E>(at), t & 2);
        const float d = at * -0.125f, inv = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int code = (int) fminf(fmaxf(floorf(x[i] * inv + 8.5f), 0.0f), 15.0f);
            w[i / 4] |= (uint32_t) code << (8 * (i % 4));
        }
        const uint32_t h0 = __builtin_amdgcn_update_dpp(0, w[0], 0x4E, 0xF, 0xF, true);   // elements 16 + .. of the block
        const uint32_t h1 = __builtin_amdgcn_update_dpp(0, w[1], 0x4E, 0xF, 0xF, true);
        if (t < 2)
            *reinterpret_cast<uint2_t*>(buf + row * (c.dim / 2) + j / 4 * 16 + 8 * t) = uint2_t{w[0] | h0 << 4, w[1] | h1 << 4};
        if (t == 0) *sc = (_Float16) d;
    }
}

// One head of LPH lanes, 4 pairs a lane: pair p(i) = 4·j + i (VEC) or j + LPH·i, elements (p, p + rot / 2) or (2p, 2p + 1);
// past rope_dim every pair is (2p, 2p + 1). T is the type of the arithmetic.
template <typename T, int LPH, bool VEC> struct Head {
    T a[4], b[4];
    int j, dim, rot;
    bool nbr;
    JAMHIP_DEV int pair(int i) const { return VEC ? 4 * j + i : j + LPH * i; }
    JAMHIP_DEV bool halves(int p) const { return !nbr && 2 * p < rot; }
    JAMHIP_DEV void load(const float* x) {
        if constexpr (VEC) {
            if (8 * j < dim) {
                const bool hv = halves(4 * j);
                const float4_t u = *reinterpret_cast<const float4_t*>(x + (hv ? 4 * j : 8 * j));
                const float4_t w = *reinterpret_cast<const float4_t*>(x + (hv ? 4 * j + rot / 2 : 8 * j + 4));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    a[i] = hv ? u[i] : i < 2 ? u[2 * i] : w[2 * i - 4];
                    b[i] = hv ? w[i] : i < 2 ? u[2 * i + 1] : w[2 * i - 3];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = b[i] = 0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = pair(i);
                const bool in = 2 * p < dim;
                a[i] = in ? x[halves(p) ? p : 2 * p] : 0.0f;
                b[i] = in ? x[halves(p) ? p + rot / 2 : 2 * p + 1] : 0.0f;
            }
        }
    }
    JAMHIP_DEV void norm(const float* w, float eps) {
        T ss = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) ss += a[i] * a[i] + b[i] * b[i];
        ss = head_sum<LPH>(ss);
        const T r = inv_sqrt(ss / (T) dim + (T) eps);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = pair(i);
            if (2 * p < dim) {
                a[i] = a[i] * r * (T) w[halves(p) ? p : 2 * p];
                b[i] = b[i] * r * (T) w[halves(p) ? p + rot / 2 : 2 * p + 1];
            }
        }
    }
    template <typename CS> JAMHIP_DEV void rotate(const CS* cs) {   // cs[p] = (cos, sin)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p = pair(i);
            if (2 * p < rot) {
                const T c = (T) cs[p].x, s = (T) cs[p].y, u = a[i], v = b[i];
                a[i] = u * c - v * s;
                b[i] = v * c + u * s;
            }
        }
    }
    JAMHIP_DEV void store(float* y) const {
        if constexpr (VEC) {
            if (8 * j < dim) {
                const bool hv = halves(4 * j);
                float4_t u, w;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    u[i] = (float) (hv ? a[i] : i & 1 ? b[i / 2] : a[i / 2]);
                    w[i] = (float) (hv ? b[i] : i & 1 ? b[2 + i / 2] : a[2 + i / 2]);
                }
                *reinterpret_cast<float4_t*>(y + (hv ? 4 * j : 8 * j)) = u;
                *reinterpret_cast<float4_t*>(y + (hv ? 4 * j + rot / 2 : 8 * j + 4)) = w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = pair(i);
                if (2 * p < dim) {
                    y[halves(p) ? p : 2 * p] = (float) a[i];
                    y[halves(p) ? p + rot / 2 : 2 * p + 1] = (float) b[i];
                }
            }
        }
    }
};

// A head's lanes are of one wave, whose shared memory operations are done in order.
JAMHIP_DEV void sync_wave() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One workgroup takes heads [y · per, (y + 1) · per) of one token's q | k (| v): every 256 / LPH of them at once. TYPE -1: keys
// go out as f32. The angles of the token are computed once per workgroup, one pair a thread.
template <int TYPE, int LPH, bool VEC> __global__ void __launch_bounds__(QK_THREADS) qk_norm_rope_kernel(QkRope g) {
    constexpr bool CACHE = TYPE >= 0;
    __shared__ double2 turn[256];                                        // rope_dim <= 512
    __shared__ __align__(16) float rows[CACHE ? QK_THREADS * 8 : 4];     // a group's rotated key, for its codes
    const int t = blockIdx.x, tid = threadIdx.x, j = tid % LPH, grp = tid / LPH;
    if (g.rot > 0) {
        if (2 * tid < g.rot) {
            double s, c;
            sin_cos((double) g.pos[t] * (double) g.inv_freq[tid], &s, &c);
            turn[tid] = make_double2(c * (double) g.scale, s * (double) g.scale);
        }
        __syncthreads();
    }
    const int all = g.q_heads + g.kv_heads * (CACHE ? 2 : 1);
    const int h1 = min(all, ((int) blockIdx.y + 1) * g.per);
    int64_t slot = 0;
    bool keep = true;
    if constexpr (CACHE) {
        slot = g.slots[t];
        keep = slot >= 0 && slot < g.cache.slots();   // others are not written
    }
    for (int h0 = (int) blockIdx.y * g.per; h0 < h1; h0 += QK_THREADS / LPH) {
        const int h = h0 + grp;
        const bool is_q = h < g.q_heads, is_k = !is_q && h < g.q_heads + g.kv_heads;
        if (h < h1 && (is_q || (is_k && !CACHE))) {
            Head<float, LPH, VEC> x;
            x.j = j, x.dim = g.dim, x.rot = g.rot, x.nbr = g.neighbours;
            const int i = is_q ? h : h - g.q_heads;
            x.load((is_q ? g.q + (int64_t) t * g.ldq : g.k + (int64_t) t * g.ldk) + (int64_t) i * g.dim);
            const float* w = is_q ? g.qw : g.kw;
            if (w != nullptr) x.norm(w, g.eps);
            x.rotate(turn);
            x.store((is_q ? g.qo + (int64_t) t * g.ldqo : g.ko + (int64_t) t * g.ldko) + (int64_t) i * g.dim);
        }
        if constexpr (CACHE) {
            float* mine = rows + grp * LPH * 8;
            if (h < h1 && is_k) {
                Head<double, LPH, VEC> x;
                x.j = j, x.dim = g.dim, x.rot = g.rot, x.nbr = g.neighbours;
                x.load(g.k + (int64_t) t * g.ldk + (int64_t) (h - g.q_heads) * g.dim);
                if (g.kw != nullptr) x.norm(g.kw, g.eps);
                x.rotate(turn);
                x.store(mine);
            }
            sync_wave();
            if (h < h1 && !is_q && keep && 8 * j < g.dim) {   // whole quads: dim is a multiple of 32, or the type has no blocks
                const int i = (h - g.q_heads) - (is_k ? 0 : g.kv_heads);
                float v[8];
                if (is_k || VEC) {
                    const float* s = is_k ? mine + 8 * j : g.v + (int64_t) t * g.ldv + (int64_t) i * g.dim + 8 * j;
                    const float4_t u = *reinterpret_cast<const float4_t*>(s), w = *reinterpret_cast<const float4_t*>(s + 4);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = u[e], v[4 + e] = w[e];
                } else {
                    const float* s = g.v + (int64_t) t * g.ldv + (int64_t) i * g.dim + 8 * j;
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = s[e];
                }
                cache_store8<TYPE>(g.cache, is_k ? g.cache.k : g.cache.v, g.cache.row(slot, i), j, v);
            }
            sync_wave();
        }
    }
}

// Slots read back: 4 elements a thread of each of U tokens, whose loads are in flight together; keys in blockIdx.y 0, values in 1.
// What many tokens bring back is more than the L2s hold and goes past them (16384 tokens of 8 x 128 in Q8_0 49 -> 30 us).
template <int TYPE, int U> __global__ void __launch_bounds__(256) kv_read_kernel(KvView c, const int* __restrict__ slots, int n, float* ko,
                                                                                 int ldk, float* vo, int ldv) {
    const bool is_v = blockIdx.y == 1 || ko == nullptr;
    const int per = c.kv * c.dim / 4, step = (n + U - 1) / U;   // 4-element pieces of a token; the thread's tokens are step apart
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    const int t0 = (int) (i / per), p = (int) (i - (int64_t) t0 * per), head = p / (c.dim / 4), e = (p - head * (c.dim / 4)) * 4;
    if (t0 >= step) return;
    const uint8_t* buf = is_v ? c.v : c.k;
    int64_t slot[U];
    float4_t x[U];
#pragma unroll
    for (int u = 0; u < U; u++) slot[u] = slots[min(t0 + u * step, n - 1)];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const bool in = slot[u] >= 0 && slot[u] < c.slots();
        x[u] = kv_load4<TYPE>(buf, c.scale_off, c.dim, c.row(in ? slot[u] : 0, head), e);
        if (!in) x[u] = float4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int t = t0 + u * step;
        if (t >= n) continue;
        float* o = (is_v ? vo + (int64_t) t * ldv : ko + (int64_t) t * ldk) + head * c.dim + e;
        if ((reinterpret_cast<uintptr_t>(o) & 15) == 0) {
            if constexpr (U > 1) __builtin_nontemporal_store(x[u], reinterpret_cast<float4_t*>(o));
            else *reinterpret_cast<float4_t*>(o) = x[u];
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = x[u][k];
        }
    }
}

template <int TYPE, int LPH> hipError_t launch_rope(QkRope g, bool vec, hipStream_t st) {
    const int all = g.q_heads + g.kv_heads * (TYPE >= 0 ? 2 : 1), at_once = QK_THREADS / LPH;
    // few tokens: a workgroup per pass of heads, so that no thread does two in a row; many: one per token, whose angles are then
    // computed once. In us, by pass / by token: 64 + 8 heads of 64, 128 tokens 5.2 / 6.7, 511 7.2 / 9.0, 768 9.7 / 10.6, 1024 12.1 / 11.8;
    // 32 + 8 of 128, 511 8.7 / 9.8, 768 12.6 / 11.8, 2048 26.7 / 26.0; with 8 more into Q8_0, 64 5.3 / 7.7, 384 9.9 / 10.5, 511 11.8 / 11.2,
    // 1024 16.8 / 15.7
    g.per = g.n < 512 ? at_once : (all + at_once - 1) / at_once * at_once;
    const dim3 grid(g.n, (all + g.per - 1) / g.per);
    if (vec) qk_norm_rope_kernel<TYPE, LPH, true><<<grid, QK_THREADS, 0, st>>>(g);
    else qk_norm_rope_kernel<TYPE, LPH, false><<<grid, QK_THREADS, 0, st>>>(g);
    return hipGetLastError();
}

template <int TYPE> hipError_t launch_rope(const QkRope& g, bool vec, hipStream_t st) {
    const int lanes = (g.dim + 7) / 8;
    return lanes <= 8 ? launch_rope<TYPE, 8>(g, vec, st) : lanes <= 16 ? launch_rope<TYPE, 16>(g, vec, st)
         : lanes <= 32 ? launch_rope<TYPE, 32>(g, vec, st) : launch_rope<TYPE, 64>(g, vec, st);
}

}  // namespace

hipError_t launch_qk_norm_rope(int type, const QkRope& g, hipStream_t st) {
    if (g.n <= 0) return hipSuccess;
    if (g.dim > 512) return hipErrorNotSupported;
    auto fits = [](const void* p, int ld) { return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 4 == 0); };
    const bool vec = g.dim % 8 == 0 && g.rot % 8 == 0 && fits(g.q, g.ldq) && fits(g.qo, g.ldqo) && fits(g.k, g.ldk) &&
                     fits(g.ko, g.ldko) && fits(g.v, g.ldv);
    switch (type) {
        case -1: return launch_rope<-1>(g, vec, st);
        case F16: return launch_rope<F16>(g, vec, st);
        case Q8_0: return launch_rope<Q8_0>(g, vec, st);
        case Q4_0: return launch_rope<Q4_0>(g, vec, st);
    }
    return hipErrorNotSupported;
}

hipError_t launch_kv_read(int type, const KvView& c, const int* slots, int n, float* ko, int ldk, float* vo, int ldv,
                          hipStream_t st) {
    if (n <= 0) return hipSuccess;
    // eight tokens a thread from where that still leaves eight workgroups a CU
    const int64_t pieces = c.kv * c.dim / 4, u = n * pieces >= 8 * 8 * 256 * 256 ? 8 : 1;
    const int64_t blocks = ((n + u - 1) / u * pieces + 255) / 256;
    if (blocks > INT32_MAX) return hipErrorNotSupported;
    const dim3 grid((uint32_t) blocks, ko != nullptr && vo != nullptr ? 2 : 1);
    auto go = [&](auto type) {
        constexpr int T = decltype(type)::value;
        if (u == 8) kv_read_kernel<T, 8><<<grid, 256, 0, st>>>(c, slots, n, ko, ldk, vo, ldv);
        else kv_read_kernel<T, 1><<<grid, 256, 0, st>>>(c, slots, n, ko, ldk, vo, ldv);
    };
    switch (type) {
        case F16: go(std::integral_constant<int, F16>{}); break;
        case Q8_0: go(std::integral_constant<int, Q8_0>{}); break;
        case Q4_0: go(std::integral_constant<int, Q4_0>{}); break;
        default: return hipErrorNotSupported;
    }
    return hipGetLastError();
}

}  // namespace jamhip
