// Rotary positions with several axes and the per-head RMS norm in the same pass (DeftRotary, include/deft_hip.h): one read and one write of
// every head, keys (and values) straight into the rows of a cache where there is one.
//
// Memory bound: 2 * D * size bytes per head against ~7 flops an element, so the layout is chosen for the loads.  A lane owns TWO 16-byte chunks
// of a head whose elements are each other's rotation partners -- (c, R + c) for split pairs, two neighbouring chunks for adjacent ones -- so the
// rotation needs no exchange between lanes and the norm one butterfly over the D / (2 V) lanes of a head (V = elements of 16 bytes).  The
// angles depend on the token alone: a wave forms its token's R sines and cosines once (in double up to the quarter turn, then two short
// polynomials) and keeps the 2 V values of its lane's chunks in registers for all heads it handles.
#include "common.h"

namespace {

template <int DT> struct Elem;
template <> struct Elem<DEFT_F32> { typedef float T; };
template <> struct Elem<DEFT_F16> { typedef _Float16 T; };
template <> struct Elem<DEFT_BF16> { typedef __bf16 T; };

constexpr int ROT_MAX_PAIRS = 128;
constexpr int ROT_WAVES = 4;

// sine and cosine of 2 pi r, r in turns: quarter turns leave in double, then |t| <= pi / 4 in fp32 (Taylor: the first dropped terms are
// t^11 / 11! < 2e-9 and t^12 / 12! < 2e-10, below half an fp32 ulp of the results)
__device__ __forceinline__ void turn_sincos(double r, float& sn, float& cs) {
    const double r4 = r * 4.0, n = rint(r4);
    const float t = (float)((r4 - n) * 1.5707963267948966);
    const int quad = (int)(n - 4.0 * floor(n * 0.25));
    const float t2 = t * t;
    const float s = t * fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), 1.f);
    const float c = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
    const float a = (quad & 1) ? c : s, b = (quad & 1) ? s : c;
    sn = (quad & 2) ? -a : a;
    cs = ((quad + 1) & 2) ? -b : b;
}

// One wave: one token, `parts` waves sharing its heads.  LPH lanes a head (a power of two >= D / 2V; the surplus lanes of D = 96 idle).
template <int DT, bool ADJ>
__global__ __launch_bounds__(64 * ROT_WAVES) void rotary_kernel(DeftRotary p, int lph_log2, int parts) {
    typedef typename Elem<DT>::T T;
    constexpr int V = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    __shared__ __attribute__((aligned(16))) float cs_s[ROT_WAVES][2][ROT_MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long unit = (long long)blockIdx.x * ROT_WAVES + wave;
    const int t = (int)(unit / parts), part = (int)(unit - (long long)t * parts);
    const bool live = t < p.T;
    float* const cs_c = cs_s[wave][0];
    float* const cs_n = cs_s[wave][1];
    if (live) {
        for (int i = lane; i < p.R; i += 64) {
            int a = p.axis[i];
            a = a < 0 ? 0 : (a < p.A ? a : p.A - 1);
            const size_t at = (size_t)t * p.A + a;
            const double x = p.pos_float ? (double)((const float*)p.pos)[at] : (double)((const int*)p.pos)[at];
            float sn, cs;
            turn_sincos(x * p.freq[i] * 0.15915494309189535, sn, cs);
            cs_c[i] = cs;
            cs_n[i] = p.inverse ? -sn : sn;
        }
    }
    __syncthreads();
    if (!live) return;
    const int lph = 1 << lph_log2, hpw = 64 >> lph_log2;
    const int c = lane & (lph - 1), sub = lane >> lph_log2;
    const bool mine = c < p.D / (2 * V);
    const bool turns = c * V < p.R;
    // this lane's two chunks, and the sines and cosines of the pairs c V .. c V + V - 1
    const int lo = ADJ || !turns ? c * 2 * V : c * V;
    const int hi = ADJ || !turns ? lo + V : p.R + c * V;
    float cv[V], sv[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        cv[e] = turns ? cs_c[c * V + e] : 1.f;
        sv[e] = turns ? cs_n[c * V + e] : 0.f;
    }
    const int Hqk = p.Hq + (p.k ? p.Hk : 0), Hall = Hqk + (p.v ? p.Hk : 0);
    long long krow = t;
    bool kput = true;
    if (p.row && p.k) {
        krow = p.row[t];
        kput = krow >= 0 && krow < p.rows;
    }
    for (int h0 = part * hpw; h0 < Hall; h0 += parts * hpw) {
        const int h = h0 + sub;
        const bool isq = h < p.Hq, isv = h >= Hqk;
        const bool on = mine && h < Hall;
        const T* src = nullptr;
        T* dst = nullptr;
        if (on) {
            if (isq) {
                src = (const T*)p.q + (long long)t * p.ldq + (long long)h * p.hsq;
                dst = (T*)p.q_out + (long long)t * p.ldqo + (long long)h * p.hsqo;
            } else if (!isv) {
                src = (const T*)p.k + (long long)t * p.ldk + (long long)(h - p.Hq) * p.hsk;
                dst = (T*)p.k_out + krow * p.ldko + (long long)(h - p.Hq) * p.hsko;
            } else {
                src = (const T*)p.v + (long long)t * p.ldv + (long long)(h - Hqk) * p.hsv;
                dst = (T*)p.v_out + krow * p.ldvo + (long long)(h - Hqk) * p.hsvo;
            }
        }
        vec a, b;
#pragma unroll
        for (int e = 0; e < V; ++e) { a[e] = (T)0.f; b[e] = (T)0.f; }
        if (on) { a = *(const vec*)(src + lo); b = *(const vec*)(src + hi); }
        float x[V], y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { x[e] = (float)a[e]; y[e] = (float)b[e]; }
        if (p.norm) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
            for (int s = 1; s < lph; s <<= 1) ss += __shfl_xor(ss, s);
            const float r = 1.f / sqrtf(ss / (float)p.D + p.eps);
            const float* w = isq ? p.q_weight : p.k_weight;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[e] *= r * (w && on ? w[lo + e] : 1.f);
                y[e] *= r * (w && on ? w[hi + e] : 1.f);
            }
        }
        if (!on || !(isq || kput)) continue;
        if (!isv) {
            if (ADJ) {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    const float x0 = x[e], x1 = x[e + 1], y0 = y[e], y1 = y[e + 1];
                    x[e] = x0 * cv[e / 2] - x1 * sv[e / 2];
                    x[e + 1] = x1 * cv[e / 2] + x0 * sv[e / 2];
                    y[e] = y0 * cv[V / 2 + e / 2] - y1 * sv[V / 2 + e / 2];
                    y[e + 1] = y1 * cv[V / 2 + e / 2] + y0 * sv[V / 2 + e / 2];
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xe = x[e], ye = y[e];
                    x[e] = xe * cv[e] - ye * sv[e];
                    y[e] = ye * cv[e] + xe * sv[e];
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e) { a[e] = (T)x[e]; b[e] = (T)y[e]; }
        }
        *(vec*)(dst + lo) = a;
        *(vec*)(dst + hi) = b;
    }
}

bool in_fits(long long ld, long long hs, int V) { return ld % V == 0 && hs % V == 0 && ld >= 0 && hs >= 0; }
// written rows must not share elements
bool out_fits(long long ld, long long hs, int V, long long rows, int H, int D) {
    return in_fits(ld, hs, V) && (rows <= 1 || ld >= D) && (H <= 1 || hs >= D);
}

template <int DT>
void rotary_launch(const DeftRotary& d, hipStream_t s, int lph_log2, int parts, unsigned grid) {
    if (d.adjacent) hipLaunchKernelGGL((rotary_kernel<DT, true>), dim3(grid), dim3(64 * ROT_WAVES), 0, s, d, lph_log2, parts);
    else hipLaunchKernelGGL((rotary_kernel<DT, false>), dim3(grid), dim3(64 * ROT_WAVES), 0, s, d, lph_log2, parts);
}

}  // namespace

extern "C" int deft_rotary(const DeftRotary* d, void* stream) {
    DEFT_CHECK(d && d->q && d->q_out && d->pos && d->freq && d->axis, -120, "deft_rotary: null pointer");
    DEFT_CHECK(!d->k || d->k_out, -120, "deft_rotary: k without k_out");
    DEFT_CHECK(!d->v || (d->k && d->v_out), -120, "deft_rotary: v needs k and v_out");
    DEFT_CHECK(d->dtype == DEFT_F32 || d->dtype == DEFT_F16 || d->dtype == DEFT_BF16, -121, "deft_rotary: dtype=%d", d->dtype);
    const int V = d->dtype == DEFT_F32 ? 4 : 8;
    DEFT_CHECK(d->D > 0 && d->D <= 2 * ROT_MAX_PAIRS && d->D % (2 * V) == 0, -122, "deft_rotary: D=%d (a multiple of %d, at most %d)", d->D, 2 * V,
               2 * ROT_MAX_PAIRS);
    DEFT_CHECK(d->R > 0 && d->R % V == 0 && 2 * d->R <= d->D, -122, "deft_rotary: R=%d pairs (a multiple of %d, 2 R <= D=%d)", d->R, V, d->D);
    DEFT_CHECK(d->A >= 1 && d->A <= 8, -122, "deft_rotary: A=%d axes (1 .. 8)", d->A);
    DEFT_CHECK(d->T >= 0 && d->Hq > 0 && (!d->k || d->Hk > 0) && d->Hq <= 4096 && d->Hk <= 4096, -123, "deft_rotary: T=%d Hq=%d Hk=%d", d->T, d->Hq, d->Hk);
    size_t al = (size_t)d->q | (size_t)d->q_out;
    const long long orows = d->row ? d->rows : d->T;
    bool fit = in_fits(d->ldq, d->hsq, V) && out_fits(d->ldqo, d->hsqo, V, d->T, d->Hq, d->D);
    if (d->k) {
        al |= (size_t)d->k | (size_t)d->k_out;
        fit = fit && in_fits(d->ldk, d->hsk, V) && out_fits(d->ldko, d->hsko, V, orows, d->Hk, d->D);
    }
    if (d->v) {
        al |= (size_t)d->v | (size_t)d->v_out;
        fit = fit && in_fits(d->ldv, d->hsv, V) && out_fits(d->ldvo, d->hsvo, V, orows, d->Hk, d->D);
    }
    DEFT_CHECK((al & 15) == 0, -124, "deft_rotary: pointers must be 16-byte aligned");
    DEFT_CHECK(fit, -125, "deft_rotary: strides must be multiples of %d elements and keep heads apart", V);
    DEFT_CHECK(!d->row || d->rows >= 0, -126, "deft_rotary: rows=%lld", d->rows);
    if (d->T == 0) return 0;
    int lph_log2 = 0;
    while ((1 << lph_log2) < d->D / (2 * V)) ++lph_log2;
    const int heads = d->Hq + (d->k ? d->Hk : 0) + (d->v ? d->Hk : 0);
    const int passes = deft_cdiv(heads, 64 >> lph_log2);
    // waves per token: one is the least angle work; few tokens take more, up to one pass each, until the chip's 256 x 16 waves are there
    int parts = 1;
    while (parts < passes && (long long)d->T * parts < 4096) ++parts;
    const long long units = (long long)d->T * parts;
    const unsigned grid = (unsigned)((units + ROT_WAVES - 1) / ROT_WAVES);
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == DEFT_F32) rotary_launch<DEFT_F32>(*d, s, lph_log2, parts, grid);
    else if (d->dtype == DEFT_F16) rotary_launch<DEFT_F16>(*d, s, lph_log2, parts, grid);
    else rotary_launch<DEFT_BF16>(*d, s, lph_log2, parts, grid);
    DEFT_CHECK_LAUNCH("rotary");
    return 0;
}
