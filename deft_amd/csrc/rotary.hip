// Rotary positions with several axes and the per-head RMS norm in the same pass (DeftRotary, include/deft_hip.h): one read and one write of
// every head, keys (and values) straight into the rows of a cache where there is one.
//
// Memory bound: 2 * D * size bytes per head against ~7 flops an element, so the layout is chosen for the loads.  A lane owns TWO 16-byte chunks
// of a head whose elements are each other's rotation partners -- (c, R + c) for split pairs, two neighbouring chunks for adjacent ones -- so the
// rotation needs no exchange between lanes and the norm one butterfly over the D / (2 V) lanes of a head (V = elements of 16 bytes).  The
// angles depend on the token alone: a wave forms its token's R sines and cosines once (in double up to the quarter turn, then two short
// polynomials) and keeps the 2 V values of its lane's chunks in registers for all heads it handles.
// Measured (one MI355X, cold inputs): 32781 tokens of 32 + 8 heads of 128, bf16, norm and rotation: 145 us, 4.65 TB/s (a large copy: 5.1); 100 fp32
// tokens of 8 + 8 heads of 32: 4.1 us on the device.
#include <type_traits>

#include "common.h"

namespace {

template <int DT> struct Elem;
template <> struct Elem<DEFT_F32> { typedef float T; };
template <> struct Elem<DEFT_F16> { typedef _Float16 T; };
template <> struct Elem<DEFT_BF16> { typedef __bf16 T; };

constexpr int ROT_MAX_PAIRS = 128;
constexpr int ROT_WAVES = 4;
constexpr int ROT_ANGLES = 512;          // angles a wave holds: tokens of the wave x pairs <= 64 V (few heads) or ROT_MAX_PAIRS (one token)

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

#ifndef DEFT_DPP_HOOK          /* the unit-test SIMT emulator pre-defines these hooks */
#define DEFT_DPP_XCHG(v, ctrl) __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true))
// v + the value of lane l ^ S, where the lanes of each aligned group of S hold the same v: exchanges inside the register file (S < 16) -- quad
// permutations, then mirrors of 8 and 16 lanes, which meet a lane of the other half
template <int S> __device__ __forceinline__ float deft_add_xor(float v) {
    if constexpr (S == 1) return v + DEFT_DPP_XCHG(v, 0xB1);
    else if constexpr (S == 2) return v + DEFT_DPP_XCHG(v, 0x4E);
    else if constexpr (S == 4) return v + DEFT_DPP_XCHG(v, 0x141);
    else if constexpr (S == 8) return v + DEFT_DPP_XCHG(v, 0x140);
    else return v + __shfl_xor(v, S);
}
__device__ __forceinline__ float deft_rsq(float x) { return __builtin_amdgcn_rsqf(x); }
__device__ __forceinline__ unsigned long long deft_ballot(bool b) { return __ballot(b); }
#endif
// sum over the LPH lanes of a head
template <int LPH> __device__ __forceinline__ float head_sum(float v) {
    if constexpr (LPH > 1) v = deft_add_xor<1>(v);
    if constexpr (LPH > 2) v = deft_add_xor<2>(v);
    if constexpr (LPH > 4) v = deft_add_xor<4>(v);
    if constexpr (LPH > 8) v = deft_add_xor<8>(v);
    if constexpr (LPH > 16) v = deft_add_xor<16>(v);
    return v;
}

// One wave: one token, `parts` waves sharing its heads; or, where all heads of a token take a fraction of the lanes, several tokens (slots lanes' heads
// each: 64 / LPH / slots tokens).  LPH lanes a head (a power of two >= D / 2V; the surplus lanes of D = 96 idle).
// The heads of the next pass are fetched before those of this one are worked on, the first ones before the angles; norm weights stay in registers.
template <int DT, bool ADJ, bool NORM, int LPH, bool MANY>
__global__ __launch_bounds__(64 * ROT_WAVES) void rotary_kernel(DeftRotary p, int parts, int slots_log2, float inv_d) {
    typedef typename Elem<DT>::T T;
    constexpr int V = 16 / (int)sizeof(T), HPW = 64 / LPH;
    typedef T vec __attribute__((ext_vector_type(V)));
    __shared__ __attribute__((aligned(16))) float cs_s[ROT_WAVES][2][MANY ? ROT_ANGLES : ROT_MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned unit = blockIdx.x * ROT_WAVES + wave;                           // (at most 2^26)
    const int c = lane & (LPH - 1), sub = lane / LPH, slots = MANY ? 1 << slots_log2 : HPW;
    const int tokens = MANY ? HPW >> slots_log2 : 1, tok = MANY ? sub >> slots_log2 : 0;      // of this wave
    const int wt = __builtin_amdgcn_readfirstlane((int)(parts == 1 ? unit : unit / (unsigned)parts)), part = __builtin_amdgcn_readfirstlane((int)(unit - (unsigned)wt * (unsigned)parts));
    const int t0 = wt * tokens, t = t0 + tok;
    const bool some = t0 < p.T, live = t < p.T;
    const bool mine = live && c < p.D / (2 * V);
    const bool turns = c * V < p.R;
    // this lane's two chunks; the pairs whose sines and cosines it needs are c V .. c V + V - 1
    const int lo = ADJ || !turns ? c * 2 * V : c * V;
    const int hi = ADJ || !turns ? lo + V : p.R + c * V;
    const int Hqk = p.Hq + (p.k ? p.Hk : 0), Hall = Hqk + (p.v ? p.Hk : 0);
    long long krow = t;
    bool kput = true;
    if (live && p.row && p.k) {
        krow = p.row[t];
        kput = krow >= 0 && krow < p.rows;
    }
    const T* const qt = (const T*)p.q + (long long)t * p.ldq;
    const T* const kt = (const T*)p.k + (long long)t * p.ldk;
    const T* const vt = (const T*)p.v + (long long)t * p.ldv;
    auto load = [&](int h, vec& a, vec& b) {
#pragma unroll
        for (int e = 0; e < V; ++e) { a[e] = (T)0.f; b[e] = (T)0.f; }
        if (mine && h < Hall) {
            const T* src = h < p.Hq ? qt + (long long)h * p.hsq : h < Hqk ? kt + (long long)(h - p.Hq) * p.hsk : vt + (long long)(h - Hqk) * p.hsv;
            a = *(const vec*)(src + lo);
            b = *(const vec*)(src + hi);
        }
    };
    int h = part * slots + (sub & (slots - 1));
    vec a, b;
    load(h, a, b);
    float* const cs_c = cs_s[wave][0];
    float* const cs_n = cs_s[wave][1];
    if (some) {
        const int n = (p.T - t0 < tokens ? p.T - t0 : tokens) * p.R;
        for (int i = lane; i < n; i += 64) {
            const int k = tokens == 1 ? 0 : i / p.R, pair = i - k * p.R;
            int ax = p.axis[pair];
            ax = ax < 0 ? 0 : (ax < p.A ? ax : p.A - 1);
            const size_t row = (size_t)(t0 + k) * p.A;
            int raw[3];                                                            // (the usual axes wait for no table)
#pragma unroll
            for (int a = 0; a < 3; ++a) raw[a] = ((const int*)p.pos)[row + (a < p.A ? a : 0)];
            int bits = ax == 0 ? raw[0] : ax == 1 ? raw[1] : raw[2];
            if (ax > 2) bits = ((const int*)p.pos)[row + ax];
            const double x = p.pos_float ? (double)__int_as_float(bits) : (double)bits;
            float sn, cs;
            turn_sincos(x * p.freq[pair] * 0.15915494309189535, sn, cs);
            cs_c[i] = cs;
            cs_n[i] = p.inverse ? -sn : sn;
        }
    }
    __syncthreads();
    if (!some) return;
    const int at = tok * p.R + c * V;                                              // (rows behind T: values nobody uses, inside the array)
    float cv[V], sv[V], wq[2 * V], wk[2 * V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        cv[e] = turns && live ? cs_c[at + e] : 1.f;
        sv[e] = turns && live ? cs_n[at + e] : 0.f;
    }
    if constexpr (NORM) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
            const int d = e < V ? lo + e : hi + e - V;
            wq[e] = p.q_weight && mine ? p.q_weight[d] : 1.f;
            wk[e] = p.k_weight && mine ? p.k_weight[d] : 1.f;
        }
    }
    T* const qo = (T*)p.q_out + (long long)t * p.ldqo;
    T* const ko = (T*)p.k_out + krow * p.ldko;
    T* const vo = (T*)p.v_out + krow * p.ldvo;
    const long long hsqo = p.hsqo, hsko = p.hsko, hsvo = p.hsvo;
    // One pass's head of this lane: norm, rotation, write.  A head is far when its squares leave fp32, or the mean comes near the end of it (where the
    // hardware's root takes no subnormal): it is brought to about 1 by a power of two first.  That is the second loop's work (in the first one its
    // registers cost a wave a SIMD: 145 -> 155 us, 40 heads of 128): the first one ends in front of a pass with such a head (false: not written).
    auto head = [&](auto any, int h, vec& a, vec& b) -> bool {
        constexpr bool ANY = decltype(any)::value;
        const bool isq = h < p.Hq, isv = h >= Hqk;
        float x[V], y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { x[e] = (float)a[e]; y[e] = (float)b[e]; }
        if constexpr (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
            ss = head_sum<LPH>(ss);
            const float m = fmaf(ss, inv_d, p.eps);
            float r = deft_rsq(m);
            const bool far = mine && h < Hqk && !(m >= 1e-30f && ss <= 1e37f);
            if constexpr (!ANY) {
                if (deft_ballot(far) != 0) return false;
            } else {
                float top = sqrtf(p.eps);
#pragma unroll
                for (int e = 0; e < V; ++e) top = fmaxf(top, fmaxf(fabsf(x[e]), fabsf(y[e])));
#pragma unroll
                for (int s = 1; s < LPH; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
                const int up = 254 - ((__float_as_int(top) >> 23) & 255);
                const float by = far ? __int_as_float((up < 1 ? 1 : up > 253 ? 253 : up) << 23) : 1.f;
                ss = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[e] *= by;
                    y[e] *= by;
                    ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
                }
                ss = head_sum<LPH>(ss);
                r = far ? 1.f / sqrtf(fmaf(ss, inv_d, p.eps * by * by)) : r;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[e] *= r * (isq ? wq[e] : wk[e]);
                y[e] *= r * (isq ? wq[V + e] : wk[V + e]);
            }
        }
        if (mine && h < Hall && (isq || kput)) {
            if (!isv) {
                if (!turns) {                                                      // (by its lanes: 1 * x - 0 * y is not x beside an infinity)
                } else if constexpr (ADJ) {
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
            T* const dst = isq ? qo + (long long)h * hsqo : !isv ? ko + (long long)(h - p.Hq) * hsko : vo + (long long)(h - Hqk) * hsvo;
            // (non-temporal stores write 671 MB in 139 us instead of 144.5, but the attention behind them then reads q and k from memory: 5000 fp32
            // tokens, both calls, 43 -> 57 us)
            *(vec*)(dst + lo) = a;
            *(vec*)(dst + hi) = b;
        }
        return true;
    };
    int h0 = part * slots;
    for (; h0 < Hall; h0 += parts * slots) {
        vec a2, b2;
        load(h + parts * slots, a2, b2);
        if (!head(std::false_type(), h, a, b)) break;
        a = a2;
        b = b2;
        h += parts * slots;
    }
    if constexpr (NORM) {
#pragma unroll 1
        for (; h0 < Hall; h0 += parts * slots, h += parts * slots) {
            load(h, a, b);
            head(std::true_type(), h, a, b);
        }
    }
}

bool in_fits(long long ld, long long hs, int V) { return ld % V == 0 && hs % V == 0 && ld >= 0 && hs >= 0; }
// written rows must not share elements
bool out_fits(long long ld, long long hs, int V, long long rows, int H, int D) {
    return in_fits(ld, hs, V) && deft_rows_apart(ld, hs, rows, H, D);
}

struct RotLaunch { unsigned grid; int parts, slots_log2; float inv_d; hipStream_t s; };
template <int DT, int LPH, bool MANY>
void rotary_launch_k(const DeftRotary& d, const RotLaunch& l) {
    const dim3 g(l.grid), b(64 * ROT_WAVES);
    if (d.norm) {
        if (d.adjacent) hipLaunchKernelGGL((rotary_kernel<DT, true, true, LPH, MANY>), g, b, 0, l.s, d, l.parts, l.slots_log2, l.inv_d);
        else hipLaunchKernelGGL((rotary_kernel<DT, false, true, LPH, MANY>), g, b, 0, l.s, d, l.parts, l.slots_log2, l.inv_d);
    } else {
        if (d.adjacent) hipLaunchKernelGGL((rotary_kernel<DT, true, false, LPH, MANY>), g, b, 0, l.s, d, l.parts, l.slots_log2, l.inv_d);
        else hipLaunchKernelGGL((rotary_kernel<DT, false, false, LPH, MANY>), g, b, 0, l.s, d, l.parts, l.slots_log2, l.inv_d);
    }
}
template <int DT, int LPH>
void rotary_launch(const DeftRotary& d, const RotLaunch& l) {
    if ((64 / LPH) >> l.slots_log2 > 1) rotary_launch_k<DT, LPH, true>(d, l);
    else rotary_launch_k<DT, LPH, false>(d, l);
}
template <int DT>
void rotary_launch_lanes(const DeftRotary& d, const RotLaunch& l, int lanes) {
    switch (lanes) {
        case 1: rotary_launch<DT, 1>(d, l); break;
        case 2: rotary_launch<DT, 2>(d, l); break;
        case 4: rotary_launch<DT, 4>(d, l); break;
        case 8: rotary_launch<DT, 8>(d, l); break;
        case 16: rotary_launch<DT, 16>(d, l); break;
        default: if constexpr (DT == DEFT_F32) rotary_launch<DT, 32>(d, l);         // (fp32, D > 128)
    }
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
    DEFT_CHECK(d->T >= 0 && d->T <= (1 << 30) && d->Hq > 0 && (!d->k || d->Hk > 0) && d->Hq <= 4096 && d->Hk <= 4096, -123, "deft_rotary: T=%d Hq=%d Hk=%d", d->T, d->Hq, d->Hk);
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
    DEFT_CHECK(fit, -125, "deft_rotary: strides must be multiples of %d elements and keep written rows apart", V);
    DEFT_CHECK(!d->norm || d->eps >= 0.f, -127, "deft_rotary: eps=%g", (double)d->eps);
    DEFT_CHECK(!d->row || d->rows >= 0, -126, "deft_rotary: rows=%lld", d->rows);
    if (d->T == 0) return 0;
    int lanes = 1;
    while (lanes < d->D / (2 * V)) lanes *= 2;
    const int heads = d->Hq + (d->k ? d->Hk : 0) + (d->v ? d->Hk : 0);
    const int passes = deft_cdiv(heads, 64 / lanes);
    // waves per token: one is the least angle work; few tokens take more, up to one pass each, until the chip has 4096 waves (200 tokens of 24 heads of 64:
    // 5.6 us against 6.4 with one)
    int parts = 1;
    while (parts < passes && (long long)d->T * parts < 4096) ++parts;
    // tokens per wave: more than one where their heads fit, as long as 4096 waves remain (60000 tokens of 1 + 1 heads, D = 32: 28 -> 9 us; of 4 + 1, D = 64:
    // 75 -> 46; a kernel of its own, since per-lane tokens cost the one-token form 7 %)
    int slots_log2 = 0, tokens = 1;
    while ((64 / lanes) >> slots_log2 > 1) ++slots_log2;
    while (slots_log2 > 0 && heads <= 1 << (slots_log2 - 1) && d->T / (2 * tokens) >= 4096) { --slots_log2; tokens *= 2; }
    const long long units = (long long)deft_cdiv(d->T, tokens) * parts;
    DEFT_CHECK(units <= (1 << 26) - ROT_WAVES, -123, "deft_rotary: T=%d (a launch has fewer than 2^32 threads)", d->T);
    const RotLaunch l = {(unsigned)((units + ROT_WAVES - 1) / ROT_WAVES), parts, slots_log2, 1.f / (float)d->D, (hipStream_t)stream};
    if (d->dtype == DEFT_F32) rotary_launch_lanes<DEFT_F32>(*d, l, lanes);
    else if (d->dtype == DEFT_F16) rotary_launch_lanes<DEFT_F16>(*d, l, lanes);
    else rotary_launch_lanes<DEFT_BF16>(*d, l, lanes);
    DEFT_CHECK_LAUNCH("rotary");
    return 0;
}
