// Attention over packed sequences of different lengths with grouped heads (DeftAttn, include/deft_hip.h).
//
//   s_j = scale * q . k_j over the keys the row sees,  o = sum_j e^(s_j - M) v_j / sum_j e^(s_j - M),  M = max_j s_j
//
// in one pass over the keys: M and the two sums are carried along and multiplied by e^(M_old - M_new) when a larger score comes.  Everything
// is fp32; the result is rounded once.
//
// This form: one wave a (query, head) row.  64 keys at a time, a lane forms the score of one key, then the lanes own the columns of o.
#include "common.h"

namespace {

template <int DT> struct Elem;
template <> struct Elem<DEFT_F32> { typedef float T; };
template <> struct Elem<DEFT_F16> { typedef _Float16 T; };
template <> struct Elem<DEFT_BF16> { typedef __bf16 T; };

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// the sequence of query row t: the last b with q_start[b] <= t; -1 when t belongs to none
__device__ __forceinline__ int seq_of(const DeftAttn& p, int t) {
    int lo = 0, hi = p.B;                       // (q_start has B + 1 entries)
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.q_start[mid] <= t) lo = mid; else hi = mid - 1;
    }
    return lo < p.B && p.q_start[lo] <= t ? lo : -1;
}

// rows of the keys of sequence b: their count m, and the element offsets of the first row
__device__ __forceinline__ int keys_of(const DeftAttn& p, int b, int nq, long long& koff, long long& voff) {
    int m = p.k_len ? p.k_len[b] : nq;
    int at = p.k_start ? p.k_start[b] : p.q_start[b];
    if (p.cap > 0) {
        m = (at < 0 || at >= p.slots) ? 0 : clampi(m, 0, p.cap);
        koff = (long long)at * p.ssk;
        voff = (long long)at * p.ssv;
    } else {
        m = (at < 0 || at >= p.slots) ? 0 : clampi(m, 0, p.slots - at);
        koff = (long long)at * p.ldk;
        voff = (long long)at * p.ldv;
    }
    if (m == 0) koff = voff = 0;
    return m;
}

template <int DT>
__global__ __launch_bounds__(256) void attn_row_kernel(DeftAttn p) {
    typedef typename Elem<DT>::T T;
    constexpr int V = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    __shared__ float qs[4][128];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long unit = (long long)blockIdx.x * 4 + wave;
    const int t = (int)(unit / p.Hq), h = (int)(unit - (long long)t * p.Hq);
    const int b = t < p.Tq ? seq_of(p, t) : -1;
    const bool live = b >= 0;
    if (live)
        for (int d = lane; d < p.D; d += 64) qs[wave][d] = (float)((const T*)p.q)[(long long)t * p.ldq + (long long)h * p.hsq + d];
    __syncthreads();
    if (!live) return;
    const int q0 = clampi(p.q_start[b], 0, p.Tq), q1 = clampi(p.q_start[b + 1], 0, p.Tq);
    if (t >= q1) return;
    long long koff, voff;
    const int m = keys_of(p, b, q1 - q0, koff, voff);
    const int hk = h / (p.Hq / p.Hk);
    const int vis = p.causal ? clampi(m - (q1 - q0) + (t - q0) + 1, 0, m) : m;
    const T* kp = (const T*)p.k + koff + (long long)hk * p.hsk;
    const T* vp = (const T*)p.v + voff + (long long)hk * p.hsv;
    float M = -INFINITY, L = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j0 = 0; j0 < vis; j0 += 64) {
        const int j = j0 + lane;
        float s = -INFINITY;
        if (j < vis) {
            const T* kr = kp + (long long)j * p.ldk;
            float a = 0.f;
            for (int d = 0; d < p.D; d += V) {
                const vec x = *(const vec*)(kr + d);
                for (int e = 0; e < V; ++e) a = fmaf((float)x[e], qs[wave][d + e], a);
            }
            s = a * p.scale;
        }
        float mx = s;
        for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
        const float Mn = fmaxf(M, mx), ref = Mn == -INFINITY ? 0.f : Mn;
        const float al = expf(M - ref), pj = expf(s - ref);
        float sum = pj;
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        L = L * al + sum;
        o0 *= al;
        o1 *= al;
        M = Mn;
        const int nj = vis - j0 < 64 ? vis - j0 : 64;
        for (int i = 0; i < nj; ++i) {
            const float w = __shfl(pj, i);
            const T* vr = vp + (long long)(j0 + i) * p.ldv;
            if (lane < p.D) o0 = fmaf(w, (float)vr[lane], o0);
            if (lane + 64 < p.D) o1 = fmaf(w, (float)vr[lane + 64], o1);
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* op = (T*)p.o + (long long)t * p.ldo + (long long)h * p.hso;
    if (lane < p.D) op[lane] = (T)(o0 * inv);
    if (lane + 64 < p.D) op[lane + 64] = (T)(o1 * inv);
    if (p.lse && lane == 0) p.lse[(long long)t * p.Hq + h] = M + logf(L);
}

bool in_fits(long long ld, long long hs, int V) { return ld % V == 0 && hs % V == 0 && ld >= 0 && hs >= 0; }

int attn_check(const DeftAttn* d) {
    DEFT_CHECK(d && d->q && d->o && d->q_start && ((d->k && d->v) || d->slots == 0), -130, "deft_attn: null pointer");
    DEFT_CHECK(d->dtype == DEFT_F32 || d->dtype == DEFT_F16 || d->dtype == DEFT_BF16, -131, "deft_attn: dtype=%d", d->dtype);
    DEFT_CHECK(d->D == 32 || d->D == 64 || d->D == 96 || d->D == 128, -132, "deft_attn: D=%d (32, 64, 96 or 128)", d->D);
    DEFT_CHECK(d->Hk > 0 && d->Hq > 0 && d->Hq % d->Hk == 0 && d->Hq <= 4096, -133, "deft_attn: Hq=%d is not a multiple of Hk=%d", d->Hq, d->Hk);
    DEFT_CHECK(d->Tq >= 0 && d->B >= 0 && d->slots >= 0 && d->cap >= 0, -134, "deft_attn: Tq=%d B=%d slots=%d cap=%d", d->Tq, d->B, d->slots, d->cap);
    DEFT_CHECK((long long)d->Tq * d->Hq < (1ll << 31) && (long long)d->B * d->Hk < (1ll << 31), -134, "deft_attn: Tq * Hq must stay below 2^31");
    DEFT_CHECK(d->cap == 0 || (d->k_start && d->k_len), -135, "deft_attn: a cache (cap=%d) needs k_start (slots) and k_len", d->cap);
    const int V = d->dtype == DEFT_F32 ? 4 : 8;
    DEFT_CHECK((((size_t)d->q | (size_t)d->k | (size_t)d->v | (size_t)d->o) & 15) == 0, -136, "deft_attn: pointers must be 16-byte aligned");
    DEFT_CHECK(in_fits(d->ldq, d->hsq, V) && in_fits(d->ldk, d->hsk, V) && in_fits(d->ldv, d->hsv, V) && in_fits(d->ldo, d->hso, V) &&
                   in_fits(d->ssk, d->ssv, V) && (d->Tq <= 1 || d->ldo >= d->D) && (d->Hq <= 1 || d->hso >= d->D),
               -137, "deft_attn: strides must be multiples of %d elements, and the rows of o apart", V);
    DEFT_CHECK(d->ldk <= (1 << 22) && d->ldv <= (1 << 22), -137, "deft_attn: ldk=%lld ldv=%lld (at most 2^22 elements between tokens)", d->ldk, d->ldv);
    return 0;
}

}  // namespace

extern "C" long long deft_attn_ws_floats(const DeftAttn* d) {
    const int rc = attn_check(d);
    return rc < 0 ? rc : 0;
}

extern "C" int deft_attn(const DeftAttn* d, void* stream) {
    const int rc = attn_check(d);
    if (rc < 0) return rc;
    if (d->Tq == 0 || d->B == 0) return 0;
    const unsigned grid = (unsigned)(((long long)d->Tq * d->Hq + 3) / 4);
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == DEFT_F32) hipLaunchKernelGGL((attn_row_kernel<DEFT_F32>), dim3(grid), dim3(256), 0, s, *d);
    else if (d->dtype == DEFT_F16) hipLaunchKernelGGL((attn_row_kernel<DEFT_F16>), dim3(grid), dim3(256), 0, s, *d);
    else hipLaunchKernelGGL((attn_row_kernel<DEFT_BF16>), dim3(grid), dim3(256), 0, s, *d);
    DEFT_CHECK_LAUNCH("attn");
    return 0;
}
