// Attention over packed sequences of different lengths with grouped heads (DeftAttn, include/deft_hip.h).
//
//   s_j = scale * q . k_j over the keys a row sees,   o = sum_j e^(s_j - M) v_j / sum_j e^(s_j - M)
//
// One pass over the keys: the reference M and both sums are carried along and rescaled when a larger score comes.  A "row" is one (query, head) pair;
// the G = Hq / Hk heads of a group are rows of the same tile (row r = query r / G, head r % G of the group), so keys and values are read once for
// the group and a single token still fills G rows.
//
// A wave works on 32 rows with S^T = K Q^T and O^T = V^T P^T (32 x 32 matrix instructions): a lane then owns ONE row (column l & 31) of both, maxima
// and sums stay inside the lane, and the accumulator of S^T is already laid out as the operand of P^T -- the keys of a 16-key step are merely
// taken in the order the accumulator holds them, 16 s + 8 (i >> 2) + 4 (l >> 5) + (i & 3), and V's fragments are read in that order too.  P never
// leaves the registers.  16-bit types: v_mfma_f32_32x32x16, V^T through the transposing LDS read; fp32: v_mfma_f32_32x32x2_f32, exact products.
//
// The reference M moves only when a score exceeds it by 2^8 (P <= 2^8 then, harmless in fp32 sums and in 16-bit P): the rescaling of O and the
// exchange between the two half-waves of a row run on few tiles instead of on all.  fp16 keeps P at 2^6 times its value, so that small
// probabilities stay out of the subnormals.
//
// 16-bit types round each probability for the matrix instruction; their sum takes the unrounded ones.  The step kernel gives the products the rounded part
// AND the rest (P to 2^-16 or better; twice the products with V): its keys' bytes are the cost, and this costs little there (24 x 32000 keys: 352.8 -> 353.8
// us, 256 x 500 64.2 -> 65.1, 2000 histories of up to 50 71.5 -> 73.4).  The prompt kernel keeps the rounded part alone, half a step relative and averaged
// over the keys: with the rest one 16384-token sequence takes 1367 us instead of 1008, six ragged ones 172 instead of 120.  Its results are off by 1.2 to 1.4
// times what rounding the output alone would leave.
//
// Two kernels:
//   attn_prompt_kernel: 128 rows (4 waves x 32), key tiles shared by the waves, double-buffered in LDS by DMA.
//   attn_step_kernel:   32 rows, one wave or four; the waves take different key tiles, each with one or two LDS stages of its own, joined at the end: single
//                       tokens over long histories, where the keys' bytes are the cost, and short histories.
// Both can split the keys over workgroups (partial O, M, L in the workspace, attn_merge_kernel joins them in order).
//
// Measured (one MI355X, a call among others): one 16384-token sequence, 16 heads over 4 of 128, bf16, causal: 1.01 - 1.07 ms, 1030 - 1090 TFLOP/s -- MFMA busy
// 59 % and VALU 51 % of the cycles, the two of them share the clock the card holds; D = 64: 905 TFLOP/s (8 heads, 16384), VALU-bound (an exponential is
// a quarter-rate instruction a score); 24 single tokens over 2000 .. 32000 keys, 32 heads over 8 of 128, bf16: 358 us, 5.25 TB/s of keys and values.
#include "common.h"

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef deft_f32x16 f32x16;

#ifndef DEFT_LDS_TR_HOOK       /* the unit-test SIMT emulator pre-defines these hooks */
// LDS-DMA of 16 bytes a lane (common.h deft_buffer_load_lds_x4), written out: after the builtin the compiler waits for ALL of a wave's DMA (vmcnt 0)
// before every transposing LDS read, the next tile's included, and the two-stage loops would not overlap anything.  Nothing is returned to a
// register; the kernels wait for their pieces themselves.  (One wait state between the write of m0 and its use.)
typedef u32x4 lds_src;
typedef unsigned lds_at;
__device__ __forceinline__ lds_at lds_address(char* lds) { return (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds; }
// `bytes` from `base` on may be read, chunks behind them arrive as zeros
__device__ __forceinline__ lds_src lds_source(const char* base, unsigned bytes) {
    const unsigned long long a = (unsigned long long)base;
    lds_src s = {(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)),
                 (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
    asm volatile("s_nop 4" : "+s"(s));               // (five wait states from a vector write of a scalar register to a memory instruction that reads it)
    return s;
}
__device__ __forceinline__ void lds_fetch(const lds_src& s, lds_at lds, unsigned off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(s) : "memory", "m0");
}
// transposing LDS read: the 16 lanes of a group address the rows (i >> 2) x 4-element chunks (i & 3) of a 4 x 16 block; lane i gets column i
__device__ __forceinline__ s16x4 deft_lds_read_tr16(const void* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(size_t)(__attribute__((address_space(3))) const void*)p);
}
__device__ __forceinline__ float deft_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float deft_log2(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ unsigned long long deft_ballot(bool b) { return __ballot(b); }
#endif

template <int DT> struct Elem;
template <> struct Elem<DEFT_F32> { typedef float T; };
template <> struct Elem<DEFT_F16> { typedef _Float16 T; };
template <> struct Elem<DEFT_BF16> { typedef __bf16 T; };

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float M_SLACK = 8.f;
// The reference M of a row starts at -2^24 and is good up to 2^24 (in log2): there s sc - M is one fma, and what M's own rounding takes off, the same for
// every key of the row, is at most a factor of two.  A row whose scores lie beyond, on either side, has its pass run again with FAR, where scores are
// rounded before the difference is taken and kept in HALF log2 units: a finite score then has a finite exponent whatever its size.  M leaves every
// pass in half units (L = 0: M_LEAST).
constexpr float M_NONE = -16777216.f, M_FAR = 16777216.f, M_LEAST = -3.4028234664e38f;
enum { BAD_VALUES = 1, FAR = 2 };             // why a pass is run again

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// What a workgroup works on: sequence b, its query rows and keys, and the tile's rows.
struct Work {
    int hk, split;
    int q0, n, m;                 // first query, queries, keys
    int row0, rows;               // first row of the tile, rows of the sequence (n * G)
    int qi, rem;                  // row0 = qi * G + rem
    const char *k, *v;            // key 0 / value 0 of this kv head
};
// The launch grid: x = kv head + Hk * split (neighbouring workgroups, on different XCDs, read different heads), y and z the flat tiles.
struct Grid { int nsplit, ntiles, piece; unsigned inv_g, inv_hk; };      // piece: see split_tiles; inv: 2^32 / n + 1, for quotients of small numbers (div_small)
// x / n for x < 2^19, n <= 4096: inv n = 2^32 + e with 0 < e <= n, and x e < 2^32
__device__ __forceinline__ int div_small(int x, unsigned inv) { return inv == 0 ? x : (int)__umulhi((unsigned)x, inv); }      // (inv = 0: n = 1)

// Flat tile t -> (sequence, tile of it).  Sequence b starts at flat tile  first(b) = q_start[b] * G / BM + b,  which leaves it at least ceil(n G / BM)
// tiles whatever the lengths are: no table of lengths is needed on the host, surplus tiles end at once.
template <int BM>
__device__ __forceinline__ bool find_work(const DeftAttn& p, int tsize, const Grid& g, Work& w) {
    const int G = p.Hq / p.Hk, lane = threadIdx.x & 63;
    w.split = g.nsplit == 1 ? 0 : div_small((int)blockIdx.x, g.inv_hk);
    w.hk = (int)blockIdx.x - w.split * p.Hk;
    const int t = g.ntiles - 1 - (int)(blockIdx.y + blockIdx.z * gridDim.y);         // causal: the long rows of a sequence first
    if (t < 0) return false;
    // the last b with first(b) <= t (first() grows): down to 448 candidates 64 at a time, then 8 loads a lane at once -- one trip to memory, which
    // brings q_start[b] and q_start[b + 1] as well
    auto start = [&](int at) { return clampi(p.q_start[at], 0, p.Tq); };
    auto before = [&](int q, int at) { return q * G / BM + at <= t; };               // (Tq * Hq < 2^30)
    int lo = 0, n = p.B;
    while (n > 448) {
        const int step = (n + 63) >> 6, at = lo + lane * step;
        const int c = __popcll(deft_ballot(at < lo + n && before(start(at), at)));
        if (c == 0) return false;
        const int left = n - (c - 1) * step;
        lo += (c - 1) * step;
        n = left < step ? left : step;
    }
    int c = 0, q0 = 0, q1 = 0;
    if (n < 64) {
        const int q = start(lo + (lane < n ? lane : n));
        c = __popcll(deft_ballot(lane < n && before(q, lo + lane)));
        if (c == 0) return false;
        q0 = __shfl(q, c - 1);
        q1 = __shfl(q, c);
    } else {
        int q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = start(lo + (i * 64 + lane < n ? i * 64 + lane : n));
#pragma unroll
        for (int i = 0; i < 8; ++i) c += __popcll(deft_ballot(i * 64 + lane < n && before(q[i], lo + i * 64 + lane)));
        if (c == 0) return false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int a = __shfl(q[i], (c - 1) & 63), b = __shfl(q[i], c & 63);
            q0 = (c - 1) >> 6 == i ? a : q0;
            q1 = c >> 6 == i ? b : q1;
        }
    }
    const int b = __builtin_amdgcn_readfirstlane(lo + c - 1);
    w.q0 = __builtin_amdgcn_readfirstlane(q0);
    w.n = __builtin_amdgcn_readfirstlane(q1) - w.q0;
    if (w.n <= 0) return false;
    w.rows = w.n * G;
    const int tile = t - (w.q0 * G / BM + b);
    if (tile < 0 || tile >= (w.rows + BM - 1) / BM) return false;                    // (negative: only where q_start does not grow)
    w.row0 = tile * BM;
    w.qi = G == 1 ? w.row0 : w.row0 / G;
    w.rem = w.row0 - w.qi * G;
    int m = p.k_len ? p.k_len[b] : w.n;
    const int at = p.k_start ? p.k_start[b] : w.q0;
    const bool there = at >= 0 && at < p.slots;
    m = there ? clampi(m, 0, p.cap > 0 ? p.cap : p.slots - at) : 0;
    w.m = m;
    const long long ko = m == 0 ? 0 : (long long)at * (p.cap > 0 ? p.ssk : p.ldk), vo = m == 0 ? 0 : (long long)at * (p.cap > 0 ? p.ssv : p.ldv);
    w.k = (const char*)p.k + (ko + (long long)w.hk * p.hsk) * tsize;
    w.v = (const char*)p.v + (vo + (long long)w.hk * p.hsv) * tsize;
    return true;
}
// keys (j < vis) that query i of the sequence sees
__device__ __forceinline__ int visible(const DeftAttn& p, const Work& w, int i) { return p.causal ? clampi(w.m - w.n + i + 1, 0, w.m) : w.m; }

// A tile of BN keys in LDS: rows of RB bytes, 16-byte chunks; chunk c of row r sits at slot c ^ f(r).
//   K is read 16 bytes a lane, 32 rows at one chunk (served in groups of 16 lanes): f spreads the 16 rows of such a group over the 16 slots of the
//   64 banks.  V of 16-bit types is read by the transposing read, 8 rows x 64 bytes: f_V moves the rows of a half-wave to different 64-byte
//   groups and the other half-wave's to the other 32 bytes.  V of fp32 is read a row at a time: no conflict to avoid.
template <int DT, int D>
struct Tile {
    typedef typename Elem<DT>::T T;
    static constexpr int TS = (int)sizeof(T), RB = D * TS, CPR = RB / 16, NF = CPR / 2, NJ = D / 32;
    static constexpr float SHIFT = DT == DEFT_F16 ? 6.f : 0.f;
    typedef T frag_t __attribute__((ext_vector_type(16 / TS)));

    static __device__ __forceinline__ int fk(int r) { return RB % 256 == 0 ? r & 15 : RB % 256 == 128 ? (r >> 1) & 7 : (r >> 2) & 3; }
    static __device__ __forceinline__ int fv(int r) {
        if (DT == DEFT_F32) return 0;
        const int two = ((r >> 2) & 1) << 1;
        return RB % 256 == 0 ? ((r & 3) << 2) | two : RB % 256 == 128 ? (((r >> 1) & 1) << 2) | two : two;
    }

    // Byte offsets (tile-relative) of the chunks this lane fetches; instruction j of the tile deposits 64 consecutive slots.
    // BN rows in BN * CPR / 64 instructions, instruction first + i * by for i < NI.
    template <int NI>
    struct Fetch {
        unsigned off[NI];
        template <typename F>
        __device__ __forceinline__ void init(int lane, int first, int by, long long ld, F f) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int s = (first + i * by) * 64 + lane, r = s / CPR, c = (s - r * CPR) ^ f(r);
                off[i] = (unsigned)(r * (int)ld) * (unsigned)TS + (unsigned)c * 16u;      // (ld <= 2^22, r < 64: below 2^31)
            }
        }
        // rows >= nv arrive as zeros: the range of the source ends with row nv - 1 (where the stride is below a row they may hold the rows in front)
        __device__ __forceinline__ void issue(const char* base, lds_at lds, int first, int by, int nv, int row_bytes) const {
            const lds_src r = lds_source(base, nv <= 0 ? 0u : nv >= 64 ? 0x7FFFFFFFu : (unsigned)((nv - 1) * row_bytes + RB));
#pragma unroll
            for (int i = 0; i < NI; ++i) lds_fetch(r, lds + (first + i * by) * 1024, off[i]);
        }
    };

    static __device__ __forceinline__ f32x16 zero16() {
        f32x16 z;
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = 0.f;
        return z;
    }
    static __device__ __forceinline__ f32x16 mfma(frag_t a, frag_t b, f32x16 c) {
        if constexpr (DT == DEFT_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
            return c;
        } else if constexpr (DT == DEFT_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }

    // State of a wave's 32 rows: lane l holds row l & 31 (both half-waves: half of the keys, half of O's columns)
    struct Rows {
        frag_t q[NF];                 // chunk 2 j + (l >> 5) of the row
        f32x16 o[NJ];                 // o[j][r]: column 32 j + 8 (r >> 2) + 4 (l >> 5) + (r & 3)
        float M, L;                   // scores are taken times scale * log2 e; P = 2^(s - M); L: this half-wave's part
        __device__ __forceinline__ void init(const T* qrow, int h) {
#pragma unroll
            for (int j = 0; j < NF; ++j) q[j] = *(const frag_t*)((const char*)qrow + (2 * j + h) * 16);
            clear(M_NONE);
            // (the loads end here: a wait for them inside the loop would wait for the tiles fetched ahead)
#pragma unroll
            for (int j = 0; j < NF; ++j) DEFT_OPAQUE(q[j]);
        }
        __device__ __forceinline__ void clear(float m) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[j] = zero16();
            M = m;
            L = 0.f;
        }
        // whether some row (that saw keys: `saw`) has scores the reference could not follow down to; NaN stays NaN
        __device__ __forceinline__ bool missed(bool saw) const { return deft_ballot(saw && M == M_NONE && L == L) != 0; }
        // whether some row's O holds an infinity or NaN that its scores do not explain: a value that is one has met a probability of 0 (a hidden key, a rest
        // of FINE) -- or is simply seen
        __device__ __forceinline__ bool odd() const {
            float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) z[r & 3] = fmaf(o[j][r], 0.f, z[r & 3]);
            const float s = (z[0] + z[1]) + (z[2] + z[3]);
            return deft_ballot(s != s && L == L) != 0;
        }
    };

    // One tile of BN = 32 NT keys for a wave: ks, vs the tile in LDS; vis: keys of the tile this lane's row sees (may be <= 0 or > BN); `partial`
    // (wave-uniform): some row does not see all of them.  Returns whether a score is beyond M_FAR (FAR).  The wave's result is not valid then, nor where
    // O is odd() at the end (BAD_VALUES): its pass is run again with CAREFUL -- with the same exponentials, or, `far`, in half log2 units (sc: scale *
    // log2 e, or half of that).  FINE: the products take the rest of a rounded probability, too.
    template <int NT, bool FINE, bool CAREFUL>
    static __device__ __forceinline__ int step(Rows& w, const char* ks, const char* vs, int vis, bool partial, float sc, int lane, bool far = false) {
        const bool half = CAREFUL && far;
        const float first = half ? sc : 1.f, then = half ? 1.f : sc, units = half ? 2.f : 1.f;       // (products with 1 change nothing)
        const int h = lane >> 5;
        f32x16 s[NT];
        {
            const int key = lane & 31;                                         // rows 32 t + key: f(32 t + key) = f(key)
            const int x = h ^ fk(key);
            const char* const kr = ks + key * RB;
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t] = zero16();
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int t = 0; t < NT; ++t) s[t] = mfma(*(const frag_t*)(kr + t * 32 * RB + (((2 * j) ^ x) << 4)), w.q[j], s[t]);
        }
        if (partial) {
            const int lim = vis - 4 * h;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[t][r] = 32 * t + 8 * (r >> 2) + (r & 3) < lim ? s[t][r] : -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if constexpr (CAREFUL) s[t][r] *= first;
                mx = t + r == 0 ? s[0][0] : fmaxf(mx, s[t][r]);
            }
        int bad = 0;
        if (deft_ballot(half ? (mx - w.M) * 2.f > SHIFT + M_SLACK : mx * sc > w.M + (SHIFT + M_SLACK)) != 0) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float Mn = fmaxf(w.M, half ? mx - SHIFT * 0.5f : mx * sc - SHIFT);
            const float al = deft_exp2(half ? (w.M - Mn) * 2.f : w.M - Mn);
            if constexpr (!CAREFUL) bad = deft_ballot(Mn > M_FAR) != 0 ? FAR : 0;
            w.M = Mn;
            w.L *= al;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) w.o[j][r] *= al;
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = deft_exp2(CAREFUL ? fmaf(s[t][r], then, -w.M) * units : fmaf(s[t][r], sc, -w.M));
                s[t][r] = e;
                sum[r & 3] += e;
            }
        w.L += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if constexpr (CAREFUL) {
            careful<NT, FINE>(w, s, vs, vis, lane);
            return 0;
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const pfrag_t p = probs(s[t], g), rest = FINE && DT != DEFT_F32 ? rest_of(s[t], g, p) : p;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        const pfrag_t v = value(vs, t, g, j, lane);
                        w.o[j] = pv(v, p, w.o[j]);
                        if constexpr (FINE && DT != DEFT_F32) w.o[j] = pv(v, rest, w.o[j]);
                    }
                }
            return bad;
        }
    }

    // ---- the products with V, 16 / TS keys a half-wave at a time: group g of a 32-key block holds the accumulator registers GK g .. GK g + GK - 1
    static constexpr int GK = DT == DEFT_F32 ? 4 : 8, NG = 16 / GK;
    typedef T pfrag_t __attribute__((ext_vector_type(GK)));
    static __device__ __forceinline__ pfrag_t probs(const f32x16& s, int g) {
        pfrag_t p;
#pragma unroll
        for (int e = 0; e < GK; ++e) p[e] = (T)s[GK * g + e];
        return p;
    }
    static __device__ __forceinline__ pfrag_t rest_of(const f32x16& s, int g, pfrag_t p) {
        pfrag_t q;
#pragma unroll
        for (int e = 0; e < GK; ++e) q[e] = (T)(s[GK * g + e] - (float)p[e]);
        return q;
    }
    // this lane's fragment of V^T: column 32 j + (l & 31), the keys of probs() of group g of block t
    static __device__ __forceinline__ pfrag_t value(const char* vs, int t, int g, int j, int lane) {
        const int h = lane >> 5;
        if constexpr (DT == DEFT_F32) {
            pfrag_t v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *(const float*)(vs + (32 * t + 8 * g + 4 * h + e) * RB + (32 * j + (lane & 31)) * 4);
            return v;
        } else {
            const int i = lane & 15, row = 4 * h + (i >> 2), c0 = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
            const char* const a = vs + row * RB + (i & 1) * 8 + (32 * t + 16 * g) * RB + (((4 * j + c0) ^ fv(row)) << 4);      // f(row + 8 x) = f(row)
            return __builtin_bit_cast(pfrag_t, __builtin_shufflevector(deft_lds_read_tr16(a), deft_lds_read_tr16(a + 8 * RB), 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    static __device__ __forceinline__ f32x16 pv(pfrag_t v, pfrag_t p, f32x16 o) {
        if constexpr (DT == DEFT_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e], p[e], o, 0, 0, 0);
            return o;
        } else return mfma(v, p, o);
    }
    // Products for tiles with infinities or NaN among values that not every row may see (0 * inf is NaN in a product): the finite values with P,
    // then, with P replaced by what is visible, how many +inf / NaN and how many -inf / NaN each row sees -- what is seen is added.
    template <int NT, bool FINE>
    static __device__ __forceinline__ void careful(Rows& w, f32x16 (&s)[NT], const char* vs, int vis, int lane) {
        const int lim = vis - 4 * (lane >> 5);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const pfrag_t p = probs(s[t], g), rest = FINE && DT != DEFT_F32 ? rest_of(s[t], g, p) : p;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    __builtin_amdgcn_sched_barrier(0);
                    pfrag_t v = value(vs, t, g, j, lane);
#pragma unroll
                    for (int e = 0; e < GK; ++e) v[e] = (float)v[e] - (float)v[e] == 0.f ? v[e] : (T)0.f;
                    w.o[j] = pv(v, p, w.o[j]);
                    if constexpr (FINE && DT != DEFT_F32) w.o[j] = pv(v, rest, w.o[j]);
                }
            }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = 32 * t + 8 * (r >> 2) + (r & 3) < lim ? 1.f : 0.f;
#pragma unroll 1
        for (float sign = 1.f; sign >= -1.f; sign -= 2.f) {
            int l = lane;
            DEFT_OPAQUE_NV(l);                                       // (no fragment is kept over the two passes: registers)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                f32x16 acc = zero16();
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        __builtin_amdgcn_sched_barrier(0);           // (nor fetched ahead)
                        pfrag_t v = value(vs, t, g, j, l);
#pragma unroll
                        for (int e = 0; e < GK; ++e) v[e] = (float)v[e] * sign <= 3.4028235e38f ? (T)0.f : (T)1.f;
                        acc = pv(v, probs(s[t], g), acc);
                    }
#pragma unroll
                for (int r = 0; r < 16; ++r) w.o[j][r] = acc[r] > 0.f ? w.o[j][r] + sign * INFINITY : w.o[j][r];
            }
        }
    }
};

// Key tiles a split takes: a fixed piece, 1 / nsplit of the longest sequence, so that the workgroups of long and short sequences take equally
// long (a short one's later splits have nothing to do); more where max_k was too low an estimate.
__device__ __forceinline__ int split_tiles(const Grid& g, int nt) {
    const int even = (nt + g.nsplit - 1) / g.nsplit;
    return even > g.piece ? even : g.piece;
}

// Where a split's partial results stand in the workspace: O [split][row][D], then (M, L) [split][row]; row = query * Hq + head
__device__ __forceinline__ size_t ws_row(const DeftAttn& p, int split, int query, int head) { return ((size_t)split * p.Tq + query) * p.Hq + head; }
__device__ __forceinline__ float* ws_ml(const DeftAttn& p, int nsplit) { return p.ws + (size_t)nsplit * p.Tq * p.Hq * p.D; }

// the log of a row's sum of exponentials from its M (half units) and L
__device__ __forceinline__ float log_sum(float M, float L) { return L == 0.f ? -INFINITY : (M + deft_log2(L) * 0.5f) * (2.f * LN2); }

// A wave's 32 rows to the output, or to the workspace where the keys are split: through its part of the LDS stages (32 rows, chunks swizzled like
// K's), so that rows leave as whole lines -- in the accumulators a lane holds 4 of every 8 columns of one row.
template <int DT, int D>
__device__ __forceinline__ void write_rows(const DeftAttn& p, const Work& w, typename Tile<DT, D>::Rows& rw, int nsplit, int query, int head, int nrows, int lane, char* part) {
    typedef Tile<DT, D> TL;
    typedef typename TL::T T;
    const int h = lane >> 5, l32 = lane & 31;
    rw.L += __shfl_xor(rw.L, 32);
    rw.M = rw.L == 0.f ? M_LEAST : rw.M;
    const bool there = l32 < nrows;
    const int at = query * p.Hq + head;                                            // (Tq * Hq < 2^30)
    if (nsplit > 1) {
        typedef Tile<DEFT_F32, D> TF;
        if (h == 0 && there) *(float2*)(ws_ml(p, nsplit) + ((size_t)w.split * p.Tq * p.Hq + at) * 2) = make_float2(rw.M, rw.L);
        if (deft_ballot(rw.L != 0.f) == 0) return;                                 // (no row saw a key of this split: nobody reads its O)
#pragma unroll
        for (int j = 0; j < TF::NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *(f32x4*)(part + l32 * TF::RB + (((8 * j + r / 2 + h) ^ TF::fk(l32)) << 4)) = f32x4{rw.o[j][r], rw.o[j][r + 1], rw.o[j][r + 2], rw.o[j][r + 3]};
        DEFT_WAVE_LGKM();
#pragma unroll
        for (int i = 0; i < TF::CPR / 2; ++i) {
            const int s = i * 64 + lane, r = s / TF::CPR, c = s - r * TF::CPR;
            const f32x4 x = *(const f32x4*)(part + r * TF::RB + ((c ^ TF::fk(r)) << 4));
            const int ar = __shfl(at, r);
            if (r < nrows) *(f32x4*)(p.ws + ((size_t)w.split * p.Tq * p.Hq + ar) * D + c * 4) = x;
        }
        return;
    }
    const float inv = rw.L == 0.f ? 0.f : 1.f / rw.L;
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int j = 0; j < TL::NJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            t4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (T)(rw.o[j][r + e] * inv);
            const int byte = (32 * j + 2 * r + 4 * h) * TL::TS;
            *(t4*)(part + l32 * TL::RB + (((byte >> 4) ^ TL::fk(l32)) << 4) + (byte & 15)) = x;
        }
    DEFT_WAVE_LGKM();
    if (p.lse && h == 0 && there) p.lse[at] = log_sum(rw.M, rw.L);
#pragma unroll
    for (int i = 0; i < TL::CPR / 2; ++i) {
        const int s = i * 64 + lane, r = s / TL::CPR, c = s - r * TL::CPR;
        const u32x4 x = *(const u32x4*)(part + r * TL::RB + ((c ^ TL::fk(r)) << 4));
        const int qr = __shfl(query, r), hr = __shfl(head, r);
        if (r < nrows) *(u32x4*)((char*)p.o + ((long long)qr * p.ldo + (long long)hr * p.hso) * TL::TS + c * 16) = x;
    }
}

constexpr int BM = 128;

template <int DT, int D>
__global__ __launch_bounds__(256, 2) void attn_prompt_kernel(DeftAttn p, Grid grid) {
    typedef Tile<DT, D> TL;
    typedef typename TL::T T;
    constexpr int NT = DT == DEFT_F32 ? 1 : 2, BN = 32 * NT, KB = BN * TL::RB, NI = BN * TL::CPR / 256;
    static_assert(NI * 256 == BN * TL::CPR, "whole DMA instructions");
    __shared__ __attribute__((aligned(1024))) char lds[4 * KB];                    // K and V of two stages (three were no faster: 124 -> 127 us, D = 64)
    __shared__ int again, far;
    const int G = p.Hq / p.Hk, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    Work w;
    if (!find_work<BM>(p, TL::TS, grid, w)) return;
    const int nsplit = grid.nsplit;
    const float sc = p.scale * LOG2E, half_sc = p.scale * (LOG2E * 0.5f);
    const int left = w.rows - w.row0 - 1, wr0 = wave * 32;                         // the tile's last row, the wave's first
    const bool on = wr0 <= left;                                                   // this wave has rows
    auto query_of = [&](int r) { return w.qi + div_small(w.rem + (r < left ? r : left), grid.inv_g); };      // of row r of the tile (the last one's behind it)
    const int rc = wr0 + (lane & 31) < left ? wr0 + (lane & 31) : left, qi = query_of(rc), query = w.q0 + qi;
    const int head = w.hk * G + w.rem + rc - (qi - w.qi) * G;
    const int vis = visible(p, w, qi);
    const int vmin = visible(p, w, query_of(wr0)), vmax = visible(p, w, query_of(wr0 + 31));                  // the wave's first and last row
    const int bmax = visible(p, w, query_of(BM - 1));
    const int nt = (bmax + BN - 1) / BN, per = split_tiles(grid, nt);
    const int t0 = w.split * per, t1 = t0 + per < nt ? t0 + per : nt;

    typename TL::template Fetch<NI> fk, fv;
    fk.init(lane, wave, 4, p.ldk, [](int r) { return TL::fk(r); });
    fv.init(lane, wave, 4, p.ldv, [](int r) { return TL::fv(r); });
    const int kr = (int)p.ldk * TL::TS, vr = (int)p.ldv * TL::TS;                  // bytes between keys (<= 2^24)
    const lds_at base = lds_address(lds);
    auto issue = [&](int t, int st) {
        const int nv = w.m - t * BN;
        fk.issue(w.k + (long long)t * BN * kr, base + st * 2 * KB, wave, 4, nv, kr);
        fv.issue(w.v + (long long)t * BN * vr, base + st * 2 * KB + KB, wave, 4, nv, vr);
    };
    if (tid == 0) again = far = 0;
    if (t0 < t1) issue(t0, 0);
    typename TL::Rows rw;                                                          // (its loads and the first tile's are one trip to memory)
    rw.init((const T*)p.q + (long long)query * p.ldq + (long long)head * p.hsq, h);
    int st = 0;
    for (int t = t0; t < t1; ++t, st ^= 1) {
        DEFT_PIPE_BARRIER(0);                                                      // tile t is here, and nobody reads tile t - 1 any more
        if (t + 1 < t1) issue(t + 1, st ^ 1);
        const int k0 = t * BN;
        const char* const ks = lds + st * 2 * KB;
        if (on && k0 < vmax) {
            if (TL::template step<NT, false, false>(rw, ks, ks + KB, vis - k0, vmin < k0 + BN, sc, lane)) far = 1;
        }
    }
    if (rw.missed(on && t0 < t1 && vis > t0 * BN)) far = 1;
    if (rw.odd()) again = 1;
    __syncthreads();
    const bool half = far != 0;
    if (again || half) {                                                           // (rare: infinities or NaN among the values, far scores)
        rw.clear(half ? M_LEAST : M_NONE);
        for (int t = t0; t < t1; ++t) {
            issue(t, 0);
            DEFT_PIPE_BARRIER(0);
            if (on && t * BN < vmax) TL::template step<NT, false, true>(rw, lds, lds + KB, vis - t * BN, true, half ? half_sc : sc, lane, half);
            __syncthreads();
        }
    }
    if (!half) rw.M *= 0.5f;
    write_rows<DT, D>(p, w, rw, nsplit, query, head, left + 1 - wr0, lane, lds + wave * KB);
}

template <int DT, int D, int NW>
__global__ __launch_bounds__(64 * NW, DT == DEFT_F32 ? (D <= 64 ? 4 : 1) : D <= 64 ? 3 : 2) void attn_step_kernel(DeftAttn p, Grid grid) {
    typedef Tile<DT, D> TL;
    typedef typename TL::T T;
    // One wave: one stage -- twice the workgroups on a compute unit are worth more than the overlap (500 fp32 histories of up to 50: 20.5 us against
    // 23.5 with two).  Four: two stages where they fit 128 KB; fp32 of D = 96, 128 takes one for the fourth wave (its matrix products are the cost).
    constexpr int NS = NW == 1 || TL::RB > 256 ? 1 : 2, KB = 32 * TL::RB, WB = NS * 2 * KB, NI = TL::CPR / 2;
    static_assert(WB >= 32 * D * 4, "a wave's rows fit its stages");
    __shared__ __attribute__((aligned(1024))) char lds[NW * WB];                // per wave: K, V of stage 0, K, V of stage 1
    __shared__ float ms[NW][32], ls[NW][32];
    const int G = p.Hq / p.Hk, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l32 = lane & 31;
    Work w;
    if (!find_work<32>(p, TL::TS, grid, w)) return;
    const int nsplit = grid.nsplit;
    const float sc = p.scale * LOG2E, half_sc = p.scale * (LOG2E * 0.5f);
    const int left = w.rows - w.row0 - 1;                                          // the tile's last row
    auto query_of = [&](int r) { return w.qi + div_small(w.rem + (r < left ? r : left), grid.inv_g); };      // of row r of the tile (the last one's behind it)
    const int rc = l32 < left ? l32 : left, qi = query_of(rc), query = w.q0 + qi, head = w.hk * G + w.rem + rc - (qi - w.qi) * G;
    const int vis = visible(p, w, qi), vmin = visible(p, w, w.qi), vmax = visible(p, w, query_of(31));
    const int nt = (vmax + 31) >> 5, per = split_tiles(grid, nt);
    const int t0 = w.split * per, t1 = t0 + per < nt ? t0 + per : nt;

    typename TL::template Fetch<NI> fk, fv;
    fk.init(lane, 0, 1, p.ldk, [](int r) { return TL::fk(r); });
    fv.init(lane, 0, 1, p.ldv, [](int r) { return TL::fv(r); });
    char* const mine = lds + wave * WB;
    const int kr = (int)p.ldk * TL::TS, vr = (int)p.ldv * TL::TS;                  // bytes between keys (<= 2^24)
    const lds_at base = lds_address(mine);
    auto issue = [&](int t, int st) {
        const int nv = w.m - t * 32;
        fk.issue(w.k + 32ll * t * kr, base + st * 2 * KB, 0, 1, nv, kr);
        fv.issue(w.v + 32ll * t * vr, base + st * 2 * KB + KB, 0, 1, nv, vr);
    };
    int st = 0, again = 0;
    if (t0 + wave < t1) issue(t0 + wave, 0);
    typename TL::Rows rw;                                                          // (its loads and the first tile's are one trip to memory)
    rw.init((const T*)p.q + (long long)query * p.ldq + (long long)head * p.hsq, h);
    if (NS == 2 && t0 + wave + NW < t1) issue(t0 + wave + NW, 1);
    for (int t = t0 + wave; t < t1; t += NW, st ^= NS - 1) {
        if (NS == 2 && t + NW < t1) { DEFT_WAVE_VM(2 * NI); } else { DEFT_WAVE_VM(0); }       // this wave's tile t is here (the stages are its own: no barrier)
        const int k0 = t * 32;
        again |= TL::template step<1, true, false>(rw, mine + st * 2 * KB, mine + st * 2 * KB + KB, vis - k0, vmin < k0 + 32, sc, lane);
        if (t + NS * NW < t1) {
            DEFT_WAVE_LGKM();                                                      // its reads have returned: the stage may be filled again
            issue(t + NS * NW, st);
        }
    }
    if (rw.missed(t0 + wave < t1 && vis > (t0 + wave) * 32)) again |= FAR;
    if (rw.odd()) again |= BAD_VALUES;
    const bool half = (again & FAR) != 0;
    if (again) {                                                                   // (rare: infinities or NaN among the values, far scores)
        rw.clear(half ? M_LEAST : M_NONE);
        for (int t = t0 + wave; t < t1; t += NW) {
            DEFT_WAVE_LGKM();
            issue(t, 0);
            DEFT_WAVE_VM(0);
            TL::template step<1, true, true>(rw, mine, mine + KB, vis - t * 32, true, half ? half_sc : sc, lane, half);
        }
    }
    if (!half) rw.M *= 0.5f;
    if constexpr (NW == 1) {
        DEFT_WAVE_LGKM();
        write_rows<DT, D>(p, w, rw, nsplit, query, head, left + 1, lane, lds);
        return;
    }
    // join the waves: everybody's M and L, then O scaled to the common M, summed in wave order
    rw.L += __shfl_xor(rw.L, 32);
    rw.M = rw.L == 0.f ? M_LEAST : rw.M;
    if (h == 0) { ms[wave][l32] = rw.M; ls[wave][l32] = rw.L; }
    __syncthreads();
    float M = ms[0][l32];
#pragma unroll
    for (int i = 1; i < NW; ++i) M = fmaxf(M, ms[i][l32]);
    const float al = deft_exp2((rw.M - M) * 2.f);
    float* const os = (float*)lds;                                                 // [wave][column][32 rows]
#pragma unroll
    for (int j = 0; j < TL::NJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) os[(wave * D + 32 * j + 8 * (r >> 2) + 4 * h + (r & 3)) * 32 + l32] = rw.o[j][r] * al;
    __syncthreads();
    // thread: a row's chunk of 4 columns
    const int nrows = left < 31 ? left + 1 : 32;
    for (int it = tid; it < nrows * (D / 4); it += 64 * NW) {
        const int r = it / (D / 4), c = (it - r * (D / 4)) * 4;
        float Mr = ms[0][r];
#pragma unroll
        for (int i = 1; i < NW; ++i) Mr = fmaxf(Mr, ms[i][r]);
        float Lr = 0.f;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            Lr += ls[i][r] * deft_exp2((ms[i][r] - Mr) * 2.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += os[(i * D + c + e) * 32 + r];
        }
        const int iq = query_of(r), qr = w.q0 + iq, hd = w.hk * G + w.rem + r - (iq - w.qi) * G;
        if (nsplit > 1) {
            *(f32x4*)(p.ws + ws_row(p, w.split, qr, hd) * D + c) = x;
            if (c == 0) *(float2*)(ws_ml(p, nsplit) + ws_row(p, w.split, qr, hd) * 2) = make_float2(Mr, Lr);
        } else {
            const float inv = Lr == 0.f ? 0.f : 1.f / Lr;
            typedef T t4 __attribute__((ext_vector_type(4)));
            t4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (T)(x[e] * inv);
            *(t4*)((T*)p.o + (long long)qr * p.ldo + (long long)hd * p.hso + c) = y;
            if (p.lse && c == 0) p.lse[(long long)qr * p.Hq + hd] = log_sum(Mr, Lr);
        }
    }
}

// Joins the splits of a row, in order: one wave a row.  Rows of no sequence have no partials and are not written; neither is any row where the starts do
// not grow (rows between two of them may have no partials, or those of two sequences): each wave looks at all of them, 64 at a time -- few, the keys are
// split only where there are at most about a thousand tiles.
template <int DT>
__global__ __launch_bounds__(256) void attn_merge_kernel(DeftAttn p, int nsplit) {
    typedef typename Elem<DT>::T T;
    const int lane = threadIdx.x & 63;
    const unsigned row = blockIdx.x * 4 + (threadIdx.x >> 6);                      // (Tq * Hq < 2^30)
    const int q = (int)(row / (unsigned)p.Hq), h = (int)(row - (unsigned)q * (unsigned)p.Hq);
    if (q >= p.Tq) return;
    bool grow = true;
    for (int b = lane; b < p.B; b += 64) grow = grow && clampi(p.q_start[b], 0, p.Tq) <= clampi(p.q_start[b + 1], 0, p.Tq);
    if (deft_ballot(!grow || q < p.q_start[0] || q >= p.q_start[p.B]) != 0) return;
    // lane s: M and L of split s (at most 64); then the splits' rows, whose loads wait for nothing
    const float2 x = lane < nsplit ? *(const float2*)(ws_ml(p, nsplit) + ws_row(p, lane, q, h) * 2) : make_float2(M_LEAST, 0.f);
    float M = x.x;
    for (int i = 1; i < 64; i <<= 1) M = fmaxf(M, __shfl_xor(M, i));
    const float al = deft_exp2((x.x - M) * 2.f);
    float L = x.y * al, o0 = 0.f, o1 = 0.f;
    for (int i = 1; i < 64; i <<= 1) L += __shfl_xor(L, i);
    const int col = lane * 2 < p.D ? lane * 2 : 0;
    const unsigned long long some = deft_ballot(x.y != 0.f);                       // splits that saw keys of this row: the others have written no O
    const int first = some ? __builtin_ctzll(some) : 0;
    if (some)
        for (int s0 = 0; s0 < nsplit; s0 += 8) {                                   // eight rows in flight
            float2 y[8];
            float a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int s = (some >> ((s0 + i) & 63)) & 1 && s0 + i < 64 ? s0 + i : first;
                y[i] = *(const float2*)(p.ws + ws_row(p, s, q, h) * p.D + col);
                a[i] = __shfl(al, s);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool has = s0 + i < 64 && (some >> ((s0 + i) & 63)) & 1;
                o0 = has ? fmaf(y[i].x, a[i], o0) : o0;
                o1 = has ? fmaf(y[i].y, a[i], o1) : o1;
            }
        }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (lane * 2 < p.D) {
        T* const op = (T*)p.o + (long long)q * p.ldo + (long long)h * p.hso + lane * 2;
        typedef T t2 __attribute__((ext_vector_type(2)));
        const t2 y = {(T)(o0 * inv), (T)(o1 * inv)};
        *(t2*)op = y;
    }
    if (p.lse && lane == 0) p.lse[row] = log_sum(M, L);
}

bool in_fits(long long ld, long long hs, int V) { return ld % V == 0 && hs % V == 0 && ld >= 0 && hs >= 0; }

int attn_check(const DeftAttn* d) {
    DEFT_CHECK(d && d->q && d->o && d->q_start && ((d->k && d->v) || d->slots == 0), -130, "deft_attn: null pointer");
    DEFT_CHECK(d->dtype == DEFT_F32 || d->dtype == DEFT_F16 || d->dtype == DEFT_BF16, -131, "deft_attn: dtype=%d", d->dtype);
    DEFT_CHECK(d->D == 32 || d->D == 64 || d->D == 96 || d->D == 128, -132, "deft_attn: D=%d (32, 64, 96 or 128)", d->D);
    DEFT_CHECK(d->Hk > 0 && d->Hq > 0 && d->Hq % d->Hk == 0 && d->Hq <= 4096, -133, "deft_attn: Hq=%d is not a multiple of Hk=%d", d->Hq, d->Hk);
    DEFT_CHECK(d->Tq >= 0 && d->B >= 0 && d->slots >= 0 && d->slots <= (1 << 30) && d->cap >= 0 && d->cap <= (1 << 30), -134, "deft_attn: Tq=%d B=%d slots=%d cap=%d", d->Tq, d->B, d->slots, d->cap);
    DEFT_CHECK((long long)d->Tq * d->Hq < (1ll << 30) && (long long)d->B * d->Hk < (1ll << 24), -134, "deft_attn: Tq=%d x Hq=%d rows, B=%d (below 2^30, 2^24 / Hk)", d->Tq, d->Hq, d->B);
    DEFT_CHECK(d->cap == 0 || (d->k_start && d->k_len), -135, "deft_attn: a cache (cap=%d) needs k_start (slots) and k_len", d->cap);
    const int V = d->dtype == DEFT_F32 ? 4 : 8;
    DEFT_CHECK((((size_t)d->q | (size_t)d->k | (size_t)d->v | (size_t)d->o) & 15) == 0, -136, "deft_attn: pointers must be 16-byte aligned");
    DEFT_CHECK(in_fits(d->ldq, d->hsq, V) && in_fits(d->ldk, d->hsk, V) && in_fits(d->ldv, d->hsv, V) && in_fits(d->ldo, d->hso, V) &&
                   in_fits(d->ssk, d->ssv, V) && deft_rows_apart(d->ldo, d->hso, d->Tq, d->Hq, d->D),
               -137, "deft_attn: strides must be multiples of %d elements and keep the rows of o apart", V);
    DEFT_CHECK(d->ldk <= (1 << 22) && d->ldv <= (1 << 22), -137, "deft_attn: ldk=%lld ldv=%lld (at most 2^22 elements between tokens)", d->ldk, d->ldv);
    DEFT_CHECK(d->scale >= 0x1p-126f && d->scale <= 0x1p126f, -138, "deft_attn: scale=%g (2^-126 .. 2^126)", (double)d->scale);
    return 0;
}

// How a call runs: the kernel, its flat tiles, and over how many workgroups the keys of a tile are split.
struct Choice { bool step; int waves, nsplit, ntiles; };
Choice choose(const DeftAttn* d) {
    const int G = d->Hq / d->Hk;
    Choice c;
    // 32-row tiles where sequences have no more rows, or one or two key tiles (200 histories of up to 50, 4 heads a group: 12.6 us against 14.4 with
    // 128-row tiles; 100 of 40 .. 120: 68 against 17; 4000 x 4000, D = 128: 186 against 70).  max_k is an estimate -- the AVERAGE length, where keys are the
    // queries' own rows and the caller says nothing: one long sequence among short ones then runs on these tiles, too (8000 + 199 x 1 tokens, 16 / 4 heads
    // of 64, bf16: 258 us against 166 on the others; 3000 + 63 x 1: 82 against 44; fp32, 8 / 8 of 32: 395 against 539).  A choice by the longest length there could be would cost the batches
    // of short ones as much, and they are the usual ones (500 of 20 .. 64 tokens: 26.5 us against 34.7; fp32 26.2 against 47.1).
    c.step = (long long)d->Tq * G <= 32ll * d->B || d->max_k <= 64;
    const int bm = c.step ? 32 : BM;
    c.ntiles = d->Tq * G / bm + d->B;                              // (below 2^26 + 2^24)
    // rows that are there fill about this many workgroups (tiles x heads)
    const long long busy = ((long long)d->Tq * G / bm + (c.step ? d->B : d->B / 2 + 1)) * d->Hk;
    const bool f32 = d->dtype == DEFT_F32;                         // (its products take 8 times as long: shorter pieces)
    const int keys = c.step || f32 ? 256 : 512;                    // keys a split should have at least
    // one wave a row tile where the keys are one or two tiles, or where that already fills the chip (256 x 8 heads over 100 .. 500 keys, D = 128: 71 us
    // against 92 with four; 200 x 4 over 30 .. 120: 10.1 against 12.3; 256 x 4 over 500, D = 64: 22 against 21)
    c.waves = c.step && (d->max_k <= 64 || (busy >= 800 && d->max_k <= 512)) ? 1 : 4;
    // key pieces: step kernel up to 2048 workgroups (24 x 32000 keys: 360 us; up to 1024: 373, 4096: 369), prompt kernel 768 (300-token chunks: 42.7 us; 512:
    // 44.0, 1024: 46.8; 4000 x 4000: 58.9, 70, 76.9); pieces of 256 keys instead of 512 help fp32 (194 -> 182 us on chunks) and not the others (42.6 -> 48.7)
    long long want = (c.step ? 2048 : 768) / busy;
    const long long most = ((long long)d->max_k + keys - 1) / keys;
    if (want > most) want = most;
    if (want > 64) want = 64;
    c.nsplit = want < 1 ? 1 : (int)want;
    return c;
}

struct Launch { Choice c; Grid g; dim3 grid; hipStream_t s; };
template <int DT, int D>
void attn_launch(const DeftAttn& d, const Launch& l) {
    if (!l.c.step) hipLaunchKernelGGL((attn_prompt_kernel<DT, D>), l.grid, dim3(256), 0, l.s, d, l.g);
    else if (l.c.waves == 1) hipLaunchKernelGGL((attn_step_kernel<DT, D, 1>), l.grid, dim3(64), 0, l.s, d, l.g);
    else hipLaunchKernelGGL((attn_step_kernel<DT, D, 4>), l.grid, dim3(256), 0, l.s, d, l.g);
}
template <int DT>
void attn_launch_d(const DeftAttn& d, const Launch& l) {
    switch (d.D) {
        case 32: attn_launch<DT, 32>(d, l); break;
        case 64: attn_launch<DT, 64>(d, l); break;
        case 96: attn_launch<DT, 96>(d, l); break;
        default: attn_launch<DT, 128>(d, l);
    }
    if (l.g.nsplit > 1) {
        const unsigned mg = (unsigned)(((long long)d.Tq * d.Hq + 3) / 4);
        hipLaunchKernelGGL((attn_merge_kernel<DT>), dim3(mg), dim3(256), 0, l.s, d, l.g.nsplit);
    }
}
unsigned inverse(int n) { return n == 1 ? 0u : (unsigned)(0x100000000ull / (unsigned)n + 1); }

}  // namespace

extern "C" long long deft_attn_ws_floats(const DeftAttn* d) {
    const int rc = attn_check(d);
    if (rc < 0) return rc;
    if (d->Tq == 0 || d->B == 0) return 0;
    const Choice c = choose(d);
    return c.nsplit > 1 ? (long long)c.nsplit * d->Tq * d->Hq * (d->D + 2) : 0;
}

extern "C" int deft_attn(const DeftAttn* d, void* stream) {
    const int rc = attn_check(d);
    if (rc < 0) return rc;
    if (d->Tq == 0 || d->B == 0) return 0;
    const Choice c = choose(d);
    const long long need = c.nsplit > 1 ? (long long)c.nsplit * d->Tq * d->Hq * (d->D + 2) : 0;
    DEFT_CHECK(need == 0 || (d->ws && d->ws_floats >= need && ((size_t)d->ws & 15) == 0), -139, "deft_attn: workspace of %lld floats, 16-byte aligned, has %lld", need,
               d->ws ? d->ws_floats : 0ll);
    Launch l;
    l.c = c;
    const int bn = c.step || d->dtype == DEFT_F32 ? 32 : 64;       // keys of a tile
    l.g = Grid{c.nsplit, c.ntiles, c.nsplit == 1 ? 0 : deft_cdiv(((long long)d->max_k + bn - 1) / bn, c.nsplit), inverse(d->Hq / d->Hk), inverse(d->Hk)};
    const int y = c.ntiles < 32768 ? c.ntiles : 32768;
    l.grid = dim3((unsigned)(d->Hk * c.nsplit), (unsigned)y, (unsigned)((c.ntiles + y - 1) / y));
    l.s = (hipStream_t)stream;
    if (d->dtype == DEFT_F32) attn_launch_d<DEFT_F32>(*d, l);
    else if (d->dtype == DEFT_F16) attn_launch_d<DEFT_F16>(*d, l);
    else attn_launch_d<DEFT_BF16>(*d, l);
    DEFT_CHECK_LAUNCH("attn");
    return 0;
}
