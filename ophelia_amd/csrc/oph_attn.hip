// Cross attention, forward: oph_seq_attn_forward.
#include "oph_attn.h"
#include "../../include/ophelia_hip.h"

#include <math.h>

#include <algorithm>

namespace ophseq {

// Running softmax of one query column: m in units of log2, l the sum over this lane's half of the keys.
struct Soft { float m, l; };

// Scores of KT keys x 32 queries (rows x columns) -> probabilities in place; returns the factor by which earlier results shrink.
template <int N> __device__ __forceinline__ float soft_step(f32x16 (&S)[N], uint64_t bits, Soft& st, float c, int half) {
    constexpr uint64_t FULL = N == 2 ? ~0ull : 0xffffffffull;
    if (bits != FULL) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t b = (uint32_t)(bits >> (32 * n)) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) S[n][r] = (b >> (8 * (r / 4) + r % 4)) & 1 ? S[n][r] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[n][r]);
    mx = fmaxf(mx, other_half(mx));
    // The reference point moves only when a score passes it by more than 2^8: probabilities stay below 256 (their relative precision is
    // the same), and results are rescaled a few times a row instead of at every new maximum.
    const float m = mx * c > st.m + 8.f ? mx * c : st.m;
    const float base = m == -INFINITY ? 0.f : m;       // a row without a finite score so far: every exponential below is 0
    const float shrink = exp2_(st.m - base);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            S[n][r] = exp2_(fmaf(S[n][r], c, -base));
            sum += S[n][r];
        }
    st.l = st.l * shrink + sum;
    st.m = m;
    return shrink;
}

// ---- many rows: a workgroup of 4 waves, 32 rows each, over all keys; key and value tiles in LDS for the four -------------------------
// waves a SIMD that the registers must leave room for: a second wave's products run under the first one's exponentials (4 x 16 heads
// of 4096 x 4096 x 128: 576 us with two waves, 970 with one; D = 64: three)
template <class T, int DP> constexpr int wide_waves() { return sizeof(T) == 4 || DP > 128 ? 1 : DP > 64 ? 2 : 3; }
template <class T, int DP, int KT>
__global__ __launch_bounds__(256, (wide_waves<T, DP>())) void attn_wide(const AttnP p) {
    constexpr int ROWS = 128, NK = KT / 32, TB = Tile<T, DP>::bytes(KT);
    __shared__ __attribute__((aligned(16))) char lds[4 * TB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
    const int M = p.Tq * p.G, tiles = (M + ROWS - 1) / ROWS;
    const Where w = where(p, on_xcd(p, blockIdx.x, tiles * p.B * p.Hk), tiles);
    const int r = w.tile * ROWS + wave * 32 + col, t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
    const float c = p.scale * LOG2E;

    const T* k = (const T*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const T* v = (const T*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    const bool any = row_time(p, w.tile * ROWS) < w.qlen;               // a tile of padding only: nothing to read
    const int nt = any ? (w.klen + KT - 1) / KT : 0;
    Stage<T, DP, KT, 256> sk, sv;
    const T *k1 = sk.own(k, p.ks[1], p.D, tid), *v1 = sv.own(v, p.vs[1], p.D, tid);
    uint64_t bits = 0;
    uint8_t byte = 0;
    auto fetch = [&](int j) {
        const int key0 = j * KT, last = w.klen - 1;
        byte = key_byte(p, w, key0, w.klen, lane);
        if (key0 + KT <= w.klen) {
            sk.load_run(k1, p.ks[1]);
            sv.load_run(v1, p.vs[1]);
            k1 += KT * p.ks[1];
            v1 += KT * p.vs[1];
            return;
        }
        sk.load([&](int i) { return k + (int64_t)min(key0 + i, last) * p.ks[1]; }, p.D, tid);
        sv.load([&](int i) { return v + (int64_t)min(key0 + i, last) * p.vs[1]; }, p.D, tid);
    };
    auto commit = [&](int j) {
        char* x = lds + (j & 1) * 2 * TB;
        bits = key_bits(byte, j * KT, w.klen, lane) & (KT == 64 ? ~0ull : 0xffffffffull);
        sk.store(x, bits, p.D, tid);
        sv.store(x + TB, bits, p.D, tid);
    };
    if (nt) fetch(0);                                    // on its way while the rows' operands are loaded

    frag_t<T> Q[DP / 16];
    f32x16 O[DP / 32];
    Soft st = {-INFINITY, 0.f};
    row_frags<T, DP>(Q, row_ptr<T>(p, p.q, w, r, p.qs[0], p.qs[1], p.qs[2]), p.D, r < M && t < w.qlen, half);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) O[d] = f32x16{};

    if (nt) commit(0);
    for (int j = 0; j < nt; ++j) {
        const uint64_t now = bits;
        __syncthreads();
        if (j + 1 < nt) fetch(j + 1);
        if (now) {
            const char *tk = lds + (j & 1) * 2 * TB, *tv = tk + TB;
            f32x16 S[NK];
#pragma unroll
            for (int i = 0; i < NK; ++i) S[i] = f32x16{};
#pragma unroll
            for (int s = 0; s < DP / 16; ++s)
#pragma unroll
                for (int i = 0; i < NK; ++i) S[i] = El<T>::mma(row_frag<T, DP>(tk, 32 * i, s, lane), Q[s], S[i]);
            const float shrink = soft_step<NK>(S, now, st, c, half);
            if (__any(shrink != 1.f)) {
#pragma unroll
                for (int d = 0; d < DP / 32; ++d) O[d] *= shrink;
            }
#pragma unroll
            for (int i = 0; i < NK; ++i)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const frag_t<T> P = next_frag<T>(S[i], s);
#pragma unroll
                    for (int d = 0; d < DP / 32; ++d) O[d] = El<T>::mma(trans_frag<T, DP>(tv, 32 * i + 16 * s, 32 * d, lane), P, O[d]);
                }
        }
        if (j + 1 < nt) commit(j + 1);
    }

    const float l = st.l + other_half(st.l);
    if (r < M) {
        const bool live = t < w.qlen && l != 0.f;                          // NaN stays NaN
        const float inv = live ? 1.f / l : 0.f;
        T* o = (T*)p.o0 + (((int64_t)w.b * p.Tq + t) * (p.Hk * p.G) + h) * p.D;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = 32 * d + 8 * g + 4 * half;
                const f32x4 x = {O[d][4 * g], O[d][4 * g + 1], O[d][4 * g + 2], O[d][4 * g + 3]};
                if (at < p.D) store4<T>(o + at, live ? x * inv : f32x4{0.f, 0.f, 0.f, 0.f});
            }
        if (half == 0) p.lse[((int64_t)w.b * (p.Hk * p.G) + h) * p.Tq + t] = live ? (st.m + log2f(l)) * LN2 : -INFINITY;
    }
}

// ---- some rows, 16 bits (fp32: attn16_forward): a workgroup of 4 waves shares 32 rows, every wave takes every fourth tile of 32 keys of its
// split; keys go straight to the matrix operand, values through a tile of the wave's own, for the transposed read.  With nsplit > 1
// the results of the splits meet in attn_join. ----
template <class T, int DP>
__global__ __launch_bounds__(256) void attn_split(const AttnP p) {
    constexpr int TB = Tile<T, DP>::bytes(32), JOIN = 4 * 32 * 36 * 4;
    __shared__ __attribute__((aligned(16))) char lds[4 * TB > JOIN ? 4 * TB : JOIN];
    __shared__ float ml[4][32][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, col = lane & 31;
    const int M = p.Tq * p.G, tiles = (M + 31) / 32;
    const int lin = on_xcd(p, blockIdx.x, tiles * p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, tiles);
    const int row0 = w.tile * 32;
    const float c = p.scale * LOG2E;
    const Span span = split_span(w.klen, 32, p.nsplit, split, row_time(p, row0) < w.qlen);
    const int kbeg = span.beg, kend = span.end;

    frag_t<T> Q[DP / 16];
    f32x16 O[DP / 32];
    Soft st = {-INFINITY, 0.f};
    {
        const int r = row0 + col;
        row_frags<T, DP>(Q, row_ptr<T>(p, p.q, w, r, p.qs[0], p.qs[1], p.qs[2]), p.D, r < M && row_time(p, r) < w.qlen, half);
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) O[d] = f32x16{};
    const T* k = (const T*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const T* v = (const T*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    for (int key0 = kbeg + wave * 32; key0 < kend; key0 += 128) {
        const uint8_t byte = key_byte(p, w, key0, kend, lane);
        frag_t<T> K[DP / 16];
        row_frags<T, DP>(K, k + (int64_t)min(key0 + col, kend - 1) * p.ks[1], p.D, true, half);
        f32x16 S[1] = {f32x16{}};
        char* tv = lds + wave * TB;
        Stage<T, DP, 32, 64> sv;
        sv.load([&](int r) { return v + (int64_t)min(key0 + r, kend - 1) * p.vs[1]; }, p.D, lane);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) S[0] = El<T>::mma(K[s], Q[s], S[0]);
        const uint64_t bits = key_bits(byte, key0, kend, lane) & 0xffffffffull;
        const float shrink = soft_step<1>(S, bits, st, c, half);
        if (__any(shrink != 1.f)) {
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) O[d] *= shrink;
        }
        wave_lds_fence();
        sv.store(tv, bits, p.D, lane);
        wave_lds_fence();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const frag_t<T> P = next_frag<T>(S[0], s);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) O[d] = El<T>::mma(trans_frag<T, DP>(tv, 16 * s, 32 * d, lane), P, O[d]);
        }
    }

    // the four waves' results: the common maximum, then 32 columns of D at a time through LDS, in the order of the waves
    const float lw = st.l + other_half(st.l);
    if (half == 0) { ml[wave][col][0] = st.m; ml[wave][col][1] = lw; }
    __syncthreads();
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, ml[i][col][0]);
    const float weight = exp2_(st.m - (m == -INFINITY ? 0.f : m));
    const int orow = tid >> 3, od = (tid & 7) * 4, r = row0 + orow;    // what this thread writes
    float om = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) om = fmaxf(om, ml[i][orow][0]);
#pragma unroll
    for (int i = 0; i < 4; ++i) l += ml[i][orow][1] * exp2_(ml[i][orow][0] - (om == -INFINITY ? 0.f : om));
    const int t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
    const bool live = r < M && t < w.qlen && l != 0.f;
    const float inv = live ? 1.f / l : 0.f;
    const int64_t unit = ((int64_t)(w.b * p.Hk + w.hk) * tiles + w.tile) * p.nsplit + split;
    float* x = (float*)lds;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
        __syncthreads();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 y = {O[d][4 * g], O[d][4 * g + 1], O[d][4 * g + 2], O[d][4 * g + 3]};
            *(f32x4*)(x + (wave * 32 + col) * 36 + 8 * g + 4 * half) = y * weight;
        }
        __syncthreads();
        f32x4 sum = *(const f32x4*)(x + orow * 36 + od);
#pragma unroll
        for (int i = 1; i < 4; ++i) sum += *(const f32x4*)(x + (i * 32 + orow) * 36 + od);
        const int at = 32 * d + od;
        if (r < M && at < p.D) {
            if (p.nsplit == 1)
                store4<T>((T*)p.o0 + (((int64_t)w.b * p.Tq + t) * (p.Hk * p.G) + h) * p.D + at, live ? sum * inv : f32x4{0.f, 0.f, 0.f, 0.f});
            else
                *(f32x4*)(p.part + (unit * 32 + orow) * DP + at) = sum;
        }
    }
    if ((tid & 7) == 0 && r < M) {
        if (p.nsplit == 1)
            p.lse[((int64_t)w.b * (p.Hk * p.G) + h) * p.Tq + t] = live ? (om + log2f(l)) * LN2 : -INFINITY;
        else {
            p.aux[(unit * 32 + orow) * 2] = om;
            p.aux[(unit * 32 + orow) * 2 + 1] = l;
        }
    }
}

// a workgroup per row: the splits' results (at most 256), weighted to their common maximum; DP/4 threads hold the columns of a split,
// the groups of threads take the splits in turn and are summed in their order
template <class T, int DP>
__global__ __launch_bounds__(256) void attn_join(const AttnP p) {
    constexpr int COLS = DP / 4, GROUPS = 256 / COLS;
    __shared__ float weight[256];
    __shared__ f32x4 sums[GROUPS][COLS];
    const int tid = threadIdx.x, lane = tid & 63, M = p.Tq * p.G, RT = unit_rows<T>(), tiles = (M + RT - 1) / RT;
    const int bh = blockIdx.x / M, r = blockIdx.x - bh * M;
    const int b = bh / p.Hk, hk = bh - b * p.Hk, t = row_time(p, r), h = hk * p.G + r - t * p.G;
    const int qlen = p.q_lens ? clampi(p.q_lens[b], 0, p.Tq) : p.Tq;
    const int64_t unit = ((int64_t)bh * tiles + r / RT) * p.nsplit;
    float m[4], l[4], top = -INFINITY;                                     // every wave for itself: splits lane, lane + 64, ...
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = lane + 64 * i;
        const float* at = p.aux + ((unit + min(s, p.nsplit - 1)) * RT + r % RT) * 2;
        m[i] = s < p.nsplit ? at[0] : -INFINITY;
        l[i] = s < p.nsplit ? at[1] : 0.f;
        top = fmaxf(top, m[i]);
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f = exp2_(m[i] - (top == -INFINITY ? 0.f : top));
        sum += l[i] * f;
        if (tid < 64) weight[lane + 64 * i] = f;
    }
#pragma unroll
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i);
    __syncthreads();
    const int g = tid / COLS, d = tid % COLS * 4;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = g; s < p.nsplit; s += GROUPS)
        if (d < p.D) o += *(const f32x4*)(p.part + ((unit + s) * RT + r % RT) * DP + d) * weight[s];
    sums[g][tid % COLS] = o;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) o += sums[i][tid];
    const bool live = t < qlen && sum != 0.f;
    const float inv = live ? 1.f / sum : 0.f;
    if (d < p.D) store4<T>((T*)p.o0 + (((int64_t)b * p.Tq + t) * (p.Hk * p.G) + h) * p.D + d, live ? o * inv : f32x4{0.f, 0.f, 0.f, 0.f});
    if (tid == 0) p.lse[((int64_t)b * (p.Hk * p.G) + h) * p.Tq + t] = live ? (top + log2f(sum)) * LN2 : -INFINITY;
}

// ---- host side --------------------------------------------------------------------------------------------------------------------
int attn_check(const oph_seq_attn* a, bool gradient) {
    if (!a) return fail(OPH_ERR_INVALID, "attention: no arguments");
    if (!type_bytes(a->dtype)) return fail(OPH_ERR_INVALID, "attention: dtype %d is not one of OPH_SEQ_*", a->dtype);
    if (a->B < 0 || a->Tq < 0 || a->Tk < 0) return fail(OPH_ERR_INVALID, "attention: negative size (B %d, Tq %d, Tk %d)", a->B, a->Tq, a->Tk);
    if (a->Hq < 1 || a->Hk < 1 || a->Hq % a->Hk) return fail(OPH_ERR_INVALID, "attention: %d query heads are not a multiple of %d key heads", a->Hq, a->Hk);
    if (a->D < 8 || a->D > 256 || a->D % 8) return fail(OPH_ERR_UNSUPPORTED, "attention: head size %d is not a multiple of 8 up to 256", a->D);
    if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(OPH_ERR_INVALID, "attention: scale %g is not positive and finite", (double)a->scale);
    // 32-bit row and workgroup numbers; the division by the group size is exact below the first bound
    if ((double)a->Tq * a->Hq / a->Hk * (a->Hq / a->Hk) > 2147483647.0 || (double)a->B * a->Hq * ((double)a->Tq + a->Tk + 64) > 4.0e9 || a->Tk > 2147483000 - 256 ||
        a->Tq > 2147483000 - 256 || (double)a->B * a->Hq > 1.0e7)
        return fail(OPH_ERR_UNSUPPORTED, "attention: too many rows (B %d, Tq %d, Tk %d, Hq %d)", a->B, a->Tq, a->Tk, a->Hq);
    // a launch has less than 2^32 threads: 256 for 128 rows or keys (fp32, D > 128: 16; 16 bits, D > 128: twice for keys), 512 for the few rows of
    // a head
    const int64_t heads = (int64_t)a->B * a->Hk, unit = gradient && a->dtype == OPH_SEQ_F32 && a->D > 128 ? 16 : 128;
    const int64_t rows = cdiv((int64_t)a->Tq * (a->Hq / a->Hk), unit), keys = gradient ? cdiv(a->Tk, unit) * (a->D > 128 && unit == 128 ? 2 : 1) : 0;
    if (std::max(std::max(rows, keys) * 256, (int64_t)512) * heads >= 1ll << 32)
        return fail(OPH_ERR_UNSUPPORTED, "attention: too many rows for one launch (B %d, Tq %d, Tk %d, Hq %d)", a->B, a->Tq, a->Tk, a->Hq);
    return OPH_OK;
}

AttnP attn_params(const oph_seq_attn* a) {
    AttnP p = {};
    p.q = a->q; p.k = a->k; p.v = a->v;
    p.q_lens = a->q_lens; p.k_lens = a->k_lens; p.mask = a->mask;
    for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; }
    p.ms[0] = a->mask_stride[0]; p.ms[1] = a->mask_stride[1];
    p.B = a->B; p.Tq = a->Tq; p.Tk = a->Tk; p.Hk = a->Hk; p.G = a->Hq / a->Hk; p.D = a->D;
    p.magic = p.G > 1 ? (unsigned)(((1ull << 32) + p.G - 1) / p.G) : 0;
    p.scale = a->scale;
    p.nsplit = 1;
    return p;
}

// Runs of 8 where lengths differ (8 sequences of up to 2000 x 2000, 16 heads of 128: 219 us, 272 with one run an XCD; their gradient 741 and
// 836); else, and for few rows, which share nothing, one run an XCD (a token over 8 x 16384 keys: 88 us, 94 dealt out singly).
int run_of(const oph_seq_attn* a, int64_t groups, bool few) {
    const int64_t run = groups / 8;
    return (int)(!few && (a->q_lens || a->k_lens) && run > 8 ? 8 : run);
}
static int pad_d(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

struct FwdPlan { bool few, wide; int nsplit, rows; int64_t units; };
static FwdPlan forward_plan(const oph_seq_attn* a) {
    const int64_t M = (int64_t)a->Tq * (a->Hq / a->Hk), heads = (int64_t)a->B * a->Hk;
    FwdPlan f;
    // without matrix instructions: 16 x 1 row over 150 keys x 256 fp32 7.7 us (29 on 32-row products), 8 x 8 heads x 4 rows over 1000 keys x 128
    // bf16 15.0 (18.9); 4 rows of D <= 64 lose (8 x 8 heads over 4000 keys 25.7 and 20.6), 4 rows of D > 128 do not fit the registers
    f.few = M <= 2 || (M <= 4 && a->D > 64 && a->D <= 128);
    // 128-row workgroups once they fill the CUs (fp32, 4 x 8 heads of 1024 x 1024 x 128: 158 us, 16-row units 254); below, units that
    // split the keys (16 sequences of 200 x 150 x 256: 18 and 58)
    f.wide = !f.few && cdiv(M, 128) * heads >= 256;
    f.rows = a->dtype == OPH_SEQ_F32 ? unit_rows<float>() : unit_rows<f16_t>();
    f.units = cdiv(M, f.rows) * heads;
    // 512 workgroups, 256 for fp32 with D > 128.  That is one round where a CU holds two (D <= 64) or, in the latter case, one; attn_split,
    // attn16_forward and most of attn_few take more than half of a CU's registers above D = 64, and 512 are two rounds of those.  And at least
    // 256 keys a split (fp32 128), since the join is a launch of its own: 16 x 200 rows over 150 keys x 64 bf16 take 7.0 us whole and 13.1 in two
    // splits, 2 x 4 heads of 100 rows over 600 keys x 128 fp32 14.7 in four and 18.3 in two.
    const int64_t fill = (a->dtype == OPH_SEQ_F32 && a->D > 128 ? 256 : 512) / (f.units > 0 ? f.units : 1);
    const int64_t most = a->Tk / (a->dtype == OPH_SEQ_F32 && !f.few ? 128 : 256);
    const int64_t n = fill < most ? fill : most;
    f.nsplit = f.wide ? 1 : (int)(n < 1 ? 1 : n > 256 ? 256 : n);
    return f;
}

int64_t attn_forward_workspace(const oph_seq_attn* a) {
    const FwdPlan f = forward_plan(a);
    return f.nsplit == 1 ? 0 : f.units * f.nsplit * f.rows * (pad_d(a->D) + 2) * (int64_t)sizeof(float);
}

template <class T, int DP, int KT> static int forward(const oph_seq_attn* a, const FwdPlan& f, AttnP& p, void* stream) {
    const int64_t M = (int64_t)p.Tq * p.G, heads = (int64_t)p.B * p.Hk, groups = f.wide ? cdiv(M, 128) * heads : f.units * f.nsplit;
    p.chunk = run_of(a, groups, f.few);
    if (f.wide) return launch<AttnP>(attn_wide<T, DP, KT>, dim3((unsigned)groups), 256, p, 0, stream);
    p.nsplit = f.nsplit;
    p.part = (float*)a->workspace;
    p.aux = p.part + f.units * f.nsplit * f.rows * DP;
    int rc;
    if (f.few) rc = attn_few_forward(p, a->dtype, groups, stream);
    else if constexpr (sizeof(T) == 4) rc = attn16_launch(p, groups, 0, stream);
    else rc = launch<AttnP>(attn_split<T, DP>, dim3((unsigned)groups), 256, p, 0, stream);
    if (rc) return rc;
    if (f.nsplit > 1) return launch<AttnP>(attn_join<T, DP>, dim3((unsigned)(M * heads)), 256, p, 0, stream);
    return OPH_OK;
}
template <class T> static int forward_d(const oph_seq_attn* a, const FwdPlan& f, AttnP& p, void* stream) {
    constexpr int KT = sizeof(T) == 2 ? 64 : 32;
    if (p.D <= 64) return forward<T, 64, 64>(a, f, p, stream);
    if (p.D <= 128) return forward<T, 128, KT>(a, f, p, stream);
    return forward<T, 256, 32>(a, f, p, stream);
}

}  // namespace ophseq

using namespace ophseq;
extern "C" {

int64_t oph_seq_attn_workspace(const oph_seq_attn* a, int gradient) {
    if (int rc = attn_check(a, gradient != 0)) return rc;
    if (!a->B || !a->Tq) return gradient && a->B && a->Tk ? attn_gradient_workspace(a) : 0;
    return gradient ? attn_gradient_workspace(a) : attn_forward_workspace(a);
}

int oph_seq_attn_forward(const oph_seq_attn* a, int device, void* stream) {
    if (int rc = attn_check(a, false)) return rc;
    if (!a->B || !a->Tq) return OPH_OK;
    if (!a->q || !a->out || !a->lse || (a->Tk && (!a->k || !a->v))) return fail(OPH_ERR_INVALID, "attention: q, k, v, out and lse must not be NULL");
    const int64_t need = attn_forward_workspace(a);
    if (need && (!a->workspace || (int64_t)a->workspace_bytes < need || ((uintptr_t)a->workspace & 15)))
        return fail(OPH_ERR_INVALID, "attention: the workspace must hold %lld bytes, 16-byte aligned", (long long)need);
    OnDevice on(device);
    if (on.status) return on.status;
    const FwdPlan f = forward_plan(a);
    AttnP p = attn_params(a);
    p.o0 = a->out;
    p.lse = a->lse;
    if (a->dtype == OPH_SEQ_F32) return forward_d<float>(a, f, p, stream);
    if (a->dtype == OPH_SEQ_BF16) return forward_d<bf16_t>(a, f, p, stream);
    return forward_d<f16_t>(a, f, p, stream);
}

}  // extern "C"
