// Gated linear recurrence h_t = a_t h_{t-1} + (1 - a_t) x_t, a = sigmoid(gate), and its gradient: oph_seq_recur_forward / _gradient.
//
// Every step is an affine map of the state, and maps compose: (A, B) then (A', B') is (A'A, A'B + B').  A workgroup owns 128 bytes of
// channels of one sequence and BLOCK steps of time: each thread runs its stretch of R steps from 0, the maps are composed over the
// 8 stretches of a wave by lane exchanges and over the waves through LDS, and the thread runs its stretch once more from the state
// it now knows.  The inputs stay in registers in between: one pass over memory, which is what bounds it.
//
// Blocks of one chain (sequence and channels) hand the state on through the workspace.  A block publishes its map as soon as it has it,
// and the state behind it once it knows that; to learn the state before it, it takes the nearest state among the WINDOW blocks before
// it (usually its neighbour's) and applies the maps from there on, one after the other: whichever it finds, the bits are those of the
// whole chain done in order.  Blocks are numbered in the order in which they start (a ticket), so that
// every block waits only for blocks that are running already, and those publish their maps without waiting for anything.
// A published word is its own flag: the workspace is filled with ones, which is a NaN that no result has (NaN is published as the
// canonical one), and words are written and read whole, past the caches that the XCDs do not share.
//
// Gradient, backwards in time with the map m_t = a_t (m_{t+1} + dh_t):  l_t = dh_t + m_{t+1}, dx = (1 - a) l, dgate = a (1 - a) (h_{t-1} - x) l.
// h_{t-1} - x has to come from a float32 state: where the state follows its input the two are nearly the same, and the half step (2^-9 of h in
// bfloat16) that the forward's result is rounded by would be all that is left of the difference.  In float32 the result is the state and
// is read; in 16 bits the states are formed again: a sequence of one block does so from the x and gate that it holds in registers, and for longer
// ones a pass of the forward's chain leaves the state before every stretch in the workspace, from which the stretch is run once more.  4 x
// 16384 x 1024 bf16: 126 us that pass, 208 the gradient; 120 and 288 with the states behind the blocks only, since composing the
// stretches again takes 250 registers; 200 in one pass from the rounded states, which cost dgate up to all of its digits.
#include "oph_seq.h"
#include "../../include/ophelia_hip.h"

#include <algorithm>

namespace ophseq {

struct RecurP {
    const void *x, *gate, *hin, *dh;
    const float *h0, *dh_last;
    void *h, *dx, *dgate;
    float *h_last, *dh0;
    const int* lens;
    int64_t xs[2], gs[2], hs[2], ds[2];
    unsigned long long* map;                                           // [chain][block][channel] {A, B}
    unsigned* state;                                                   // [chain][block][channel] state behind the block
    unsigned* ticket;
    float* stretch;                                                    // gradient in 16 bits: [chain][block][stretch][channel] state before it
    int B, T, C, blocks;
};
constexpr int R = 4, WINDOW = 16;                                      // steps of a stretch | maps taken at once
// Waves of a workgroup, and with them the steps of a block (8 stretches a wave).  Up to 256 steps are one block of 8 waves, with
// nothing to hand on (16 x 200 x 256 fp32: 6.9 us; as two blocks of 4 waves and the clearing launch 11.4).  Longer ones are
// blocks of 4 waves: more of them wait for memory side by side (4 x 16384 x 1024 bf16, forward, and gradient in one pass: 326 us; 8 waves 360,
// 16 waves 404).
constexpr int ONE = 8, MANY = 4;
constexpr int block_steps(int nw) { return nw * 8 * R; }

template <class T> struct Piece {                                     // 16 bytes of channels, `left` of the row's remain
    static constexpr int PER = El<T>::PER16;
    typedef T vec __attribute__((ext_vector_type(PER)));
    static __device__ __forceinline__ u32x4 load(const T* at, int left) {
        if (left >= PER) return load16(at);
        vec v;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = j < left ? at[j] : (T)0.f;
        return __builtin_bit_cast(u32x4, v);
    }
    static __device__ __forceinline__ void store(T* at, const float (&f)[PER], int left) {
        vec v;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = (T)f[j];
        if (left >= PER) store16(at, __builtin_bit_cast(u32x4, v));
        else
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (j < left) at[j] = v[j];
    }
    static __device__ __forceinline__ float at(u32x4 x, int j) { return (float)__builtin_bit_cast(vec, x)[j]; }
};

// sigmoid and 1 - sigmoid, each without cancellation: a state that is held for thousands of steps has 1 - a of 1e-4 and less
__device__ __forceinline__ void gate_of(float g, float& a, float& keep) {
    const float e = exp2_(-fabsf(g) * LOG2E), r = __builtin_amdgcn_rcpf(1.f + e);
    a = g >= 0.f ? r : e * r;
    keep = g >= 0.f ? e * r : r;
}

__device__ __forceinline__ unsigned word(float x) { return x != x ? 0x7fc00000u : __builtin_bit_cast(unsigned, x); }

template <int PER, int NW> struct Shared {
    static constexpr int CH = 8 * PER;
    float wave[NW][CH][2];                                               // maps of the waves' stretches
    float before[WINDOW][CH][2];                                         // what the blocks before have published: a map, or a state in [1]
    int kind[WINDOW];                                                    // 0 nothing there, 1 map, 2 state
    float carry[CH];
    unsigned ticket;
};

// which (chain, block) this workgroup is
template <int PER, int NW> __device__ __forceinline__ int2 place(const RecurP& p, int chains, Shared<PER, NW>& sh) {
    if (NW == ONE) return make_int2(blockIdx.x, 0);
    if (threadIdx.x == 0) sh.ticket = atomicAdd(p.ticket, 1u);
    __syncthreads();
    const int n = (int)sh.ticket, k = n / chains;
    return make_int2(n - k * chains, k);
}

// Maps (A, B) of this thread's stretch -> `in`, the state before the stretch; returns the state behind the block for channel
// threadIdx.x (of the first CH threads).  first: the state before block 0, for the same channel.  All threads call it.
template <int PER, int NW>
__device__ __forceinline__ float compose(const RecurP& p, float (&A)[PER], float (&B)[PER], float first, float (&in)[PER], int chain, int k, bool last,
                                         Shared<PER, NW>& sh) {
    constexpr int CH = 8 * PER;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, cg = (lane & 7) * PER;
#pragma unroll
    for (int off = 8; off < 64; off <<= 1)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float a = __shfl_up(A[j], off), b = __shfl_up(B[j], off);
            if (lane >= off) {
                B[j] = fmaf(A[j], b, B[j]);
                A[j] *= a;
            }
        }
    if (lane >= 56)
#pragma unroll
        for (int j = 0; j < PER; ++j) { sh.wave[wave][cg + j][0] = A[j]; sh.wave[wave][cg + j][1] = B[j]; }
    __syncthreads();
    const int64_t at = ((int64_t)chain * p.blocks + k) * CH;
    float a = 1.f, b = 0.f, carry = first, behind = 0.f;
    if (tid < CH)
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            a *= sh.wave[w][tid][0];
            b = fmaf(sh.wave[w][tid][0], b, sh.wave[w][tid][1]);
        }
    if (NW != ONE && k > 0) {
        if (!last && tid < CH)
            __hip_atomic_store(p.map + at + tid, (unsigned long long)word(a) | (unsigned long long)word(b) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (;;) {
            constexpr int PW = WINDOW / NW;
#pragma unroll
            for (int i = 0; i < PW; ++i) {                                // each wave waits for its blocks: one channel per lane
                const int slot = wave * PW + i, q = k - 1 - slot;
                int kind = 0;
                if (q >= 0) {
                    const int64_t from = ((int64_t)chain * p.blocks + q) * CH + lane;
                    unsigned s = ~0u;
                    unsigned long long m = ~0ull;
                    while (!kind) {
                        if (lane < CH) {
                            s = __hip_atomic_load(p.state + from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                            m = __hip_atomic_load(p.map + from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                        }
                        kind = __all(lane >= CH || s != ~0u) ? 2 : __all(lane >= CH || m != ~0ull) ? 1 : 0;
                    }
                    if (lane < CH) {
                        sh.before[slot][lane][0] = __builtin_bit_cast(float, (unsigned)m);
                        sh.before[slot][lane][1] = __builtin_bit_cast(float, kind == 2 ? s : (unsigned)(m >> 32));
                    }
                }
                if (lane == 0) sh.kind[slot] = kind;
            }
            __syncthreads();
            int known = 0;
            while (known < WINDOW && sh.kind[known] != 2) ++known;
            if (known < WINDOW && tid < CH) {                             // forwards from there: the same operations whichever block it is
                carry = sh.before[known][tid][1];
                for (int slot = known - 1; slot >= 0; --slot) carry = fmaf(sh.before[slot][tid][0], carry, sh.before[slot][tid][1]);
            }
            if (known < WINDOW) break;
            __syncthreads();
        }
    }
    if (tid < CH) {
        behind = fmaf(a, carry, b);
        if (NW != ONE && !last) __hip_atomic_store(p.state + at + tid, word(behind), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.carry[tid] = carry;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        float pa = __shfl_up(A[j], 8), pb = __shfl_up(B[j], 8), s = sh.carry[cg + j];
        if (lane < 8) { pa = 1.f; pb = 0.f; }
        for (int w = 0; w < wave; ++w) s = fmaf(sh.wave[w][cg + j][0], s, sh.wave[w][cg + j][1]);
        in[j] = fmaf(pa, s, pb);
    }
    return behind;
}

// STATES: no results but the states before the stretches
template <class T, int NW, bool STATES> __global__ __launch_bounds__(64 * NW) void recur_forward(const RecurP p) {
    constexpr int PER = El<T>::PER16, CH = 8 * PER, BLOCK = block_steps(NW);
    __shared__ Shared<PER, NW> sh;
    const int tid = threadIdx.x, sub = tid >> 3, slabs = (p.C + CH - 1) / CH;
    const int2 at = place<PER, NW>(p, p.B * slabs, sh);
    const int b = at.x / slabs, c0 = (at.x - b * slabs) * CH, c = c0 + (tid & 7) * PER, left = p.C - c;
    const int len = p.lens ? min(max(p.lens[b], 0), p.T) : p.T;
    const int cc = left > 0 ? c : 0, cl = left > 0 ? left : p.C;        // lanes beyond the channels read the first ones and write nothing
    const bool mine = tid < CH && c0 + tid < p.C;                        // this thread's channel of the state
    const int64_t one = (int64_t)b * p.C + c0 + tid;
    const int t = at.y * BLOCK + sub * R;
    T* h = (T*)p.h + (int64_t)b * p.T * p.C + cc;
    const float zero[PER] = {};
    if (STATES && at.y * BLOCK >= len) return;
    if (at.y * BLOCK >= len) {                                           // nothing to do here but zeros; block 0 hands the state on
        if (left > 0)
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (t + r < p.T) Piece<T>::store(h + (int64_t)(t + r) * p.C, zero, left);
        if (at.y == 0 && mine) p.h_last[one] = p.h0 ? p.h0[one] : 0.f;
        return;
    }
    const T* x = (const T*)p.x + b * p.xs[0] + cc;
    const T* g = (const T*)p.gate + b * p.gs[0] + cc;
    u32x4 xr[R], gr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t tt = min(t + r, len - 1);
        xr[r] = Piece<T>::load(x + tt * p.xs[1], cl);
        gr[r] = Piece<T>::load(g + tt * p.gs[1], cl);
    }
    const float first = at.y == 0 && mine && p.h0 ? p.h0[one] : 0.f;
    float A[PER], B[PER], s[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        A[j] = 1.f;
        B[j] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float a, keep;
            gate_of(Piece<T>::at(gr[r], j), a, keep);
            if (t + r < len) {
                A[j] *= a;
                B[j] = fmaf(a, B[j], keep * Piece<T>::at(xr[r], j));
            }
        }
    }
    const bool last = (at.y + 1) * BLOCK >= len;
    const float behind = compose<PER, NW>(p, A, B, first, s, at.x, at.y, last, sh);
    if (STATES) {
        float* to = p.stretch + (((int64_t)at.x * p.blocks + at.y) * (NW * 8) + sub) * CH + c - c0;
#pragma unroll
        for (int j = 0; j < PER; j += 4) *(f32x4*)(to + j) = f32x4{s[j], s[j + 1], s[j + 2], s[j + 3]};
        return;
    }
    if (last && mine) p.h_last[one] = behind;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float out[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            float a, keep;
            gate_of(Piece<T>::at(gr[r], j), a, keep);
            s[j] = fmaf(a, s[j], keep * Piece<T>::at(xr[r], j));
            out[j] = t + r < len ? s[j] : 0.f;
        }
        if (t + r < p.T && left > 0) Piece<T>::store(h + (int64_t)(t + r) * p.C, out, left);
    }
}

// The state before this thread's steps t-R+1, ..., t of the only block -> s, which comes as the state before the block: the forward's operations,
// with the later of two stretches in the lower lanes and waves.  All threads call it.
template <class T, int NW>
__device__ __forceinline__ void before_stretch(float (&s)[El<T>::PER16], const u32x4 (&xr)[R], const u32x4 (&gr)[R], int t, int len,
                                               float (&maps)[NW][8 * El<T>::PER16][2]) {
    constexpr int PER = El<T>::PER16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cg = (lane & 7) * PER;
    float A[PER], B[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        A[j] = 1.f;
        B[j] = 0.f;
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            float a, keep;
            gate_of(Piece<T>::at(gr[r], j), a, keep);
            if (t - r < len) {
                A[j] *= a;
                B[j] = fmaf(a, B[j], keep * Piece<T>::at(xr[r], j));
            }
        }
    }
#pragma unroll
    for (int off = 8; off < 64; off <<= 1)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float a = __shfl_down(A[j], off), b = __shfl_down(B[j], off);
            if (lane + off < 64) {
                B[j] = fmaf(A[j], b, B[j]);
                A[j] *= a;
            }
        }
    if (lane < 8)
#pragma unroll
        for (int j = 0; j < PER; ++j) { maps[wave][cg + j][0] = A[j]; maps[wave][cg + j][1] = B[j]; }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        float pa = __shfl_down(A[j], 8), pb = __shfl_down(B[j], 8);
        if (lane >= 56) { pa = 1.f; pb = 0.f; }
        for (int w = NW - 1; w > wave; --w) s[j] = fmaf(maps[w][cg + j][0], s[j], maps[w][cg + j][1]);
        s[j] = fmaf(pa, s[j], pb);
    }
}

// the forward's blocks, latest first; those behind the sequence's end come after them
template <class T, int NW> __global__ __launch_bounds__(64 * NW) void recur_gradient(const RecurP p) {
    constexpr int PER = El<T>::PER16, CH = 8 * PER, BLOCK = block_steps(NW);
    constexpr bool AGAIN = sizeof(T) == 2;                               // the forward's result is not the state
    __shared__ Shared<PER, NW> sh;
    __shared__ float maps[AGAIN && NW == ONE ? NW : 1][CH][2];
    const int tid = threadIdx.x, sub = tid >> 3, slabs = (p.C + CH - 1) / CH;
    const int2 at = place<PER, NW>(p, p.B * slabs, sh);
    const int b = at.x / slabs, c0 = (at.x - b * slabs) * CH, c = c0 + (tid & 7) * PER, left = p.C - c;
    const int len = p.lens ? min(max(p.lens[b], 0), p.T) : p.T, blocks = (len + BLOCK - 1) / BLOCK;
    const int cc = left > 0 ? c : 0, cl = left > 0 ? left : p.C;
    const bool mine = tid < CH && c0 + tid < p.C;
    const int64_t one = (int64_t)b * p.C + c0 + tid;
    const int block = at.y < blocks ? blocks - 1 - at.y : at.y;          // in time
    const int t = block * BLOCK + BLOCK - 1 - sub * R;                   // this thread: t, t-1, ..., t-R+1
    T* dx = (T*)p.dx + (int64_t)b * p.T * p.C + cc;
    T* dg = (T*)p.dgate + (int64_t)b * p.T * p.C + cc;
    const float zero[PER] = {};
    if (at.y >= blocks) {
        if (left > 0)
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (t - r < p.T) {
                    Piece<T>::store(dx + (int64_t)(t - r) * p.C, zero, left);
                    Piece<T>::store(dg + (int64_t)(t - r) * p.C, zero, left);
                }
        if (at.y == 0 && mine && p.dh0) p.dh0[one] = p.dh_last ? p.dh_last[one] : 0.f;
        return;
    }
    const T* x = (const T*)p.x + b * p.xs[0] + cc;
    const T* g = (const T*)p.gate + b * p.gs[0] + cc;
    const T* h = (const T*)p.hin + b * p.hs[0] + cc;
    const T* d = (const T*)p.dh + b * p.ds[0] + cc;
    u32x4 xr[R], gr[R], hr[R], dr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t tt = min(t - r, len - 1);
        gr[r] = Piece<T>::load(g + tt * p.gs[1], cl);
        dr[r] = Piece<T>::load(d + tt * p.ds[1], cl);
        xr[r] = Piece<T>::load(x + tt * p.xs[1], cl);
        if (!AGAIN) hr[r] = Piece<T>::load(h + max(tt - 1, (int64_t)0) * p.hs[1], cl);
    }
    const float first = at.y == 0 && mine && p.dh_last ? p.dh_last[one] : 0.f;
    float A[PER], B[PER], s[PER], h0[PER];                               // h0: the state before step 0; 16 bits, later: before the stretch
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        h0[j] = p.h0 && block == 0 && j < left ? p.h0[(int64_t)b * p.C + c + j] : 0.f;
        A[j] = 1.f;
        B[j] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float a, keep;
            gate_of(Piece<T>::at(gr[r], j), a, keep);
            if (t - r < len) {
                A[j] *= a;
                B[j] = a * (B[j] + Piece<T>::at(dr[r], j));
            }
        }
    }
    if (AGAIN && NW != ONE) {
        const float* from = p.stretch + (((int64_t)at.x * p.blocks + block) * (NW * 8) + NW * 8 - 1 - sub) * CH + c - c0;
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
            const f32x4 v = *(const f32x4*)(from + j);
            h0[j] = v[0]; h0[j + 1] = v[1]; h0[j + 2] = v[2]; h0[j + 3] = v[3];
        }
    }
    const bool last = block == 0;
    const float behind = compose<PER, NW>(p, A, B, first, s, at.x, at.y, last, sh);
    if (last && mine && p.dh0) p.dh0[one] = behind;
    if constexpr (AGAIN && NW == ONE) before_stretch<T, NW>(h0, xr, gr, t, len, maps);
    float hb[R][PER];                                                    // h_{t-1} of the steps
#pragma unroll
    for (int r = R - 1; r >= 0; --r)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            hb[r][j] = AGAIN || t - r == 0 ? h0[j] : Piece<T>::at(hr[r], j);
            if (AGAIN) {
                float a, keep;
                gate_of(Piece<T>::at(gr[r], j), a, keep);
                h0[j] = fmaf(a, h0[j], keep * Piece<T>::at(xr[r], j));
            }
        }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float ox[PER], og[PER];
        const bool there = t - r < len;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            float a, keep;
            gate_of(Piece<T>::at(gr[r], j), a, keep);
            const float l = Piece<T>::at(dr[r], j) + s[j];
            ox[j] = there ? keep * l : 0.f;
            og[j] = there ? a * keep * (hb[r][j] - Piece<T>::at(xr[r], j)) * l : 0.f;
            if (there) s[j] = a * l;
        }
        if (t - r < p.T && left > 0) {
            Piece<T>::store(dx + (int64_t)(t - r) * p.C, ox, left);
            Piece<T>::store(dg + (int64_t)(t - r) * p.C, og, left);
        }
    }
}

struct ClearP { u32x4* at; int64_t n, chain; };
__global__ __launch_bounds__(256) void recur_clear(const ClearP p) {       // ones; the first piece of each chain's space (its ticket) zero
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < p.n) p.at[i] = i && i != p.chain ? u32x4{~0u, ~0u, ~0u, ~0u} : u32x4{0, 0, 0, 0};
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------------
static int check(const oph_seq_recur* a) {
    if (!a) return fail(OPH_ERR_INVALID, "recurrence: no arguments");
    if (!type_bytes(a->dtype)) return fail(OPH_ERR_INVALID, "recurrence: dtype %d is not one of OPH_SEQ_*", a->dtype);
    if (a->B < 0 || a->T < 0 || a->C < 1) return fail(OPH_ERR_INVALID, "recurrence: bad size (B %d, T %d, C %d)", a->B, a->T, a->C);
    if (a->T > 2147483647 - 4096 || a->C > 1 << 28 || (double)a->B * (a->C / 32 + 1) * (a->T / block_steps(MANY) + 1) > 8.0e6)
        return fail(OPH_ERR_UNSUPPORTED, "recurrence: too large (B %d, T %d, C %d)", a->B, a->T, a->C);
    return OPH_OK;
}
static RecurP params(const oph_seq_recur* a) {
    RecurP p = {};
    p.x = a->x; p.gate = a->gate; p.h0 = a->h0; p.lens = a->lens;
    p.B = a->B; p.T = a->T; p.C = a->C;
    for (int i = 0; i < 2; ++i) { p.xs[i] = a->x_stride[i]; p.gs[i] = a->gate_stride[i]; p.hs[i] = a->h_stride[i]; p.ds[i] = a->dh_stride[i]; }
    return p;
}
struct Plan { int64_t chains, blocks, words; };                            // words: published states
static Plan plan(const oph_seq_recur* a) {
    const int ch = 128 / type_bytes(a->dtype);
    Plan l;
    l.chains = a->B * cdiv(a->C, ch);
    l.blocks = a->T > block_steps(ONE) ? cdiv(a->T, block_steps(MANY)) : 1;
    l.words = l.blocks > 1 ? l.chains * l.blocks * ch : 0;
    return l;
}
// one chain's space: ticket, maps, states
static int64_t chain_bytes(const Plan& l) { return l.words ? 16 + l.words * 12 : 0; }
// the gradient in 16 bits: a chain's space for each of its passes, and the states before the stretches
static int64_t workspace(const oph_seq_recur* a, bool gradient) {
    const Plan l = plan(a);
    return gradient && type_bytes(a->dtype) == 2 ? 2 * chain_bytes(l) + l.words * (MANY * 8) * (int64_t)sizeof(float) : chain_bytes(l);
}
static void use_chain(RecurP& p, const Plan& l, char* at) {
    p.ticket = (unsigned*)at;
    p.map = (unsigned long long*)(at + 16);
    p.state = (unsigned*)(p.map + l.words);
}
static int start(const oph_seq_recur* a, RecurP& p, bool gradient, void* stream) {          // clears what the blocks hand on
    const Plan l = plan(a);
    p.blocks = (int)l.blocks;
    if (!l.words) return OPH_OK;
    use_chain(p, l, (char*)a->workspace);
    const int64_t each = chain_bytes(l) / 16;
    const ClearP c = {(u32x4*)a->workspace, gradient && type_bytes(a->dtype) == 2 ? 2 * each : each, each};
    return launch<ClearP>(recur_clear, dim3((unsigned)cdiv(c.n, 256)), 256, c, 0, stream);
}
template <class F> static int run(F one, F many, const oph_seq_recur* a, const RecurP& p, void* stream) {
    const Plan l = plan(a);
    return launch<RecurP>(l.blocks == 1 ? one : many, dim3((unsigned)(l.chains * l.blocks)), 64 * (l.blocks == 1 ? ONE : MANY), p, 0, stream);
}
template <class T> static int gradient(const oph_seq_recur* a, RecurP& p, void* stream) {
    const Plan l = plan(a);
    if constexpr (sizeof(T) == 2)
        if (l.words) {
            p.stretch = (float*)((char*)a->workspace + 2 * chain_bytes(l));
            if (int rc = launch<RecurP>(recur_forward<T, MANY, true>, dim3((unsigned)(l.chains * l.blocks)), 64 * MANY, p, 0, stream)) return rc;
            use_chain(p, l, (char*)a->workspace + chain_bytes(l));
        }
    return run(recur_gradient<T, ONE>, recur_gradient<T, MANY>, a, p, stream);
}
static int check_workspace(const oph_seq_recur* a, bool gradient) {
    const int64_t need = workspace(a, gradient);
    if (need && (!a->workspace || (int64_t)a->workspace_bytes < need || ((uintptr_t)a->workspace & 15)))
        return fail(OPH_ERR_INVALID, "recurrence: the workspace must hold %lld bytes, 16-byte aligned", (long long)need);
    return OPH_OK;
}

}  // namespace ophseq

using namespace ophseq;
extern "C" {

int64_t oph_seq_recur_workspace(const oph_seq_recur* a, int gradient) {
    if (int rc = check(a)) return rc;
    return workspace(a, gradient != 0);
}

int oph_seq_recur_forward(const oph_seq_recur* a, int device, void* stream) {
    if (int rc = check(a)) return rc;
    if (!a->B) return OPH_OK;
    if (!a->h_last || (a->T && (!a->x || !a->gate || !a->h))) return fail(OPH_ERR_INVALID, "recurrence: x, gate, h and h_last must not be NULL");
    if (int rc = check_workspace(a, false)) return rc;
    OnDevice on(device);
    if (on.status) return on.status;
    RecurP p = params(a);
    p.h = a->h;
    p.h_last = a->h_last;
    if (int rc = start(a, p, false, stream)) return rc;
    if (a->dtype == OPH_SEQ_F32) return run(recur_forward<float, ONE, false>, recur_forward<float, MANY, false>, a, p, stream);
    if (a->dtype == OPH_SEQ_BF16) return run(recur_forward<bf16_t, ONE, false>, recur_forward<bf16_t, MANY, false>, a, p, stream);
    return run(recur_forward<f16_t, ONE, false>, recur_forward<f16_t, MANY, false>, a, p, stream);
}

int oph_seq_recur_gradient(const oph_seq_recur* a, int device, void* stream) {
    if (int rc = check(a)) return rc;
    if (!a->B) return OPH_OK;
    if (a->T && (!a->x || !a->gate || !a->h || !a->dh || !a->dx || !a->dgate))
        return fail(OPH_ERR_INVALID, "recurrence: x, gate, h, dh, dx and dgate must not be NULL");
    if (int rc = check_workspace(a, true)) return rc;
    OnDevice on(device);
    if (on.status) return on.status;
    RecurP p = params(a);
    p.hin = a->h; p.dh = a->dh; p.dh_last = a->dh_last; p.dx = a->dx; p.dgate = a->dgate; p.dh0 = a->dh0;
    if (int rc = start(a, p, true, stream)) return rc;
    if (a->dtype == OPH_SEQ_F32) return gradient<float>(a, p, stream);
    if (a->dtype == OPH_SEQ_BF16) return gradient<bf16_t>(a, p, stream);
    return gradient<f16_t>(a, p, stream);
}

}  // extern "C"
