// Gated linear recurrence along a long axis and its backward pass.
//
//   forward    h_s = a_s h_(s-1) + x_s,   h_(-1) = h0                       (s: order of processing)
//   backward   d_s = g_s + e_(s+1),  e_s = a_s d_s,  e_(len) = d_last       (g = dL/dh)
//              dL/dx_s = d_s,  dL/da_s = sum over the channels of a gate of d_s h_(s-1),  dL/dh0 = e_0
//
// Both directions are compositions of maps s -> A s + H, which are associative: the steps of a column (two
// neighbouring channels of one sequence) are cut into runs, each run is reduced to its (A, H),
// the (A, H) of the runs in front are composed onto the state at the start, and every run is then walked
// again from its own start state, out of registers.  State, products and sums are fp32 throughout.
//
// A workgroup holds 2^LC columns x (256 >> LC) runs of SC_U steps ("a tile") and walks along the sequence
// tile by tile, so a sequence that one workgroup walks whole has every input read once.  The forward pass of a training step keeps the fp32 state in
// front of every 32nd step; the backward pass walks the tiles from the last to the first and rebuilds the
// states inside a tile from these and x, which costs no more bytes than reading h and keeps dL/da free
// of the rounding of h.
//
// Where there are too few columns to fill the chip the sequence itself is cut into stretches (grid.y): a
// first launch reduces every stretch to its (A, H), the second composes those in front of its own and walks.
//
// What bounds it, and the measurements behind the constants (MI355X; a copy reaches 4.8 TB/s here).  The walk is
// a chain of load, compose, store per tile, so what counts is wavefronts in flight, not work per thread:
//   two channels a thread (90-115 registers, 4-5 wavefronts a SIMD) against four (140-190, 2-3): 123 against
//   215 us forward + backward for 4096 ragged sequences x 192 x 64 in bf16 with one fp32 gate a step, 312 against
//   389 us for 2 x 32768 x 1024; one channel a thread: 146 and 403 us.
//   8 steps a run against 4: 123 / 146 us and 312 / 375 us.
//   Short sequences pay for what happens once a workgroup: the longest length by lane shifts and not by an LDS
//   atomic, and rows walked by pointer (multiples of five strides no longer fill the scalar registers), took
//   4096 x 192 x 64 from 123 to 98 us (31 forward, 67 backward; its bytes cost 64 at 5.55 TB/s).
//   Loading the next tile ahead in the backward pass costs registers and loses (280 against 164 us); in the
//   forward pass it gains.
// 2 x 32768 x 1024 in bf16 then takes 124 us forward (53 of them the first launch, 5.1 TB/s; the walk
// moves 5.6 TB/s with the first launch's reads partly cached) and 184 us backward, against 145 us that the bytes of
// one pass over every tensor cost at 5.55 TB/s; reading a and x (a and g) twice is what is left.
#include "nk_common.h"

namespace {

enum { SC_THREADS = 256, SC_VC = 2, SC_U = 8, SC_KEEP = 32,
       SC_NONE = -(1 << 30) };      // a limit below every step: nothing is loaded, not even from in front of the first step
struct ScanArgs {
    const void* a; const void* x; const void* g;    // g: dL/dh (backward)
    const float* h0; const float* first;            // first: state the walk starts from (h0 or d_last)
    void* o; void* d_a;                             // o: h or dL/dx
    float* last;                                    // state behind the walk (h_last, dL/dh0)
    float* states;                                  // [B][ceil(T / 32)][C]: state in front of step 32 k
    float* sums;                                    // [stretch][2][columns * VC]: A, H of every stretch
    float* gate_part;                               // [part][B * T * J]: partial sums of dL/da of a wide gate
    const int32_t* lengths;
    int64_t C, a_sb, a_st, x_sb, x_st, g_sb, g_st;
    int64_t cols, B, J;
    int32_t T, stretch;                             // steps, steps per stretch
    int32_t G, LG, per_b, LC, reverse;              // channels per gate, columns per gate, columns per sequence
};

// Channels of a column.  A load or store of two takes any address that their type allows: the memory path splits what
// crosses a line, and odd rows (C odd, sliced tensors) start anywhere.  The last column of an odd number of channels takes the
// one before once more (the same values to the same place) rather than a branch: 781 x 237 x 127 in fp16, forward +
// backward, 113 us against 176 with one channel a column; 2 x 32768 x 999 in bf16 424 against 479.
template <typename T, int VC> struct Pack { T v[VC]; };
template <typename T, int VC> NK_D Pack<T, VC> ld(const T* p) {
    Pack<T, VC> r;
    if constexpr (VC == 1) r.v[0] = *p;
    else {
        typedef __attribute__((ext_vector_type(VC), aligned(sizeof(T)))) T vec;
        const vec w = *(const vec*)p;
#pragma unroll
        for (int k = 0; k < VC; ++k) r.v[k] = w[k];
    }
    return r;
}
template <typename T, int VC> NK_D void st(T* p, const float* v) {
    if constexpr (VC == 1) *p = (T)v[0];
    else {
        typedef __attribute__((ext_vector_type(VC), aligned(sizeof(T)))) T vec;
        vec w;
#pragma unroll
        for (int k = 0; k < VC; ++k) w[k] = (T)v[k];
        *(vec*)p = w;
    }
}

// A s + H on a state; a state of exactly zero gives H even where the product of the gates has left the
// range of fp32
NK_D float apply(float A, float H, float s) { return s == 0.0f ? H : fmaf(A, s, H); }

// What a thread works on: its column and which run of a tile.
struct Place {
    int64_t b, c, gate, col;    // sequence, first channel, gate, column
    int k;                      // which column of the gate
    int run;
    int len;                    // live steps of the sequence; 0 for columns that only round a gate up
    bool on;                    // has channels
    bool twice;                 // the last column of an odd number of channels: its first channel is the column's before as well
};
template <int VC, bool SHARED> NK_D Place place(const ScanArgs& A) {
    Place p;
    const int lcol = 1 << A.LC;
    p.run = threadIdx.x >> A.LC;
    p.col = (int64_t)blockIdx.x * lcol + (threadIdx.x & (lcol - 1));
    p.b = p.col / A.per_b;
    const int r = (int)(p.col - p.b * A.per_b);
    p.on = p.col < A.cols;
    if (SHARED) {
        const int j = r / A.LG;
        p.k = r - j * A.LG;
        p.on = p.on && p.k * VC < A.G;
        p.twice = VC > 1 && p.k * VC == A.G - 1;
        p.gate = j; p.c = (int64_t)j * A.G + (int64_t)p.k * VC - (p.twice ? 1 : 0);
    } else {
        p.twice = VC > 1 && (int64_t)r * VC == A.C - 1;
        p.k = 0; p.c = (int64_t)r * VC - (p.twice ? 1 : 0); p.gate = p.c;
    }
    p.len = !p.on ? 0 : A.lengths ? max(0, min(A.T, A.lengths[p.b])) : A.T;
    return p;
}

// Steps s0 .. s0 + SC_U - 1 of a column; `fill` where s reaches `lim`.  base: the row of step s0.  whole: no lane
// of the wavefront reaches it.
template <typename T, int VC>
NK_D void fetch(Pack<T, VC> (&r)[SC_U], const T* base, int64_t step, int s0, int lim, float fill, bool whole) {
    if (whole) {
#pragma unroll
        for (int u = 0; u < SC_U; ++u, base += step) r[u] = ld<T, VC>(base);
    } else {
#pragma unroll
        for (int u = 0; u < SC_U; ++u, base += step) {
#pragma unroll
            for (int v = 0; v < VC; ++v) r[u].v[v] = (T)fill;
            if (s0 + u < lim) r[u] = ld<T, VC>(base);
        }
    }
}
// row of step s of a sequence of len steps
NK_D int64_t time_of(int s, int len, int reverse) { return reverse ? len - 1 - s : s; }

// Largest live length of the workgroup's columns.
NK_D int longest(const Place& p, const ScanArgs& A) {
    if (!A.lengths) return A.T;
    __shared__ int most[SC_THREADS / 64];
    const int mine = (int)nk_wave_max((uint32_t)p.len);
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = mine;
    __syncthreads();
    int m = most[0];
#pragma unroll
    for (int w = 1; w < SC_THREADS / 64; ++w) m = max(m, most[w]);
    return m;
}

template <int VC> struct Buf { float v[4][3 * VC][64]; };

// Runs of a tile in ascending order.  In: (Ar, Hr) of this thread's run and `carry`, the state in front of the
// tile.  Out: s, the state in front of this run; carry, the one behind the tile.  Runs of one wavefront are
// composed with lane shuffles, wavefronts through LDS (`buf` alternates, so one barrier a tile is enough).
template <int VC>
NK_D void compose_up(const float* Ain, const float* Hin, float* carry, float* s, int LC, Buf<VC>& buf) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lcol = 1 << LC, cl = lane & (lcol - 1);
    if (LC == 8) {          // every thread has a column of its own
#pragma unroll
        for (int v = 0; v < VC; ++v) { s[v] = carry[v]; carry[v] = apply(Ain[v], Hin[v], carry[v]); }
        return;
    }
    float Ar[VC], Hr[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) { Ar[v] = Ain[v]; Hr[v] = Hin[v]; }
    for (int off = lcol; off < 64; off <<= 1) {         // inclusive over the runs of the wavefront
#pragma unroll
        for (int v = 0; v < VC; ++v) {
            const float A0 = __shfl_up(Ar[v], off, 64), H0 = __shfl_up(Hr[v], off, 64);
            if (lane >= off) { Hr[v] = apply(Ar[v], Hr[v], H0); Ar[v] *= A0; }
        }
    }
    if (LC >= 6 || lane >= 64 - lcol) {
#pragma unroll
        for (int v = 0; v < VC; ++v) { buf.v[wave][v][cl] = Ar[v]; buf.v[wave][VC + v][cl] = Hr[v]; }
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VC; ++v) {
        float c = carry[v];
        s[v] = c;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            c = apply(buf.v[w][v][cl], buf.v[w][VC + v][cl], c);
            if (w + 1 == wave) s[v] = c;
        }
        carry[v] = c;
        if (LC < 6) {
            const float A0 = __shfl_up(Ar[v], lcol, 64), H0 = __shfl_up(Hr[v], lcol, 64);
            if (lane >= lcol) s[v] = apply(A0, H0, s[v]);
        }
    }
}

// The backward pass's two compositions with one barrier: (A, H) ascending from the kept state `hs` in front of
// the tile (out: h, the state in front of this run), and (A, E) descending from `carry` behind the tile
// (out: e, what this run starts from; carry, in front of the tile).
template <int VC>
NK_D void compose_both(const float* Ain, const float* Hin, const float* Ein, const float* hs, float* carry, float* h, float* e,
                       int LC, Buf<VC>& buf) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lcol = 1 << LC, cl = lane & (lcol - 1);
    if (LC == 8) {
#pragma unroll
        for (int v = 0; v < VC; ++v) { h[v] = hs[v]; e[v] = carry[v]; carry[v] = apply(Ain[v], Ein[v], carry[v]); }
        return;
    }
    float Au[VC], Hr[VC], Ad[VC], Er[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) { Au[v] = Ad[v] = Ain[v]; Hr[v] = Hin[v]; Er[v] = Ein[v]; }
    for (int off = lcol; off < 64; off <<= 1) {
#pragma unroll
        for (int v = 0; v < VC; ++v) {
            const float A0 = __shfl_up(Au[v], off, 64), H0 = __shfl_up(Hr[v], off, 64);
            const float A1 = __shfl_down(Ad[v], off, 64), E1 = __shfl_down(Er[v], off, 64);
            if (lane >= off) { Hr[v] = apply(Au[v], Hr[v], H0); Au[v] *= A0; }
            if (lane + off < 64) { Er[v] = apply(Ad[v], Er[v], E1); Ad[v] *= A1; }
        }
    }
    if (LC >= 6 || lane >= 64 - lcol) {
#pragma unroll
        for (int v = 0; v < VC; ++v) { buf.v[wave][v][cl] = Au[v]; buf.v[wave][VC + v][cl] = Hr[v]; }
    }
    if (LC >= 6 || lane < lcol) {
#pragma unroll
        for (int v = 0; v < VC; ++v) buf.v[wave][2 * VC + v][cl] = Er[v];
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VC; ++v) {
        float c = hs[v], d = carry[v];
        h[v] = c; e[v] = d;
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            c = apply(buf.v[w][v][cl], buf.v[w][VC + v][cl], c);
            if (w + 1 == wave) h[v] = c;
        }
#pragma unroll
        for (int w = 3; w >= 0; --w) {
            d = apply(buf.v[w][v][cl], buf.v[w][2 * VC + v][cl], d);
            if (w - 1 == wave) e[v] = d;
        }
        carry[v] = d;
        if (LC < 6) {
            const float A0 = __shfl_up(Au[v], lcol, 64), H0 = __shfl_up(Hr[v], lcol, 64);
            const float A1 = __shfl_down(Ad[v], lcol, 64), E1 = __shfl_down(Er[v], lcol, 64);
            if (lane >= lcol) h[v] = apply(A0, H0, h[v]);
            if (lane + lcol < 64) e[v] = apply(A1, E1, e[v]);
        }
    }
}

// state at the start of stretch y of this launch: the (A, H) of the stretches walked before it composed
// onto the given one (ascending in the forward pass, descending in the backward pass).  The runs of a column
// share them, each a contiguous part, and meet as the runs of a tile do.
template <int VC, bool BWD> NK_D void stretch_start(const ScanArgs& A, const Place& p, float* carry, Buf<VC>& buf) {
    const int n = BWD ? gridDim.y - 1 - blockIdx.y : blockIdx.y;
    if (n == 0) return;             // workgroup-uniform
    const int runs = SC_THREADS >> A.LC, per = (n + runs - 1) / runs;
    // q: in the order of the walk; the backward composition takes the runs from the last to the first
    const int mine = BWD ? runs - 1 - p.run : p.run, q0 = mine * per, q1 = min(n, q0 + per);
    float Ar[VC], Hr[VC], s[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) { Ar[v] = 1.0f; Hr[v] = 0.0f; }
    if (p.on) {
#pragma unroll 4
        for (int q = q0; q < q1; ++q) {
            const int y = BWD ? gridDim.y - 1 - q : q;
            const float* w = A.sums + (int64_t)y * 2 * A.cols * VC + p.col * VC;
#pragma unroll
            for (int v = 0; v < VC; ++v) { Hr[v] = apply(w[v], w[A.cols * VC + v], Hr[v]); Ar[v] *= w[v]; }
        }
    }
    if (BWD) {
        float zero[VC], h[VC];
#pragma unroll
        for (int v = 0; v < VC; ++v) zero[v] = 0.0f;
        compose_both<VC>(Ar, zero, Hr, zero, carry, h, s, A.LC, buf);
    } else {
        compose_up<VC>(Ar, Hr, carry, s, A.LC, buf);
    }
}

// First launch of a split sequence: (A, H) of a stretch, or (A, E) of the backward pass.  Nothing has to be
// written in order here, so a thread takes one long run of the stretch and the runs are composed once.
template <typename T, typename GT, int VC, bool SHARED, bool BWD>
__global__ __launch_bounds__(SC_THREADS) void k_scan_sum(const ScanArgs A) {
    __shared__ Buf<VC> buf[2];
    const Place p = place<VC, SHARED>(A);
    constexpr int GV = SHARED ? 1 : VC;
    const int y = blockIdx.y + (BWD ? 1 : 0);        // the stretch walked last needs no sum
    const int per = A.stretch / (SC_THREADS >> A.LC), lo = y * A.stretch + p.run * per;
    const int hi = min(lo + per, p.len);
    float Ar[VC], Hr[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) { Ar[v] = 1.0f; Hr[v] = 0.0f; }
    const int64_t as = A.reverse ? -A.a_st : A.a_st, xs = A.reverse ? -A.x_st : A.x_st;
    const GT* ab = (const GT*)A.a + p.b * A.a_sb + p.gate;
    const T* xb = (const T*)A.x + p.b * A.x_sb + p.c;
    const int rows = hi - lo, turns = rows > 0 ? (rows + SC_U - 1) / SC_U : 0;
    for (int q = 0; q < turns; ++q) {
        const int s0 = lo + (BWD ? turns - 1 - q : q) * SC_U;
        const int64_t t0 = time_of(s0, p.len, A.reverse);
        Pack<GT, GV> ra[SC_U];
        Pack<T, VC> rx[SC_U];
        const bool whole = __all(s0 + SC_U <= hi);
        fetch<GT, GV>(ra, ab + t0 * A.a_st, as, s0, hi, 1.0f, whole);
        fetch<T, VC>(rx, xb + t0 * A.x_st, xs, s0, A.x ? hi : SC_NONE, 0.0f, whole && A.x);
#pragma unroll
        for (int w = 0; w < SC_U; ++w) {
            const int u = BWD ? SC_U - 1 - w : w;
#pragma unroll
            for (int v = 0; v < VC; ++v) {
                const float a = (float)ra[u].v[SHARED ? 0 : v], x = (float)rx[u].v[v];
                Hr[v] = BWD ? a * (x + Hr[v]) : fmaf(a, Hr[v], x);
                Ar[v] *= a;
            }
        }
    }
    // H from a start of zero, A from a start of one without summands
    float zero[VC], one[VC], H[VC], s[VC], e[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) { zero[v] = H[v] = 0.0f; one[v] = 1.0f; }
    if (BWD) {
        compose_both<VC>(Ar, zero, Hr, zero, H, s, e, A.LC, buf[0]);
        compose_both<VC>(Ar, zero, zero, zero, one, s, e, A.LC, buf[1]);
    } else {
        compose_up<VC>(Ar, Hr, H, s, A.LC, buf[0]);
        compose_up<VC>(Ar, zero, one, s, A.LC, buf[1]);
    }
    if (p.on && p.run == 0) {
        float* w = A.sums + (int64_t)y * 2 * A.cols * VC + p.col * VC;
#pragma unroll
        for (int v = 0; v < VC; ++v) { w[v] = one[v]; w[A.cols * VC + v] = H[v]; }
    }
}

template <typename T, typename GT, int VC, bool SHARED>
__global__ __launch_bounds__(SC_THREADS) void k_scan_fwd(const ScanArgs A) {
    __shared__ Buf<VC> buf[2];
    constexpr int GV = SHARED ? 1 : VC;
    const Place p = place<VC, SHARED>(A);
    const int tile = (SC_THREADS >> A.LC) * SC_U;
    const int begin = blockIdx.y * A.stretch, end = min(A.T, begin + A.stretch);
    const int stop = min(end, longest(p, A));           // behind it every column is dead
    float carry[VC], s[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) carry[v] = 0.0f;
    if (p.on && A.first) for (int v = 0; v < VC; ++v) carry[v] = A.first[p.b * A.C + p.c + v];
    stretch_start<VC, false>(A, p, carry, buf[1]);
    const int64_t as = A.reverse ? -A.a_st : A.a_st, xs = A.reverse ? -A.x_st : A.x_st, os = A.reverse ? -A.C : A.C;
    const GT* ab = (const GT*)A.a + p.b * A.a_sb + p.gate;
    const T* xb = (const T*)A.x + p.b * A.x_sb + p.c;
    T* ob = (T*)A.o + p.b * A.T * A.C + p.c;
    const int kept = (A.T + SC_KEEP - 1) / SC_KEEP;
    const int lim = min(p.len, end);
    Pack<GT, GV> ra[SC_U];
    Pack<T, VC> rx[SC_U];
    int s0 = begin + p.run * SC_U;
    bool whole = __all(s0 + SC_U <= lim);
    {
        const int64_t t0 = time_of(s0, p.len, A.reverse);
        fetch<GT, GV>(ra, ab + t0 * A.a_st, as, s0, lim, 1.0f, whole);
        fetch<T, VC>(rx, xb + t0 * A.x_st, xs, s0, lim, 0.0f, whole);
    }
    int flip = 0, at = begin;
    for (; at < stop; at += tile, s0 += tile, flip ^= 1) {
        Pack<GT, GV> na[SC_U];
        Pack<T, VC> nx[SC_U];
        const bool next = __all(s0 + tile + SC_U <= lim);
        {       // the next tile's loads are in flight while this one is composed and written
            const int s1 = s0 + tile;
            const int64_t t1 = time_of(s1, p.len, A.reverse);
            fetch<GT, GV>(na, ab + t1 * A.a_st, as, s1, lim, 1.0f, next);
            fetch<T, VC>(nx, xb + t1 * A.x_st, xs, s1, lim, 0.0f, next);
        }
        float Ar[VC], Hr[VC];
#pragma unroll
        for (int v = 0; v < VC; ++v) { Ar[v] = 1.0f; Hr[v] = 0.0f; }
#pragma unroll
        for (int u = 0; u < SC_U; ++u)
#pragma unroll
            for (int v = 0; v < VC; ++v) {
                const float a = (float)ra[u].v[SHARED ? 0 : v];
                Hr[v] = fmaf(a, Hr[v], (float)rx[u].v[v]);
                Ar[v] *= a;
            }
        compose_up<VC>(Ar, Hr, carry, s, A.LC, buf[flip]);
        if (A.states && (s0 & (SC_KEEP - 1)) == 0 && s0 < lim) st<float, VC>(A.states + ((int64_t)p.b * kept + s0 / SC_KEEP) * A.C + p.c, s);
        T* o = ob + time_of(s0, p.len, A.reverse) * A.C;
        if (whole) {
#pragma unroll
            for (int u = 0; u < SC_U; ++u, o += os) {
#pragma unroll
                for (int v = 0; v < VC; ++v) s[v] = fmaf((float)ra[u].v[SHARED ? 0 : v], s[v], (float)rx[u].v[v]);
                st<T, VC>(o, s);
            }
        } else {
            T* behind = ob + (int64_t)s0 * A.C;         // rows behind the sequence: zeros, in place
#pragma unroll
            for (int u = 0; u < SC_U; ++u, o += os, behind += A.C) {
                float w[VC];
                const bool live = s0 + u < lim;
#pragma unroll
                for (int v = 0; v < VC; ++v) { s[v] = fmaf((float)ra[u].v[SHARED ? 0 : v], s[v], (float)rx[u].v[v]); w[v] = live ? s[v] : 0.0f; }
                if (live || (p.on && s0 + u < end)) st<T, VC>(live ? o : behind, w);
            }
        }
        whole = next;
#pragma unroll
        for (int u = 0; u < SC_U; ++u) { ra[u] = na[u]; rx[u] = nx[u]; }
    }
    float z[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) z[v] = 0.0f;
    if (p.on) for (int t = at + p.run; t < end; t += SC_THREADS >> A.LC) st<T, VC>(ob + (int64_t)t * A.C, z);
    if (p.on && p.run == 0 && A.last && end == A.T)
        for (int v = 0; v < VC; ++v) A.last[p.b * A.C + p.c + v] = carry[v];
}

// Sums of SC_U values over the `wide` (a power of two) neighbouring lanes of a gate: while a lane holds more
// than one value it trades half of them with its partner, so U values cost about U shuffles instead of
// U log2(wide).  On return the lane holds sums of steps u0 .. u0 + n - 1, all of them if `mine`.
NK_D void gate_sums(float (&v)[SC_U], int wide, int k, int* u0, int* n, bool* mine) {
    int off = wide >> 1, held = SC_U, first = 0;
    if (off > 0) {
        const bool up = (k & off) != 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float keep = up ? v[4 + i] : v[i], send = up ? v[i] : v[4 + i];
            v[i] = keep + __shfl_xor(send, off, 64);
        }
        first += up ? 4 : 0; held = 4; off >>= 1;
    }
    if (off > 0) {
        const bool up = (k & off) != 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float keep = up ? v[2 + i] : v[i], send = up ? v[i] : v[2 + i];
            v[i] = keep + __shfl_xor(send, off, 64);
        }
        first += up ? 2 : 0; held = 2; off >>= 1;
    }
    if (off > 0) {
        const bool up = (k & off) != 0;
        const float keep = up ? v[1] : v[0], send = up ? v[0] : v[1];
        v[0] = keep + __shfl_xor(send, off, 64);
        first += up ? 1 : 0; held = 1; off >>= 1;
    }
    *mine = (k & (2 * off - (off > 0 ? 1 : 0))) == 0;
    for (; off > 0; off >>= 1) v[0] += __shfl_xor(v[0], off, 64);
    *u0 = first; *n = held;
}

template <typename T, typename GT, int VC, bool SHARED>
__global__ __launch_bounds__(SC_THREADS, 4) void k_scan_bwd(const ScanArgs A) {
    __shared__ Buf<VC> buf[2];
    constexpr int GV = SHARED ? 1 : VC;
    const Place p = place<VC, SHARED>(A);
    const int tile = (SC_THREADS >> A.LC) * SC_U;
    const int begin = blockIdx.y * A.stretch, end = min(A.T, begin + A.stretch);
    const int stop = min(end, longest(p, A));
    float carry[VC];
#pragma unroll
    for (int v = 0; v < VC; ++v) carry[v] = 0.0f;
    if (p.on && A.first) for (int v = 0; v < VC; ++v) carry[v] = A.first[p.b * A.C + p.c + v];
    stretch_start<VC, true>(A, p, carry, buf[1]);
    const bool gates = A.d_a != nullptr;
    const int64_t as = A.reverse ? -A.a_st : A.a_st, xs = A.reverse ? -A.x_st : A.x_st, gs = A.reverse ? -A.g_st : A.g_st;
    const GT* ab = (const GT*)A.a + p.b * A.a_sb + p.gate;
    const T* xb = (const T*)A.x + p.b * A.x_sb + p.c;
    const T* gb = (const T*)A.g + p.b * A.g_sb + p.c;
    T* ob = (T*)A.o + p.b * A.T * A.C + p.c;
    const int kept = (A.T + SC_KEEP - 1) / SC_KEEP;
    const int lim = min(p.len, end);
    // the gate's share of a row of dL/da: `wide` lanes hold it, `parts` such shares make it
    const int wide = min(min(A.LG, 1 << A.LC), 64);
    GT* db = (GT*)A.d_a + (SHARED ? p.b * A.T * A.J + p.gate : p.b * A.T * A.C + p.c);
    float* pb = A.gate_part + (int64_t)(p.k / wide) * A.B * A.T * A.J + p.b * A.T * A.J + p.gate;
    const bool part = A.LG > wide;
    const int64_t drow = SHARED ? A.J : A.C;
    const int tiles = stop > begin ? (stop - begin + tile - 1) / tile : 0;
    int flip = 0;
    // rows behind the last tile with a live step
    {
        float z[VC];
#pragma unroll
        for (int v = 0; v < VC; ++v) z[v] = 0.0f;
        for (int t = begin + tiles * tile + p.run; t < end; t += SC_THREADS >> A.LC) {
            if (p.on && A.o) st<T, VC>(ob + (int64_t)t * A.C, z);
            if (gates && p.col < A.cols) {
                if (!SHARED) st<GT, VC>(db + t * drow, z);
                else if (part) { if ((p.k & (wide - 1)) == 0) pb[t * drow] = 0.0f; }
                else if (p.k == 0) db[t * drow] = (GT)0.0f;
            }
        }
    }
    for (int q = tiles - 1; q >= 0; --q, flip ^= 1) {
        const int at = begin + q * tile, s0 = at + p.run * SC_U;
        const int64_t t0 = time_of(s0, p.len, A.reverse);
        Pack<GT, GV> ra[SC_U];
        Pack<T, VC> rx[SC_U], rg[SC_U];
        float hs[VC], h[VC], e[VC];
        const bool whole = __all(s0 + SC_U <= lim);
        float Ar[VC], Hr[VC], Er[VC];
#pragma unroll
        for (int v = 0; v < VC; ++v) { Ar[v] = 1.0f; Hr[v] = Er[v] = hs[v] = 0.0f; }
        fetch<GT, GV>(ra, ab + t0 * A.a_st, as, s0, lim, 1.0f, whole);
        fetch<T, VC>(rg, gb + t0 * A.g_st, gs, s0, A.g ? lim : SC_NONE, 0.0f, whole && A.g);
        fetch<T, VC>(rx, xb + t0 * A.x_st, xs, s0, gates ? lim : SC_NONE, 0.0f, whole && gates);
        if (gates && at < lim) {            // the state in front of the tile
            const float* from = at == 0 ? (A.h0 ? A.h0 + p.b * A.C + p.c : nullptr)
                                        : A.states + ((int64_t)p.b * kept + at / SC_KEEP) * A.C + p.c;
            if (from) for (int v = 0; v < VC; ++v) hs[v] = from[v];
        }
#pragma unroll
        for (int u = 0; u < SC_U; ++u)
#pragma unroll
            for (int v = 0; v < VC; ++v) {
                const float a = (float)ra[u].v[SHARED ? 0 : v];
                Hr[v] = fmaf(a, Hr[v], (float)rx[u].v[v]);
                Ar[v] *= a;
            }
#pragma unroll
        for (int u = SC_U - 1; u >= 0; --u)
#pragma unroll
            for (int v = 0; v < VC; ++v) Er[v] = (float)ra[u].v[SHARED ? 0 : v] * ((float)rg[u].v[v] + Er[v]);
        compose_both<VC>(Ar, Hr, Er, hs, carry, h, e, A.LC, buf[flip]);
        float prev[SC_U][VC], d[SC_U][VC], sum[SC_U];
#pragma unroll
        for (int u = 0; u < SC_U; ++u)
#pragma unroll
            for (int v = 0; v < VC; ++v) { prev[u][v] = h[v]; h[v] = fmaf((float)ra[u].v[SHARED ? 0 : v], h[v], (float)rx[u].v[v]); }
#pragma unroll
        for (int u = SC_U - 1; u >= 0; --u) {
            sum[u] = 0.0f;
#pragma unroll
            for (int v = 0; v < VC; ++v) {
                d[u][v] = (float)rg[u].v[v] + e[v];
                e[v] = (float)ra[u].v[SHARED ? 0 : v] * d[u][v];
                prev[u][v] *= d[u][v];              // dL/da of the channel
                if (VC > 1 && v == 0 && p.twice) continue;
                sum[u] += prev[u][v];
            }
        }
        const int64_t os = A.reverse ? -A.C : A.C, ds = A.reverse ? -drow : drow;
        if (whole) {
            if (A.o) {
                T* o = ob + t0 * A.C;
#pragma unroll
                for (int u = 0; u < SC_U; ++u, o += os) st<T, VC>(o, d[u]);
            }
            if (!SHARED && gates) {
                GT* o = db + t0 * drow;
#pragma unroll
                for (int u = 0; u < SC_U; ++u, o += ds) st<GT, VC>(o, prev[u]);
            }
        } else {
            int64_t row = t0;
#pragma unroll
            for (int u = 0; u < SC_U; ++u, row += A.reverse ? -1 : 1) {
                const bool live = s0 + u < lim;
                if (!live) {
                    sum[u] = 0.0f;
#pragma unroll
                    for (int v = 0; v < VC; ++v) d[u][v] = prev[u][v] = 0.0f;
                }
                if (live || (p.on && s0 + u < end)) {
                    const int64_t at_row = live ? row : s0 + u;         // behind the sequence: zeros, in place
                    if (A.o) st<T, VC>(ob + at_row * A.C, d[u]);
                    if (!SHARED && gates) st<GT, VC>(db + at_row * drow, prev[u]);
                }
            }
        }
        if (SHARED && gates) {
            int u0, n;
            bool mine;
            gate_sums(sum, wide, p.k, &u0, &n, &mine);
            // the live steps of the sequence, whether or not this lane has channels
            const int len = p.col >= A.cols ? 0 : A.lengths ? max(0, min(A.T, A.lengths[p.b])) : A.T;
            if (mine && p.col < A.cols) {
#pragma unroll
                for (int i = 0; i < SC_U; ++i)
                    if (i < n && s0 + u0 + i < end) {
                        const int sx = s0 + u0 + i;
                        const int64_t row = sx < len ? time_of(sx, len, A.reverse) : sx;
                        if (part) pb[row * drow] = sum[i]; else db[row * drow] = (GT)sum[i];
                    }
            }
        }
    }
    if (p.on && p.run == 0 && A.last && begin == 0)
        for (int v = 0; v < VC; ++v) A.last[p.b * A.C + p.c + v] = carry[v];
}

// dL/da of gates wider than a wavefront's share of a tile: the parts are added in one order
template <typename GT>
__global__ __launch_bounds__(256) void k_gate_sum(const float* __restrict__ part, GT* __restrict__ d_a, int64_t n, int parts) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.0f;
    for (int k = 0; k < parts; ++k) s += part[(int64_t)k * n + i];
    d_a[i] = (GT)s;
}

struct Shape {
    int VC, LC, S, parts;
    int64_t cols;
    int32_t stretch;
    int32_t G, LG, per_b;
    bool shared;
    int64_t sums_bytes, part_bytes;
};

inline int ceil_log2(int64_t x) { int k = 0; while (((int64_t)1 << k) < x) ++k; return k; }
inline int64_t up256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// The variant for a shape.
void shape_of(const nk_scan_opts* o, int bwd, Shape* s) {
    s->G = (int32_t)(o->C / o->gates);
    s->shared = s->G > 1;
    s->VC = o->C >= SC_VC ? SC_VC : 1;
    const int64_t unit = s->shared ? (s->G + s->VC - 1) / s->VC : (o->C + s->VC - 1) / s->VC;
    const int64_t row = unit * (s->shared ? o->gates : 1);
    // As many columns as a row has, up to a wavefront of them: neighbouring lanes then read neighbouring
    // channels, and narrow rows neighbouring steps (3038 x 3648 x 2: 123 us with 4 columns x 64 runs, 393 us
    // with 64 x 4; 64 channels: 32 x 8 and 64 x 4 the same).
    int LC = ceil_log2(row);
    LC = LC > 6 ? 6 : LC < 2 ? 2 : LC;
    const int runs_wanted = ceil_log2((o->T + SC_U - 1) / SC_U);
    if (runs_wanted < 8 - LC) LC = 8 - runs_wanted;
    if (LC == 7) LC = 6;
    s->LC = LC;
    const int lcol = 1 << LC;
    if (s->shared) {
        // the backward pass adds over a gate's columns with lane shuffles: a power of two of them, or whole wavefronts
        const int64_t p2 = (int64_t)1 << ceil_log2(unit);
        s->LG = (int32_t)(!bwd ? unit : p2 <= lcol ? p2 : (unit + lcol - 1) / lcol * lcol);
        s->per_b = (int32_t)(s->LG * o->gates);
    } else {
        s->LG = 1;
        s->per_b = (int32_t)unit;
    }
    s->cols = o->B * s->per_b;
    const int wide = lcol < 64 ? lcol : 64;
    s->parts = bwd && s->shared && s->LG > wide ? s->LG / wide : 1;
    const int64_t groups = (s->cols + lcol - 1) / lcol, tile = (int64_t)(SC_THREADS >> LC) * SC_U;
    const int64_t tiles = (o->T + tile - 1) / tile;
    // 128 groups: 70 us split, 147 whole; 256: 68 and 81; 384: 61 and 59 (forward + backward, 16 M elements).  To 1024
    // workgroups, four a CU: 512 are 10 to 25 % slower, 2048 up to 20 %.
    int64_t S = 1;
    if (groups < 384) { S = (1024 + groups - 1) / groups; if (S > tiles) S = tiles; }
    s->stretch = (int32_t)((tiles + S - 1) / S * tile);
    s->S = (int)((o->T + s->stretch - 1) / s->stretch);
    s->sums_bytes = s->S > 1 ? up256((int64_t)s->S * 2 * s->cols * s->VC * 4) : 0;
    s->part_bytes = bwd && s->parts > 1 ? (int64_t)s->parts * o->B * o->T * o->gates * 4 : 0;
}

int check(const nk_scan_opts* o, const char* who) {
    if (!o) NK_FAIL(NK_ERR_ARG, "%s: null options", who);
    if (o->B < 0 || o->T < 0 || o->C < 1 || o->gates < 1 || o->C % o->gates != 0)
        NK_FAIL(NK_ERR_ARG, "%s: B=%lld T=%lld C=%lld gates=%lld (gates divides C)", who, (long long)o->B, (long long)o->T, (long long)o->C, (long long)o->gates);
    if (o->dtype < NK_F32 || o->dtype > NK_F16 || (o->gate_dtype != o->dtype && o->gate_dtype != NK_F32))
        NK_FAIL(NK_ERR_UNSUPPORTED, "%s: dtype %d with gates of dtype %d (the same, or fp32)", who, o->dtype, o->gate_dtype);
    const int64_t most = (int64_t)1 << 29;
    if (o->C > most || o->T > most || o->B > most || o->B * o->C > ((int64_t)1 << 34))
        NK_FAIL(NK_ERR_UNSUPPORTED, "%s: B, T, C up to 2^29 and B * C up to 2^34", who);
    if (o->a_stride_b < 0 || o->a_stride_t < 0 || o->x_stride_b < 0 || o->x_stride_t < 0 || o->g_stride_b < 0 || o->g_stride_t < 0)
        NK_FAIL(NK_ERR_ARG, "%s: negative stride", who);
    return NK_OK;
}

template <typename T, typename GT, int VC, bool SHARED, bool BWD>
void launch(const ScanArgs& A, const Shape& s, hipStream_t st) {
    const unsigned groups = (unsigned)((s.cols + (1 << s.LC) - 1) >> s.LC);
    if (s.S > 1) {
        ScanArgs B = A;
        if (BWD) { B.x = A.g; B.x_sb = A.g_sb; B.x_st = A.g_st; }
        hipLaunchKernelGGL((k_scan_sum<T, GT, VC, SHARED, BWD>), dim3(groups, s.S - 1), dim3(SC_THREADS), 0, st, B);
    }
    if constexpr (BWD) hipLaunchKernelGGL((k_scan_bwd<T, GT, VC, SHARED>), dim3(groups, s.S), dim3(SC_THREADS), 0, st, A);
    else hipLaunchKernelGGL((k_scan_fwd<T, GT, VC, SHARED>), dim3(groups, s.S), dim3(SC_THREADS), 0, st, A);
}
template <typename T, typename GT, bool BWD>
void launch_vc(const ScanArgs& A, const Shape& s, hipStream_t st) {
    if (s.shared) launch<T, GT, SC_VC, true, BWD>(A, s, st);        // two channels at least
    else if (s.VC > 1) launch<T, GT, SC_VC, false, BWD>(A, s, st);
    else launch<T, GT, 1, false, BWD>(A, s, st);
}
template <bool BWD>
int launch_types(const nk_scan_opts* o, const ScanArgs& A, const Shape& s, hipStream_t st) {
    const bool g32 = o->gate_dtype == NK_F32;
    if (o->dtype == NK_F32) launch_vc<float, float, BWD>(A, s, st);
    else if (o->dtype == NK_BF16) { if (g32) launch_vc<__bf16, float, BWD>(A, s, st); else launch_vc<__bf16, __bf16, BWD>(A, s, st); }
    else { if (g32) launch_vc<_Float16, float, BWD>(A, s, st); else launch_vc<_Float16, _Float16, BWD>(A, s, st); }
    NK_CHECK_LAUNCH("k_scan");
    if (BWD && s.parts > 1 && A.d_a) {
        const int64_t n = o->B * o->T * o->gates;
        const dim3 grid((unsigned)((n + 255) / 256));
        if (g32) hipLaunchKernelGGL(k_gate_sum<float>, grid, dim3(256), 0, st, A.gate_part, (float*)A.d_a, n, s.parts);
        else if (o->dtype == NK_BF16) hipLaunchKernelGGL(k_gate_sum<__bf16>, grid, dim3(256), 0, st, A.gate_part, (__bf16*)A.d_a, n, s.parts);
        else hipLaunchKernelGGL(k_gate_sum<_Float16>, grid, dim3(256), 0, st, A.gate_part, (_Float16*)A.d_a, n, s.parts);
        NK_CHECK_LAUNCH("k_gate_sum");
    }
    return NK_OK;
}

ScanArgs args_of(const nk_scan_opts* o, const Shape& s, void* ws) {
    ScanArgs A = {};
    A.lengths = o->lengths; A.T = (int32_t)o->T; A.C = o->C; A.B = o->B; A.J = o->gates;
    A.a_sb = o->a_stride_b; A.a_st = o->a_stride_t; A.x_sb = o->x_stride_b; A.x_st = o->x_stride_t;
    A.g_sb = o->g_stride_b; A.g_st = o->g_stride_t;
    A.stretch = s.stretch; A.cols = s.cols; A.G = s.G; A.LG = s.LG; A.per_b = s.per_b; A.LC = s.LC; A.reverse = o->reverse != 0;
    A.sums = (float*)ws; A.gate_part = (float*)((char*)ws + s.sums_bytes);
    return A;
}

int64_t bytes_of(const Shape& s) { return s.sums_bytes + s.part_bytes; }

int check_launch(const nk_scan_opts* o, const Shape& s, const void* workspace, int64_t workspace_bytes, const char* who) {
    if (((s.cols + (1 << s.LC) - 1) >> s.LC) >= (1 << 24) || (s.parts > 1 && o->B * o->gates > ((int64_t)1 << 31) / o->T))
        NK_FAIL(NK_ERR_UNSUPPORTED, "%s: more columns than the 2^32 threads of a launch", who);
    if (bytes_of(s) > workspace_bytes || (bytes_of(s) && (!workspace || ((uintptr_t)workspace & 255))))
        NK_FAIL(NK_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", who, (long long)workspace_bytes, (long long)bytes_of(s));
    return NK_OK;
}

}  // namespace

extern "C" int64_t nk_gated_scan_workspace_bytes(const nk_scan_opts* o, int backward) {
    const int rc = check(o, "nk_gated_scan_workspace_bytes");
    if (rc < 0) return rc;
    if (o->B == 0 || o->T == 0) return 0;
    Shape s;
    shape_of(o, backward, &s);
    return bytes_of(s);
}

extern "C" int64_t nk_gated_scan_states_bytes(const nk_scan_opts* o) {
    const int rc = check(o, "nk_gated_scan_states_bytes");
    if (rc < 0) return rc;
    return o->B * ((o->T + SC_KEEP - 1) / SC_KEEP) * o->C * 4;
}

extern "C" int nk_gated_scan_fwd(const nk_scan_opts* o, const void* a, const void* x, const float* h0, void* h, float* h_last,
                                 float* states, void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check(o, "nk_gated_scan_fwd");
    if (rc < 0) return rc;
    if (o->B == 0) return NK_OK;
    if (o->T == 0) NK_FAIL(NK_ERR_ARG, "nk_gated_scan_fwd: T = 0 (the state does not change: nothing to launch)");
    if (!a || !x || !h) NK_FAIL(NK_ERR_ARG, "nk_gated_scan_fwd: null pointer");
    Shape s;
    shape_of(o, 0, &s);
    if ((rc = check_launch(o, s, workspace, workspace_bytes, "nk_gated_scan_fwd")) < 0) return rc;
    ScanArgs A = args_of(o, s, workspace);
    A.a = a; A.x = x; A.first = h0; A.o = h; A.last = h_last; A.states = states;
    return launch_types<false>(o, A, s, nk_stream(stream));
}

extern "C" int nk_gated_scan_bwd(const nk_scan_opts* o, const void* a, const void* x, const float* states, const float* h0,
                                 const void* d_h, const float* d_h_last, void* d_a, void* d_x, float* d_h0, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
    int rc = check(o, "nk_gated_scan_bwd");
    if (rc < 0) return rc;
    if (o->B == 0) return NK_OK;
    if (o->T == 0) NK_FAIL(NK_ERR_ARG, "nk_gated_scan_bwd: T = 0");
    if (!a || (d_a && (!x || !states)) || (!d_a && !d_x && !d_h0)) NK_FAIL(NK_ERR_ARG, "nk_gated_scan_bwd: null pointer");
    Shape s;
    shape_of(o, 1, &s);
    if ((rc = check_launch(o, s, workspace, workspace_bytes, "nk_gated_scan_bwd")) < 0) return rc;
    ScanArgs A = args_of(o, s, workspace);
    A.a = a; A.x = x; A.g = d_h; A.h0 = h0; A.states = (float*)states; A.first = d_h_last; A.o = d_x; A.d_a = d_a; A.last = d_h0;
    return launch_types<true>(o, A, s, nk_stream(stream));
}
