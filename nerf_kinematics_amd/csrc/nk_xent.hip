// Softmax cross entropy of a linear head, without ever holding the logits:
//
//   z_(n,v) = <hidden_n, weight_v>        loss_n = lse_n - z_(n,t_n),  lse_n = log sum_v exp z_(n,v)
//   dz_(n,v) = c_n (exp(z_(n,v) - lse_n) - [v = t_n])      d_hidden = dz weight,  d_weight = dz^T hidden
//
// Forward: one product weight x hidden^T on the matrix cores whose tiles end in registers; a tile leaves
// the maximum and the sum of exponentials of its vocabulary rows for every token (8 bytes per token and tile),
// a second kernel joins them.  Backward: the vocabulary is walked in pieces; per piece the logits are
// computed again, turned into dz (rounded once to the operands' type: the two products that follow take it as
// a matrix operand) and multiplied into d_weight's rows of the piece and onto d_hidden's fp32 sums.
//
// All products have the form C[m][n] = sum_k A[m][k] B[n][k].  For 16-bit types an operand may have k along its rows
// or along its columns, so weight and dz serve both products as they are; fp32 has k contiguous in both operands:
// where the mathematics wants the other order (weight^T, hidden^T) a piece is transposed once by a copy, and dz
// is written in both orders by the tile that computes it.
//
// What bounds it (MI355X; a library product of 8192^3 reaches 1 383 TFLOP/s in bf16): power and the way to memory.  The
// matrix units are 55 % busy at 2.1 GHz, LDS 21 %; over data that stays in the caches the loop is a quarter faster.
// 8192 x 2048 x 65536 in bf16, forward and backward: 7.0 to 7.3 ms from card to card, 1 204 to 1 257 TFLOP/s over the
// four products (the logits twice); forward alone 1.75 ms.  4096 x 1024 x 32003: 1.0 ms, the epilogue of dz costs more
// where k is short.  16 x 1024 x 50000 forward: 24 us, 4.3 TB/s of weight.  Small calls: launches.
#include "nk_common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// Scratch of a piece (its dz, and the copies of its rows), unless the caller names one.  Kernel time of a training pass of 8192 x 2048 x 65536 /
// 4096 x 1024 x 32003: 64 MB 8.4 / 1.41 ms, 128 MB 7.75 / 1.25, 256 MB 7.64 / 1.20, 512 MB 7.61 / 1.25.
enum { XENT_PIECE_MB = 256 };

constexpr float LOG2E = 1.4426950408889634f;

// ---- operand types: 16 bytes of k per lane and fragment --------------------------------------
template <typename T> struct Op;
template <> struct Op<__bf16> {
    static constexpr float SCALE = 1.0f;    // dz is multiplied by this before it is rounded
    NK_D static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Op<_Float16> {
    // softmax values of a large vocabulary fall below fp16's smallest normal value (2^-14): 2^14 of headroom
    // keeps |dz| <= 1 at most 16 384 and makes 2^-28 the smallest normal one
    static constexpr float SCALE = 16384.0f;
    NK_D static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct Op<float> {
    static constexpr float SCALE = 1.0f;
    // element j of every lane's four is one 16x16x4 product; any order of k serves as long as A and B agree
    NK_D static f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};

// ---- the tile product -------------------------------------------------------------------------
// A workgroup computes BM x BN of C with WGM x WGN wavefronts, each TM x TN tiles of 16 x 16 (with 32 x 32 x 16
// instructions the largest products take 6 % longer: half as many independent sums).  k advances
// by 128 bytes of every row; the rows of a step are loaded straight into LDS (16 bytes a lane, 8 rows a
// wavefront and instruction) STAGES - 1 steps ahead.  Row r keeps its eight 16-byte chunks in the order
// chunk ^ (r & 7), so that the 16 rows a fragment read touches fall on different banks; the order is made by the
// source address, the LDS side of such a load being fixed.  Rows behind the matrix and the end of k
// are outside the buffer resource's range and arrive as zeros.
//
// An operand may also come with k along its rows ("k-major": A[k][m]), for 16-bit types: a step is then 64 rows of BM
// (BN) elements, and the fragments are read with the transposing LDS read, which hands the 16 lanes of a group the
// columns of four rows.  Chunk c of row k lies at c ^ f(k), f even and different for the rows that a wavefront reads at
// once.  This takes the products of the backward pass straight from dz [token][row], weight and hidden: with
// transposed copies of the three, 8192 x 2048 x 65536 took 7.64 ms of kernels and 4096 x 1024 x 32003 1.20 ms.
struct Mat { const char* p; int64_t rows, stride, width; };      // bytes: stride, a multiple of 16, as is p; width of a row that may be read

template <int BM_, int BN_, int WGM_, int WGN_, int STAGES_> struct Cfg {
    static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, STAGES = STAGES_;
    static constexpr int WAVES = WGM * WGN, THREADS = WAVES * 64;
    static constexpr int TM = BM / WGM / 16, TN = BN / WGN / 16;
    static constexpr int STAGE_BYTES = (BM + BN) * 128, LDS = STAGE_BYTES * STAGES;
    static constexpr int PA = BM / 8 / WAVES, PB = BN / 8 / WAVES, PIECES = PA + PB;    // load instructions per wavefront and step
    static_assert(PA * 8 * WAVES == BM && PB * 8 * WAVES == BN, "every wavefront loads the same share of A and of B");
};

NK_D void lds_load(uint32_t lds_at, u32x4 srd, uint32_t voff, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(lds_at), "v"(voff), "s"(srd), "s"(soff) : "memory");
}
template <int N> NK_D void wait_loads_and_meet() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory"); }

NK_D u32x4 resource(const char* p, int64_t bytes) {
    const uint64_t a = (uint64_t)p;
    u32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) & 0xFFFF;
    r[2] = __builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : bytes > 0x7FFFFFFF ? 0x7FFFFFFF : bytes));
    r[3] = 0x00027000;
    return r;
}

// Place of chunk c of row k of a k-major operand of CH chunks a row.
template <int CH> NK_D int k_major_chunk(int c, int k) { return c ^ ((2 * ((k & 3) | ((k >> 3) & 3) << 2)) & (CH - 2)); }

// One tile's product in two parts: begin() starts the loads of the first steps, run() does the rest.  The
// LDS of the operands has to be idle at begin().  KA, KB: the operand is k-major.
template <typename T, class C, bool KA = false, bool KB = false> struct TileProduct {
    static_assert(sizeof(T) == 2 || !(KA || KB), "the transposing read takes 16-bit elements");
    // What a wavefront loads of an operand: P instructions a step.
    template <int P, bool K> struct Source {
        u32x4 r;
        uint32_t v[P];
        uint64_t base;              // k-major: address of the next step's first row
        int left;                   // and the rows that are left from there on
        uint32_t stride, width;
        template <int ROWS> NK_D void begin(const Mat& M, int64_t at, int64_t row_bytes, int wave, int lane) {
            if constexpr (K) {
                constexpr int CH = ROWS / 8;
                const uint64_t a = (uint64_t)(M.p + at * sizeof(T));
                base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)) << 32;
                left = __builtin_amdgcn_readfirstlane((int)M.rows);
                stride = __builtin_amdgcn_readfirstlane((int)M.stride);
                width = __builtin_amdgcn_readfirstlane((int)(M.width - at * (int64_t)sizeof(T)));
                r[3] = 0x00027000;
                asm volatile("s_nop 4" : "+s"(base), "+s"(left), "+s"(stride), "+s"(width));    // scalars written by the vector unit, read by loads issued from asm
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int l = (wave * P + i) * 64 + lane, k = l / CH;
                    v[i] = (uint32_t)k * (uint32_t)M.stride + (uint32_t)k_major_chunk<CH>(l % CH, k) * 16;
                }
            } else {
                r = resource(M.p + at * M.stride, (M.rows - at - 1) * M.stride + row_bytes);
                asm volatile("s_nop 4" : "+s"(r));
                // this lane's place in a load instruction: row (lane / 8) of eight, chunk of the row by the order above
                const int lrow = lane >> 3, lchunk = (lane & 7) ^ (lrow & 7);
#pragma unroll
                for (int i = 0; i < P; ++i) v[i] = (uint32_t)((wave * P + i) * 8 + lrow) * (uint32_t)M.stride + lchunk * 16;
            }
        }
        // The loads of step s, behind the end of k as well (out of range: no memory is touched), so that the loop has no
        // branches and the number of loads in flight is always the same.
        NK_D void issue(uint32_t at, int s, uint32_t out, int wave) {
            if constexpr (K) {
                const int rows = left < 64 ? left : 64;
                r[0] = (uint32_t)base; r[1] = (uint32_t)(base >> 32) & 0xFFFF; r[2] = rows > 0 ? (uint32_t)(rows - 1) * stride + width : 0;
                base += (uint64_t)stride * 64; left -= 64;
#pragma unroll
                for (int i = 0; i < P; ++i) lds_load(at + (wave * P + i) * 1024, r, v[i], 0);
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) lds_load(at + (wave * P + i) * 1024, r, v[i] | out, (uint32_t)s * 128);
            }
        }
    };
    // Where a lane finds its fragments of an operand of ROWS rows (columns, if k-major): TILES of 16 from `first` on.
    template <int ROWS, int TILES, bool K> struct Fragments {
        const char* p;
        int x0, x1;
        int c[K ? TILES : 1];
        NK_D Fragments(const char* lds, int first, int lane) {
            if constexpr (K) {
                constexpr int CH = ROWS / 8;
                const int q = lane >> 4, j = lane & 15, k = 8 * q + (j >> 2);
                p = lds + k * CH * 16 + (j & 1) * 8;
                x0 = 0; x1 = 32 * CH * 16;
#pragma unroll
                for (int i = 0; i < TILES; ++i) c[i] = k_major_chunk<CH>(first / 8 + 2 * i + ((j >> 1) & 1), k) * 16;
            } else {
                const int frow = lane & 15, fchunk = lane >> 4;
                p = lds + (first + frow) * 128;
                x0 = (fchunk ^ (frow & 7)) * 16; x1 = ((fchunk + 4) ^ (frow & 7)) * 16;
                c[0] = 0;
            }
        }
        NK_D void read(u32x4 (&f)[TILES], int at, int x) const {
            const char* a = p + at + x;
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                if constexpr (K) {
                    constexpr int CH = ROWS / 8;
                    typedef __attribute__((ext_vector_type(4))) short s16x4;
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((NK_LDS s16x4*)(a + c[i])));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((NK_LDS s16x4*)(a + c[i] + 4 * CH * 16)));
                    f[i] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                } else {
                    f[i] = *(const u32x4*)(a + i * 2048);
                }
            }
        }
    };

    Source<C::PA, KA> sa;
    Source<C::PB, KB> sb;
    uint32_t lds0;
    int steps, last, wave;
    char* lds;

    NK_D void issue(int s, int slot) {
        const uint32_t out = s < last ? 0u : 0x80000000u;
        const uint32_t at = lds0 + slot * C::STAGE_BYTES;
        sa.issue(at, s, out, wave);
        sb.issue(at + C::BM * 128, s, out, wave);
    }

    NK_D void begin(const Mat& A, const Mat& B, int64_t m0, int64_t n0, int64_t kbytes, char* lds_) {
        const int lane = threadIdx.x & 63;
        lds = lds_;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        // the last byte that a row of this stretch of k may be read to; rows and steps behind it arrive as zeros
        const int64_t row_bytes = (kbytes + 15) & ~(int64_t)15;
        sa.template begin<C::BM>(A, m0, row_bytes, wave, lane);
        sb.template begin<C::BN>(B, n0, row_bytes, wave, lane);
        lds0 = (uint32_t)(uintptr_t)(NK_LDS char*)lds;
        steps = (int)((kbytes + 127) / 128);
        const int lchunk = (lane & 7) ^ ((lane >> 3) & 7);
        last = (int)((kbytes - lchunk * 16 + 127) / 128);       // steps in which this lane's chunk is inside k
#pragma unroll
        for (int s = 0; s < C::STAGES; ++s) issue(s, s);
    }

    NK_D void run(f32x4 (&acc)[C::TM][C::TN]) {
        const int lane = threadIdx.x & 63, wm = wave / C::WGN, wn = wave % C::WGN;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int j = 0; j < C::TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
        const Fragments<C::BM, C::TM, KA> fa(lds, wm * C::TM * 16, lane);
        const Fragments<C::BN, C::TN, KB> fb(lds + C::BM * 128, wn * C::TN * 16, lane);
        u32x4 a0[C::TM], b0[C::TN], a1[C::TM], b1[C::TN];
        auto read = [&](u32x4 (&a)[C::TM], u32x4 (&b)[C::TN], int slot, bool second) {
            fb.read(b, slot * C::STAGE_BYTES, second ? fb.x1 : fb.x0);
            fa.read(a, slot * C::STAGE_BYTES, second ? fa.x1 : fa.x0);
        };
        auto multiply = [&](const u32x4 (&a)[C::TM], const u32x4 (&b)[C::TN]) {
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int j = 0; j < C::TN; ++j) acc[i][j] = Op<T>::mma(a[i], b[j], acc[i][j]);
            // one LDS read between every few products (0x100: LDS read, 0x008: matrix product)
            constexpr int READS = C::TM * (KA ? 2 : 1) + C::TN * (KB ? 2 : 1), EACH = C::TM * C::TN / READS;
#pragma unroll
            for (int q = 0; q < READS; ++q) {
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, EACH > 0 ? EACH : 1, 0);
            }
        };
        constexpr int S = C::STAGES;
        wait_loads_and_meet<(S - 1) * C::PIECES>();
        read(a0, b0, 0, false);
        int slot = 0;
        for (int s = 0; s < steps; ++s) {
            const int next = slot + 1 == S ? 0 : slot + 1;
            // the second half of the step's fragments arrives while the first is multiplied
            read(a1, b1, slot, true);
            multiply(a0, b0);
            __builtin_amdgcn_sched_barrier(0);
            // everyone has read this step; the next one has landed when at most the loads behind it are outstanding
            wait_loads_and_meet<(S - 2) * C::PIECES>();
            issue(s + S, slot);
            __builtin_amdgcn_sched_barrier(0);
            read(a0, b0, next, false);
            multiply(a1, b1);
            __builtin_amdgcn_sched_barrier(0);
            slot = next;
        }
        wait_loads_and_meet<0>();           // nothing is in flight into LDS any more: it is free
    }
};

template <typename T, class C, bool KA = false, bool KB = false>
NK_D void tile_product(const Mat& A, const Mat& B, int64_t m0, int64_t n0, int64_t kbytes, char* lds, f32x4 (&acc)[C::TM][C::TN]) {
    TileProduct<T, C, KA, KB> p;
    p.begin(A, B, m0, n0, kbytes, lds);
    p.run(acc);
}

// Workgroup -> tile.  Consecutive workgroups go to the eight XCDs in turn; every XCD gets a contiguous
// range of tiles, walked in patches of 8 rows of tiles, so that what its L2 holds is used again.
NK_D void tile_of(int64_t id, int64_t mt, int64_t nt, int64_t* m, int64_t* n) {
    const int64_t total = mt * nt;
    const int64_t per = total / 8, extra = total % 8, x = id % 8;
    const int64_t t = x * per + (x < extra ? x : extra) + id / 8;
    const int64_t band = 8 * nt, b = t / band, left = mt - b * 8, h = left < 8 ? left : 8;
    const int64_t r = t - b * band;
    *m = b * 8 + r % h;
    *n = r / h;
}

// ---- forward ----------------------------------------------------------------------------------
struct LseArgs {
    Mat w, h;
    int64_t kbytes, v0, N;                 // rows v0 .. of the vocabulary are w's rows 0 ..
    const int64_t* target;
    float2* part; int64_t part0;            // [tile of vocabulary][token]: maximum, sum of exponentials
    float* zt;                              // logit of the target
};

// The workgroups stay and take tiles in turn: the loads of the next tile's first steps are under way while
// this one's registers are reduced.
template <typename T, class C>
__global__ __launch_bounds__(C::THREADS) void k_xent_lse(const LseArgs g) {
    __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
    __shared__ float2 meet[C::WGM][C::BN];
    const int64_t mt = (g.w.rows + C::BM - 1) / C::BM, nt = (g.N + C::BN - 1) / C::BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / C::WGN, wn = wave % C::WGN;
    int64_t mi, ni;
    tile_of(blockIdx.x, mt, nt, &mi, &ni);
    TileProduct<T, C> p;
    p.begin(g.w, g.h, mi * C::BM, ni * C::BN, g.kbytes, lds);
    for (int64_t tile = blockIdx.x; tile < mt * nt; tile += gridDim.x) {
        f32x4 acc[C::TM][C::TN];
        p.run(acc);
        const int64_t m_at = mi, n_at = ni;
        if (tile + gridDim.x < mt * nt) {
            tile_of(tile + gridDim.x, mt, nt, &mi, &ni);
            p.begin(g.w, g.h, mi * C::BM, ni * C::BN, g.kbytes, lds);
        }
        const int64_t row0 = m_at * C::BM + wm * C::TM * 16 + 4 * (lane >> 4);       // of w; rows row0 + 16 i + e
        const int live = (int)(g.w.rows - row0 < 16 * C::TM ? g.w.rows - row0 : 16 * C::TM);        // rows from row0 on that this wavefront has
#pragma unroll
        for (int j = 0; j < C::TN; ++j) {
            const int col = wn * C::TN * 16 + j * 16 + (lane & 15);
            const int64_t n = n_at * C::BN + col;
            const int64_t t64 = n < g.N ? g.target[n] - g.v0 - row0 : -1;
            const int t = t64 < 0 || t64 >= live ? -1 : (int)t64;
            float m = -__builtin_inff(), zt = 0.0f;
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (16 * i + e >= live) acc[i][j][e] = -__builtin_inff();
                    if (16 * i + e == t) zt = acc[i][j][e];
                    m = fmaxf(m, acc[i][j][e]);
                }
            if (t >= 0 && (t & 15) < 4) g.zt[n] = zt;        // a lane holds rows 0..3 of every 16
            const float ms = m == -__builtin_inff() ? 0.0f : m;
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < C::TM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f((acc[i][j][e] - ms) * LOG2E);
#pragma unroll
            for (int off = 16; off < 64; off <<= 1) {
                const float mo = __shfl_xor(m, off, 64), so = __shfl_xor(s, off, 64);
                const float mn = fmaxf(m, mo), mz = mn == -__builtin_inff() ? 0.0f : mn;
                s = s * __builtin_amdgcn_exp2f((m - mz) * LOG2E) + so * __builtin_amdgcn_exp2f((mo - mz) * LOG2E);
                m = mn;
            }
            if (lane < 16) meet[wm][col] = make_float2(m, s);
        }
        // LDS only: the loads of the next tile stay in flight
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        for (int c = threadIdx.x; c < C::BN; c += C::THREADS) {
            const int64_t n = n_at * C::BN + c;
            if (n >= g.N) break;
            float m = meet[0][c].x, s = meet[0][c].y;
#pragma unroll
            for (int w = 1; w < C::WGM; ++w) {
                const float mo = meet[w][c].x, so = meet[w][c].y;
                const float mn = fmaxf(m, mo), mz = mn == -__builtin_inff() ? 0.0f : mn;
                s = s * __builtin_amdgcn_exp2f((m - mz) * LOG2E) + so * __builtin_amdgcn_exp2f((mo - mz) * LOG2E);
                m = mn;
            }
            g.part[(g.part0 + m_at) * g.N + n] = make_float2(m, s);
        }
    }
}

NK_D float2 join(float2 a, float2 b) {
    const float mn = fmaxf(a.x, b.x), mz = mn == -__builtin_inff() ? 0.0f : mn;
    return make_float2(mn, a.y * expf(a.x - mz) + b.y * expf(b.x - mz));
}

// lse and loss of TOK tokens a workgroup: 256 / TOK threads a token take the tiles in turn, then meet in one order.
// sums: NULL, or per workgroup the sum of its losses and how many of its tokens count.
template <int TOK>
__global__ __launch_bounds__(256) void k_xent_join(const float2* __restrict__ part, int64_t tiles, int64_t N, int64_t V,
                                                   const int64_t* __restrict__ target, int64_t ignore, const float* __restrict__ zt,
                                                   float* __restrict__ lse, float* __restrict__ loss, double2* __restrict__ sums) {
    __shared__ float2 meet[256];
    constexpr int TH = 256 / TOK;
    const int c = threadIdx.x % TOK, q = threadIdx.x / TOK;
    const int64_t n = (int64_t)blockIdx.x * TOK + c;
    float2 r = make_float2(-__builtin_inff(), 0.0f);
    if (n < N)
        for (int64_t t = q; t < tiles; t += TH) r = join(r, part[t * N + n]);
    meet[q * TOK + c] = r;
    __syncthreads();
    for (int half = TH / 2; half > 0; half >>= 1) {
        if (q < half) meet[q * TOK + c] = join(meet[q * TOK + c], meet[(q + half) * TOK + c]);
        __syncthreads();
    }
    double total = 0.0, count = 0.0;
    if (q == 0 && n < N) {
        const float l = meet[c].x + logf(meet[c].y);
        const int64_t t = target[n];
        const float mine = t == ignore ? 0.0f : (t < 0 || t >= V) ? __builtin_nanf("") : l - zt[n];
        lse[n] = l;
        loss[n] = mine;
        total = (double)mine; count = t != ignore ? 1.0 : 0.0;
    }
    if (!sums) return;
    for (int off = TOK / 2; off > 0; off >>= 1) { total += __shfl_xor(total, off, 64); count += __shfl_xor(count, off, 64); }
    if (threadIdx.x == 0) sums[blockIdx.x] = make_double2(total, count);
}

// Sum or mean over the tokens that count, in one order, by one workgroup of 1024 threads.
NK_D void reduce_losses(double s, double k, int mean, float* out) {
    __shared__ double sums[16], counts[16];
    for (int off = 32; off > 0; off >>= 1) { s += __shfl_xor(s, off, 64); k += __shfl_xor(k, off, 64); }
    if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6] = s; counts[threadIdx.x >> 6] = k; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) { s += sums[w]; k += counts[w]; }
        out[0] = (float)(mean ? s / (k > 0.0 ? k : 1.0) : s);
    }
}

// k_xent_join and k_xent_reduce in one launch where a thread per token is enough (N <= 1024, few tiles)
__global__ __launch_bounds__(1024) void k_xent_join_reduce(const float2* __restrict__ part, int tiles, int N, int64_t V, const int64_t* __restrict__ target,
                                                           int64_t ignore, const float* __restrict__ zt, int mean, float* __restrict__ lse,
                                                           float* __restrict__ loss, float* __restrict__ out) {
    const int n = threadIdx.x;
    float l = 0.0f;
    double k = 0.0;
    if (n < N) {
        float2 r = part[n];
#pragma unroll 4
        for (int t = 1; t < tiles; ++t) r = join(r, part[(int64_t)t * N + n]);
        const float e = r.x + logf(r.y);
        const int64_t t = target[n];
        l = t == ignore ? 0.0f : (t < 0 || t >= V) ? __builtin_nanf("") : e - zt[n];
        k = t != ignore ? 1.0 : 0.0;
        lse[n] = e;
        loss[n] = l;
    }
    reduce_losses((double)l, k, mean, out);
}

__global__ __launch_bounds__(1024) void k_xent_reduce(const double2* __restrict__ sums, int64_t n, int mean, float* __restrict__ out) {
    double s = 0.0, k = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < n; i += 1024) { s += sums[i].x; k += sums[i].y; }
    reduce_losses(s, k, mean, out);
}

// ---- backward ---------------------------------------------------------------------------------
// Row factors of dz and the factor that is left for the end: the products see dz with |c| <= 1.
//   mean / sum: c = 1 for tokens that count, rest = d_loss / count or d_loss
//   none:       c = d_loss_n / rest with rest the power of two above the largest finite |d_loss|
struct Tally { int count; uint32_t peak; };     // tokens that count, bits of the largest finite |d_loss| among them
enum { TALLY_TOKENS = 4096 };

template <int THREADS> NK_D Tally tally(const int64_t* target, int64_t n0, int64_t n1, int64_t ignore, int reduction, const float* d_loss) {
    Tally r = {0, 0};
#pragma unroll 4
    for (int64_t n = n0 + threadIdx.x; n < n1; n += THREADS)
        if (target[n] != ignore) {
            ++r.count;
            if (reduction == NK_REDUCE_NONE) {
                const uint32_t b = __float_as_uint(d_loss[n]) & 0x7FFFFFFFu;
                if (b < 0x7F800000u) r.peak = max(r.peak, b);       // an infinite one would shrink all others to nothing
            }
        }
    return r;
}
// over the workgroup; the result is in thread 0
template <int THREADS> NK_D Tally meet_tally(Tally r) {
    __shared__ Tally meet[THREADS / 64];
    for (int off = 32; off > 0; off >>= 1) { r.count += __shfl_xor(r.count, off, 64); r.peak = max(r.peak, (uint32_t)__shfl_xor((int)r.peak, off, 64)); }
    if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = r;
    __syncthreads();
    if (threadIdx.x == 0) for (int w = 1; w < THREADS / 64; ++w) { r.count += meet[w].count; r.peak = max(r.peak, meet[w].peak); }
    return r;
}

// Where one workgroup would take long over the tokens, TALLY_TOKENS of them a workgroup first; k_xent_factors then
// adds these up in every workgroup, each of which writes the factors of as many tokens.  196 608 tokens: 10 us instead of 66.
__global__ __launch_bounds__(1024) void k_xent_tally(const int64_t* __restrict__ target, int64_t N, int64_t ignore, int reduction,
                                                     const float* __restrict__ d_loss, Tally* __restrict__ out) {
    const int64_t n0 = (int64_t)blockIdx.x * TALLY_TOKENS, n1 = n0 + TALLY_TOKENS < N ? n0 + TALLY_TOKENS : N;
    const Tally r = meet_tally<1024>(tally<1024>(target, n0, n1, ignore, reduction, d_loss));
    if (threadIdx.x == 0) out[blockIdx.x] = r;
}

struct FactorArgs {
    const int64_t* target; int64_t N, V, ignore;
    int reduction, n_parts;
    const float* d_loss;
    const Tally* parts;         // NULL: every workgroup counts all tokens itself
    float* c; float* rest;
};
template <int THREADS> NK_D void factors(const FactorArgs& f, int64_t block, int64_t blocks) {
    __shared__ float unit;
    Tally r = {0, 0};
    if (f.parts) {
        for (int i = threadIdx.x; i < f.n_parts; i += THREADS) { r.count += f.parts[i].count; r.peak = max(r.peak, f.parts[i].peak); }
    } else {
        r = tally<THREADS>(f.target, 0, f.N, f.ignore, f.reduction, f.d_loss);
    }
    r = meet_tally<THREADS>(r);
    if (threadIdx.x == 0) {
        float left;
        if (f.reduction == NK_REDUCE_NONE) {
            const int e = min(max((int)(r.peak >> 23) + 1, 27), 227);          // 2^-100 .. 2^100; infinities and NaN stay in c
            unit = __uint_as_float((uint32_t)(254 - e) << 23);
            left = __uint_as_float((uint32_t)e << 23);
        } else {
            unit = 1.0f;
            left = f.reduction == NK_REDUCE_MEAN ? f.d_loss[0] / (float)(r.count > 0 ? r.count : 1) : f.d_loss[0];
        }
        if (block == 0) *f.rest = left;
    }
    __syncthreads();
#pragma unroll 4
    for (int64_t n = block * THREADS + threadIdx.x; n < f.N; n += blocks * THREADS) {
        const int64_t t = f.target[n];
        f.c[n] = t == f.ignore ? 0.0f : (t < 0 || t >= f.V) ? __builtin_nanf("") : f.reduction == NK_REDUCE_NONE ? f.d_loss[n] * unit : 1.0f;
    }
}
__global__ __launch_bounds__(1024) void k_xent_factors(const FactorArgs f) { factors<1024>(f, blockIdx.x, gridDim.x); }

struct DzArgs {
    Mat w, h;
    int64_t kbytes, v0, N;
    const int64_t* target;
    const float* lse; const float* c;
    void* dz; int64_t dz_ld;                // [token][row of the piece], zero up to dz_ld
    void* dzt; int64_t dzt_ld;              // fp32 only: [row of the piece][token], zero up to dzt_ld
};

// dz leaves in the orders that the products take: one for 16-bit types, both for fp32
template <typename T> constexpr bool BOTH_ORDERS = sizeof(T) == 4;

template <typename T, class C>
__global__ __launch_bounds__(C::THREADS) void k_xent_dz(const DzArgs g) {
    __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
    int64_t mi, ni;
    // up to the padded token count: those columns of dzt have to be zero
    tile_of(blockIdx.x, (g.w.rows + C::BM - 1) / C::BM, ((BOTH_ORDERS<T> ? g.dzt_ld : g.N) + C::BN - 1) / C::BN, &mi, &ni);
    f32x4 acc[C::TM][C::TN];
    tile_product<T, C>(g.w, g.h, mi * C::BM, ni * C::BN, g.kbytes, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / C::WGN, wn = wave % C::WGN;
    const int r0 = wm * C::TM * 16 + 4 * (lane >> 4), c0 = wn * C::TN * 16 + (lane & 15);      // this lane's first row and column of the tile
    const int live = (int)(g.w.rows - mi * C::BM < C::BM ? g.w.rows - mi * C::BM : C::BM);
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
        const int64_t n = ni * C::BN + c0 + 16 * j;
        const bool in = n < g.N;
        const int64_t t64 = in ? g.target[n] - g.v0 - mi * C::BM : -1;
        const int t = t64 < 0 || t64 >= C::BM ? -1 : (int)t64;
        const float lse = in ? g.lse[n] : 0.0f, c = in ? g.c[n] : 0.0f, cs = c * Op<T>::SCALE;
#pragma unroll
        for (int i = 0; i < C::TM; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r0 + 16 * i + e;
                float p = __builtin_amdgcn_exp2f((acc[i][j][e] - lse) * LOG2E);
                if (r == t) p -= 1.0f;
                acc[i][j][e] = (c == 0.0f || r >= live) ? 0.0f : p * cs;
            }
    }
    if constexpr (!BOTH_ORDERS<T>) {
        // The tile leaves through LDS, as whole rows of it: straight from the registers a store would touch 16
        // rows with 32 bytes each.  Rows of 16-byte chunks, chunk ^ (row & mask) against bank conflicts.
        typedef __attribute__((ext_vector_type(4))) T vec;
        static_assert(C::BM * C::BN * 2 <= C::LDS, "the tile fits the operands' LDS");
        constexpr int CH = C::BM / 8;           // [token][row]
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int i = 0; i < C::TM; ++i) {
                const int r = r0 + 16 * i, c = c0 + 16 * j;
                vec w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = (T)acc[i][j][e];
                *(u32x2*)(lds + (c * CH + ((r >> 3) ^ (c & (CH - 1)))) * 16 + (r & 4) * 2) = __builtin_bit_cast(u32x2, w);
            }
        __syncthreads();
        T* dz = (T*)g.dz + mi * C::BM;
#pragma unroll 4
        for (int q = threadIdx.x; q < C::BN * CH; q += C::THREADS) {
            const int c = q / CH, k = q % CH;
            const int64_t n = ni * C::BN + c;
            if (n < g.N && mi * C::BM + k * 8 < g.dz_ld) *(u32x4*)(dz + n * g.dz_ld + k * 8) = *(const u32x4*)(lds + (c * CH + (k ^ (c & (CH - 1)))) * 16);
        }
    } else {
#pragma unroll
        for (int j = 0; j < C::TN; ++j)
#pragma unroll
            for (int i = 0; i < C::TM; ++i) {
                const int64_t v = mi * C::BM + r0 + 16 * i, n = ni * C::BN + c0 + 16 * j;
                if (n < g.N && v < g.dz_ld) *(f32x4*)((float*)g.dz + n * g.dz_ld + v) = acc[i][j];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n < g.dzt_ld && v + e < g.w.rows) ((float*)g.dzt)[(v + e) * g.dzt_ld + n] = acc[i][j][e];
            }
    }
}

struct ProductArgs {
    Mat a, b;
    int64_t kbytes, kslice;                 // bytes of k: slice z takes z * kslice .. (kslice a multiple of 128)
    int64_t M, N;
    void* out; int64_t ld;                  // [n][m]
    int slices;
    float* sums; int add;                   // fp32 sums [slice][n][m] instead; add: onto what is there
    const float* rest; float scale;
    const float* row_on;                    // out: rows n with row_on[n] = 0 are zero
};

// C[m][n] -> out[n][m]: a lane holds four consecutive m of one n
template <typename T, class C, bool SUMS, bool KA, bool KB> NK_D void product(const ProductArgs& g, char* lds) {
    int64_t mi, ni;
    tile_of(blockIdx.x, (g.M + C::BM - 1) / C::BM, (g.N + C::BN - 1) / C::BN, &mi, &ni);
    const int64_t at = blockIdx.y * g.kslice, left = g.kbytes - at;
    Mat a = g.a, b = g.b;
    const int64_t row = at / (int64_t)sizeof(T);
    if (KA) { a.p += row * a.stride; a.rows -= row; } else a.p += at;
    if (KB) { b.p += row * b.stride; b.rows -= row; } else b.p += at;
    f32x4 acc[C::TM][C::TN];
    tile_product<T, C, KA, KB>(a, b, mi * C::BM, ni * C::BN, left < 0 ? 0 : left < g.kslice ? left : g.kslice, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / C::WGN, wn = wave % C::WGN;
    const float f = SUMS ? 1.0f : *g.rest * g.scale;
    const bool vec = SUMS ? (g.M & 3) == 0 : (g.ld & 3) == 0 && ((uintptr_t)g.out & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int j = 0; j < C::TN; ++j) {
        const int64_t n = ni * C::BN + wn * C::TN * 16 + j * 16 + (lane & 15);
        if (n >= g.N) continue;
        const bool off = !SUMS && g.row_on && g.row_on[n] == 0.0f;
#pragma unroll
        for (int i = 0; i < C::TM; ++i) {
            const int64_t m = mi * C::BM + wm * C::TM * 16 + i * 16 + 4 * (lane >> 4);
            if (m >= g.M) continue;
            if (SUMS) {
                float* s = g.sums + (blockIdx.y * g.N + n) * g.M + m;
                if (vec) {
                    f32x4 o = acc[i][j];
                    if (g.add) o += *(f32x4*)s;
                    *(f32x4*)s = o;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (m + e < g.M) s[e] = acc[i][j][e] + (g.add ? s[e] : 0.0f);
                }
            } else {
                T* o = (T*)g.out + n * g.ld + m;
                if (off) acc[i][j] = f32x4{0, 0, 0, 0};
                if (vec && m + 4 <= g.M) {
                    typedef __attribute__((ext_vector_type(4))) T vt;
                    vt w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = (T)(acc[i][j][e] * f);
                    *(vt*)o = w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (m + e < g.M) o[e] = (T)(acc[i][j][e] * f);
                }
            }
        }
    }
}

template <typename T, class C, bool SUMS, bool KA, bool KB>
__global__ __launch_bounds__(C::THREADS) void k_xent_product(const ProductArgs g) {
    __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
    product<T, C, SUMS, KA, KB>(g, lds);
}
// d_weight (z = 0) and d_hidden (z = 1) of a small call in one launch: each alone leaves most of the chip idle, and
// the host's time for launches is what such a call costs.  With k_xent_prepare and the finish of both in one, the backward
// pass of 1024 x 256 x 1000 in fp32 takes four launches instead of eight: 35 us instead of 47, 35 of host instead of 44.
struct PairArgs { ProductArgs p[2]; };
template <typename T, class C, bool SUMS>
__global__ __launch_bounds__(C::THREADS) void k_xent_pair(const PairArgs g) {
    __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
    const ProductArgs& p = g.p[blockIdx.z];
    if (blockIdx.x >= ((p.M + C::BM - 1) / C::BM) * ((p.N + C::BN - 1) / C::BN) || blockIdx.y >= p.slices) return;
    constexpr bool K = !BOTH_ORDERS<T>;
    if (blockIdx.z == 0) product<T, C, SUMS, K, K>(p, lds); else product<T, C, SUMS, K, false>(p, lds);
}

// A grid over many elements: the launch holds fewer than 2^32 threads along x.
inline dim3 flat_grid(int64_t blocks) {
    const int64_t x = blocks < (1 << 20) ? blocks : 1 << 20;
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
NK_D int64_t flat_block() { return blockIdx.x + (int64_t)blockIdx.y * gridDim.x; }

// out [N][D] from its fp32 sums, the slices in one order.  c: NULL, or rows with c = 0 (tokens that do not count) are
// zero.  VEC elements a thread.
struct FinishArgs { const float* sums; int slices, vec; int64_t N, D; const float* c; const float* rest; float scale; void* out; int64_t blocks; };
template <typename T, int VEC> NK_D void finish_block(const FinishArgs& g, int64_t block) {
    const int64_t i = (block * 256 + threadIdx.x) * VEC;
    if (i >= g.N * g.D) return;
    typedef __attribute__((ext_vector_type(VEC))) float fvec;
    typedef __attribute__((ext_vector_type(VEC))) T tvec;
    fvec s = *(const fvec*)(g.sums + i);
#pragma unroll 8
    for (int k = 1; k < g.slices; ++k) s += *(const fvec*)(g.sums + (int64_t)k * g.N * g.D + i);
    const float f = *g.rest * g.scale;
    const bool on = !g.c || g.c[i / g.D] != 0.0f;
    tvec w;
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = (T)(on ? s[e] * f : 0.0f);
    *(tvec*)((T*)g.out + i) = w;
}
template <typename T> __global__ __launch_bounds__(256) void k_xent_finish(const FinishArgs a, const FinishArgs b) {      // b: what is behind a's workgroups
    const int64_t block = flat_block();
    const FinishArgs& g = block < a.blocks ? a : b;
    const int64_t at = block < a.blocks ? block : block - a.blocks;
    if (at >= g.blocks) return;
    if (g.vec) finish_block<T, 4>(g, at); else finish_block<T, 1>(g, at);
}

// A copy [rows][cols] into rows of dst_ld (PAD: rows whose start or length the wide loads cannot take), or transposed into
// [cols][dst_ld]; zeros behind.  target: NULL, or rows whose target is `ignore` become zeros (their values may be anything).
struct CopyArgs { const void* src; int64_t ld, rows, cols; const int64_t* target; int64_t ignore; void* dst; int64_t dst_ld, blocks; int vec, across; };     // vec: source rows start on 16 bytes

// 16 bytes a thread
template <typename T> NK_D void pad_block(const CopyArgs& g, int64_t block) {
    constexpr int E = 16 / sizeof(T);
    typedef __attribute__((ext_vector_type(E))) T vec;
    const int64_t i = (block * 256 + threadIdx.x) * E;
    if (i >= g.rows * g.dst_ld) return;
    const int64_t r = i / g.dst_ld, c = i - r * g.dst_ld;           // dst_ld is a multiple of E
    const T* src = (const T*)g.src + r * g.ld + c;
    vec v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (T)0.0f;
    if (!(g.target && g.target[r] == g.ignore)) {
        if (g.vec && c + E <= g.cols) v = *(const vec*)src;
        else {
#pragma unroll
            for (int e = 0; e < E; ++e) if (c + e < g.cols) v[e] = src[e];
        }
    }
    *(vec*)((T*)g.dst + i) = v;
}

// 64 x 64; `across` blocks cover dst_ld
template <typename T> NK_D void transpose_block(const CopyArgs& g, int64_t block) {
    constexpr int E = 16 / sizeof(T), CH = 64 / E, LD = 64 + 4 / sizeof(T);     // elements per 16 bytes, such pieces per row
    typedef __attribute__((ext_vector_type(E))) T vec;
    __shared__ T tile[64 * LD];
    const int64_t r0 = (block % g.across) * 64, c0 = (block / g.across) * 64;
#pragma unroll
    for (int q = threadIdx.x; q < 64 * CH; q += 256) {
        const int k = q / CH, x = (q % CH) * E;
        const int64_t r = r0 + k, c = c0 + x;
        const T* src = (const T*)g.src + r * g.ld + c;
        vec v;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = (T)0.0f;
        if (r < g.rows && !(g.target && g.target[r] == g.ignore)) {
            if (g.vec && c + E <= g.cols) v = *(const vec*)src;
            else {
#pragma unroll
                for (int e = 0; e < E; ++e) if (c + e < g.cols) v[e] = src[e];
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) tile[k * LD + x + e] = v[e];
    }
    __syncthreads();
#pragma unroll
    for (int q = threadIdx.x; q < 64 * CH; q += 256) {
        const int x = q / CH, k = (q % CH) * E;         // column of the source, first row of the piece
        const int64_t c = c0 + x, r = r0 + k;
        if (c < g.cols && r < g.dst_ld) {               // dst_ld is a multiple of E
            vec v;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = tile[(k + e) * LD + x];
            *(vec*)((T*)g.dst + c * g.dst_ld + r) = v;
        }
    }
}
template <typename T> __global__ __launch_bounds__(256) void k_xent_pad(const CopyArgs g) { pad_block<T>(g, flat_block()); }
template <typename T> __global__ __launch_bounds__(256) void k_xent_transpose(const CopyArgs g) {
    const int64_t block = flat_block();
    if (block < g.blocks) transpose_block<T>(g, block);
}

// What the backward pass of a few tokens starts with, in one launch: the factors (workgroup 0) and the copies that the type
// needs (fp32: both transposed; 16 bits: hidden).
template <typename T> __global__ __launch_bounds__(256) void k_xent_prepare(const FactorArgs f, const CopyArgs a, const CopyArgs b) {
    const int64_t block = (int64_t)blockIdx.x - 1;
    if (block < 0) factors<256>(f, 0, 1);
    else if constexpr (BOTH_ORDERS<T>) { if (block < a.blocks) transpose_block<T>(a, block); else transpose_block<T>(b, block - a.blocks); }
    else if (block < a.blocks) pad_block<T>(a, block);
}

// ---- host -------------------------------------------------------------------------------------
typedef Cfg<256, 256, 2, 4, 2> Large;
typedef Cfg<128, 128, 2, 2, 2> Middle;
typedef Cfg<64, 64, 2, 2, 4> Small;
typedef Cfg<128, 32, 4, 1, 3> Few;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t up(int64_t a, int64_t b) { return cdiv(a, b) * b; }
inline int elem(int dt) { return dt == NK_F32 ? 4 : 2; }

template <auto K, typename... ARGS>
int start(dim3 grid, int threads, hipStream_t st, const char* name, const ARGS&... args) {
    hipLaunchKernelGGL(K, grid, dim3(threads), 0, st, args...);
    NK_CHECK_LAUNCH(name);
    return NK_OK;
}
template <auto K, typename... ARGS>
int start(int64_t blocks, int threads, hipStream_t st, const char* name, const ARGS&... args) {
    if (blocks * threads > 0xFFFFFFFFll) NK_FAIL(NK_ERR_UNSUPPORTED, "%s: too many tiles", name);
    return start<K>(dim3((unsigned)blocks), threads, st, name, args...);
}

// Which tile for an M x N product cut into `slices` stretches of k: the largest that still fills the 256 CUs.
enum { LARGE = NK_TILE_256x256, MIDDLE = NK_TILE_128x128, FEW = NK_TILE_128x32, SMALL = NK_TILE_64x64 };
int tile_kind(int64_t M, int64_t N, int64_t slices = 1) {
    if (N <= 32) return FEW;
    if (cdiv(M, 256) * cdiv(N, 256) * slices >= 224) return LARGE;
    return cdiv(M, 128) * cdiv(N, 128) * slices >= 200 ? MIDDLE : SMALL;
}
int kind_bm(int kind) { return kind == LARGE ? 256 : kind == SMALL ? 64 : 128; }

// Into how many stretches the k of an M x N product is cut where it has too few tiles to fill the chip: large tiles if
// the stretches stay long, otherwise small ones of eight steps at least.  64 at most: their fp32 sums are read
// once more.  d_weight of 196 608 tokens x 64 with 16 labels in bf16: 667 us whole, 21 us cut into 64; 65 536 x 256
// with 150 labels in fp32: 1 165 and 83 us.
int64_t cut_of(int64_t M, int64_t N, int64_t k, int64_t step) {
    const int64_t large = cdiv(M, 256) * cdiv(N, 256), tiles = cdiv(M, N <= 32 ? 128 : 64) * cdiv(N, N <= 32 ? 32 : 64);
    int64_t cut = 1;
    if (N > 32 && large < 224 && k / cdiv(256, large) >= 2048) cut = cdiv(256, large);
    else if (large < 224 && tiles < 256) cut = cdiv(512, tiles);
    const int64_t most = k / (8 * step);
    if (cut > most) cut = most;
    if (cut > 64) cut = 64;
    return cut < 1 ? 1 : cut;
}

struct Plan {
    int64_t Dp, Np, piece;                  // padded k of the logits' product; tokens padded to a step; vocabulary rows per piece
    bool pad_h, pad_w, copy_h;
    int kind, slices;
    int64_t parts, zt, losses, h, w, c, rest, tally, wt, ht, dz, dzt, sums, wsums, total;
};

int plan_of(const nk_xent_opts* o, const void* hidden, const void* weight, int backward, Plan* p, const char* who) {
    if (!o) NK_FAIL(NK_ERR_ARG, "%s: null options", who);
    if (o->N < 0 || o->D < 1 || o->V < 1) NK_FAIL(NK_ERR_ARG, "%s: N=%lld D=%lld V=%lld", who, (long long)o->N, (long long)o->D, (long long)o->V);
    if (o->dtype < NK_F32 || o->dtype > NK_F16) NK_FAIL(NK_ERR_ARG, "%s: unknown dtype %d", who, o->dtype);
    if (o->reduction < NK_REDUCE_NONE || o->reduction > NK_REDUCE_SUM) NK_FAIL(NK_ERR_ARG, "%s: unknown reduction %d", who, o->reduction);
    if (o->hidden_stride < o->D || o->weight_stride < o->D) NK_FAIL(NK_ERR_ARG, "%s: row strides below D", who);
    if (o->piece < 0) NK_FAIL(NK_ERR_ARG, "%s: piece < 0", who);
    const int es = elem(o->dtype);
    // 256 rows of an operand are addressed with 31 bits
    if (o->D > (1 << 20) || o->hidden_stride * es > (1 << 22) || o->weight_stride * es > (1 << 22) || o->N > (1 << 24) || o->V > (1 << 26))
        NK_FAIL(NK_ERR_UNSUPPORTED, "%s: D up to 2^20, row strides up to 2^22 bytes, N up to 2^24, V up to 2^26", who);
    const int64_t step = 128 / es;          // elements of k per step
    p->Dp = up(o->D, step);
    auto aligned = [&](const void* q, int64_t stride) { return ((uintptr_t)q & 15) == 0 && (stride * es) % 16 == 0 && (o->D * es) % 16 == 0; };
    p->pad_h = !aligned(hidden, o->hidden_stride); p->pad_w = !aligned(weight, o->weight_stride);
    p->Np = up(o->N, step);
    const int64_t asked = o->piece < o->V ? up(o->piece, 256) : up(o->V, 256);       // 0: not asked for
    const bool both = o->dtype == NK_F32;               // dz in both orders, transposed copies of weight and hidden
    // bytes of scratch that a row of the piece takes: its dz, and its copies
    const int64_t row = ((backward ? p->Np * (both ? 2 : 1) + (both ? o->D : 0) : 0) + (p->pad_w ? p->Dp : 0)) * es;
    int64_t piece = up(((int64_t)XENT_PIECE_MB << 20) / (row > 0 ? row : 1), 256);
    if (piece < 2048) piece = 2048;
    // pieces of one length, up to an eighth longer rather than one more: a training pass of 16384 x 1023 x 32003 in bf16 takes 4.46 ms in
    // four, 4.73 ms with a fifth of 259 rows behind them
    piece = up(cdiv(o->V, cdiv(o->V, piece + piece / 8)), 256);
    if (!backward) piece = !p->pad_w ? up(o->V, 256) : piece < 16384 ? piece : 16384;
    if (asked && (backward || p->pad_w)) piece = asked;
    if (piece > (1 << 22) / es) piece = (1 << 22) / es;         // a row of dz: up to 2^22 bytes, as of the other operands
    if (piece > o->V) piece = up(o->V, step);           // the only one
    if (backward && both && o->N > (1 << 20)) NK_FAIL(NK_ERR_UNSUPPORTED, "%s: fp32 gradients of up to 2^20 tokens a call", who);
    p->piece = piece;
    int64_t off = 0;
    auto take = [&](int64_t bytes) { const int64_t at = off; off = up(off + bytes, 1024); return at; };
    p->copy_h = p->pad_h || (backward && !both);        // without the values of tokens that do not count
    p->h = take(p->copy_h ? o->N * p->Dp * es : 0);
    p->w = take(p->pad_w ? piece * p->Dp * es : 0);
    p->kind = tile_kind(piece < o->V ? piece : o->V, o->N);
    p->slices = 1;
    if (!backward) {
        p->parts = take(cdiv(o->V, piece) * cdiv(piece, kind_bm(p->kind)) * o->N * 8);
        p->zt = take(o->N * 4);
        p->losses = take(cdiv(o->N, o->N <= 1024 ? 1 : 16) * sizeof(double2));
    } else {
        p->c = take(o->N * 4);
        p->rest = take(4);
        p->tally = take(cdiv(o->N, TALLY_TOKENS) * sizeof(Tally));
        p->wt = take(both ? o->D * piece * es : 0);
        p->ht = take(both ? o->D * p->Np * es : 0);
        p->dz = take(o->N * piece * es);
        p->dzt = take(both ? piece * p->Np * es : 0);
        p->slices = o->N > 0 ? (int)cut_of(o->D, o->N, piece, step) : 1;
        p->sums = take(p->slices == 1 && piece >= o->V ? 0 : (int64_t)p->slices * o->N * o->D * 4);
        // d_weight of a whole piece, and of the last one
        int64_t most = 0;
        for (const int64_t rows : {piece < o->V ? piece : o->V, (o->V - 1) % piece + 1}) {
            const int64_t cut = cut_of(o->D, rows, p->Np, step);
            if (cut > 1 && cut * rows > most) most = cut * rows;
        }
        p->wsums = take(most * o->D * 4);
    }
    p->total = off;
    return NK_OK;
}

template <typename T, class C> int lse_start(const LseArgs& g, hipStream_t st) {
    const int64_t tiles = cdiv(g.w.rows, C::BM) * cdiv(g.N, C::BN), fit = 256 * (163840 / (C::LDS + C::WGM * C::BN * 8));     // resident workgroups
    return start<k_xent_lse<T, C>>(tiles < fit ? tiles : fit, C::THREADS, st, "k_xent_lse", g);
}
template <typename T, class C> int dz_start(const DzArgs& g, hipStream_t st) {
    return start<k_xent_dz<T, C>>(cdiv(g.w.rows, C::BM) * cdiv(BOTH_ORDERS<T> ? g.dzt_ld : g.N, C::BN), C::THREADS, st, "k_xent_dz", g);
}
template <typename T, class C, bool SUMS, bool KA, bool KB> int product_start(const ProductArgs& g, int slices, hipStream_t st) {
    const int64_t tiles = cdiv(g.M, C::BM) * cdiv(g.N, C::BN);
    if (tiles * C::THREADS > 0xFFFFFFFFll) NK_FAIL(NK_ERR_UNSUPPORTED, "k_xent_product: too many tiles");
    return start<k_xent_product<T, C, SUMS, KA, KB>>(dim3((unsigned)tiles, (unsigned)slices), C::THREADS, st, "k_xent_product", g);
}
template <typename T> int lse_launch(int kind, const LseArgs& g, hipStream_t st) {
    return kind == LARGE ? lse_start<T, Large>(g, st) : kind == MIDDLE ? lse_start<T, Middle>(g, st) : kind == FEW ? lse_start<T, Few>(g, st)
                                                                                                        : lse_start<T, Small>(g, st);
}
template <typename T> int dz_launch(int kind, const DzArgs& g, hipStream_t st) {
    return kind == LARGE ? dz_start<T, Large>(g, st) : kind == MIDDLE ? dz_start<T, Middle>(g, st) : kind == FEW ? dz_start<T, Few>(g, st)
                                                                                                      : dz_start<T, Small>(g, st);
}
template <typename T, bool SUMS, bool KA, bool KB> int product_launch(const ProductArgs& g, int slices, hipStream_t st) {
    const int kind = tile_kind(g.M, g.N, slices);
    return kind == LARGE ? product_start<T, Large, SUMS, KA, KB>(g, slices, st) : kind == MIDDLE ? product_start<T, Middle, SUMS, KA, KB>(g, slices, st)
         : kind == FEW ? product_start<T, Few, SUMS, KA, KB>(g, slices, st) : product_start<T, Small, SUMS, KA, KB>(g, slices, st);
}

template <typename T, bool SUMS> int pair_start(const PairArgs& g, hipStream_t st) {
    auto tiles = [](const ProductArgs& p) { return cdiv(p.M, Small::BM) * cdiv(p.N, Small::BN); };        // some hundreds: SMALL
    const int64_t x = tiles(g.p[0]) > tiles(g.p[1]) ? tiles(g.p[0]) : tiles(g.p[1]);
    const int y = g.p[0].slices > g.p[1].slices ? g.p[0].slices : g.p[1].slices;
    return start<k_xent_pair<T, Small, SUMS>>(dim3((unsigned)x, (unsigned)y, 2), Small::THREADS, st, "k_xent_pair", g);
}

template <typename T> CopyArgs pad_of(const void* src, int64_t ld, int64_t rows, int64_t cols, const int64_t* target, int64_t ignore, void* dst, int64_t dst_ld) {
    return CopyArgs{src, ld, rows, cols, target, ignore, dst, dst_ld, cdiv(rows * dst_ld, 256 * (16 / (int64_t)sizeof(T))), ((uintptr_t)src & 15) == 0 && ld * sizeof(T) % 16 == 0, 0};
}
template <typename T> CopyArgs transpose_of(const void* src, int64_t ld, int64_t rows, int64_t cols, const int64_t* target, int64_t ignore, void* dst, int64_t dst_ld) {
    const int64_t across = cdiv(dst_ld, 64);
    return CopyArgs{src, ld, rows, cols, target, ignore, dst, dst_ld, across * cdiv(cols, 64), ((uintptr_t)src & 15) == 0 && ld * sizeof(T) % 16 == 0, (int)across};
}
template <typename T> int pad(const CopyArgs& g, hipStream_t st) {
    hipLaunchKernelGGL(k_xent_pad<T>, flat_grid(g.blocks), dim3(256), 0, st, g);
    NK_CHECK_LAUNCH("k_xent_pad");
    return NK_OK;
}
template <typename T> int transpose(const CopyArgs& g, hipStream_t st) {
    hipLaunchKernelGGL(k_xent_transpose<T>, flat_grid(g.blocks), dim3(256), 0, st, g);
    NK_CHECK_LAUNCH("k_xent_transpose");
    return NK_OK;
}
template <typename T> FinishArgs finish_of(const float* sums, int slices, int64_t rows, int64_t D, const float* c, const float* rest, void* out) {
    const int vec = D % 4 == 0 && ((uintptr_t)out & (4 * sizeof(T) - 1)) == 0;
    return FinishArgs{sums, slices, vec, rows, D, c, rest, 1.0f / Op<T>::SCALE, out, cdiv(rows * D, vec ? 1024 : 256)};
}
template <typename T> int finish(const FinishArgs& a, const FinishArgs& b, hipStream_t st) {
    hipLaunchKernelGGL(k_xent_finish<T>, flat_grid(a.blocks + b.blocks), dim3(256), 0, st, a, b);
    NK_CHECK_LAUNCH("k_xent_finish");
    return NK_OK;
}

template <typename T>
int forward(const nk_xent_opts* o, const Plan& p, const void* hidden, const void* weight, const int64_t* target, float* loss, float* lse, float* reduced,
            char* ws, hipStream_t st) {
    const int es = sizeof(T);
    int rc;
    Mat h = {(const char*)hidden, o->N, o->hidden_stride * es, o->D * es};
    if (p.copy_h) {
        if ((rc = pad<T>(pad_of<T>(hidden, o->hidden_stride, o->N, o->D, nullptr, 0, ws + p.h, p.Dp), st)) < 0) return rc;
        h = Mat{ws + p.h, o->N, p.Dp * es, p.Dp * es};
    }
    int64_t tiles = 0;
    for (int64_t v0 = 0; v0 < o->V; v0 += p.piece) {
        const int64_t rows = o->V - v0 < p.piece ? o->V - v0 : p.piece;
        const char* src = (const char*)weight + v0 * o->weight_stride * es;
        Mat w = {src, rows, o->weight_stride * es, o->D * es};
        if (p.pad_w) {
            if ((rc = pad<T>(pad_of<T>(src, o->weight_stride, rows, o->D, nullptr, 0, ws + p.w, p.Dp), st)) < 0) return rc;
            w = Mat{ws + p.w, rows, p.Dp * es, p.Dp * es};
        }
        const LseArgs g = {w, h, o->D * es, v0, o->N, target, (float2*)(ws + p.parts), tiles, (float*)(ws + p.zt)};
        if ((rc = lse_launch<T>(p.kind, g, st)) < 0) return rc;
        tiles += cdiv(rows, kind_bm(p.kind));
    }
    if (o->reduction != NK_REDUCE_NONE && o->N <= 1024 && tiles <= 32) {
        hipLaunchKernelGGL(k_xent_join_reduce, dim3(1), dim3(1024), 0, st, (const float2*)(ws + p.parts), (int)tiles, (int)o->N, o->V, target,
                           o->ignore_index, (const float*)(ws + p.zt), (int)(o->reduction == NK_REDUCE_MEAN), lse, loss, reduced);
        NK_CHECK_LAUNCH("k_xent_join_reduce");
        return NK_OK;
    }
    double2* losses = o->reduction != NK_REDUCE_NONE ? (double2*)(ws + p.losses) : nullptr;
    // few tokens: all threads of a workgroup on one of them
    if (o->N <= 1024)
        hipLaunchKernelGGL(k_xent_join<1>, dim3((unsigned)o->N), dim3(256), 0, st, (const float2*)(ws + p.parts), tiles, o->N, o->V, target,
                           o->ignore_index, (const float*)(ws + p.zt), lse, loss, losses);
    else
        hipLaunchKernelGGL(k_xent_join<16>, dim3((unsigned)cdiv(o->N, 16)), dim3(256), 0, st, (const float2*)(ws + p.parts), tiles, o->N, o->V,
                           target, o->ignore_index, (const float*)(ws + p.zt), lse, loss, losses);
    NK_CHECK_LAUNCH("k_xent_join");
    if (o->reduction != NK_REDUCE_NONE) {
        hipLaunchKernelGGL(k_xent_reduce, dim3(1), dim3(1024), 0, st, losses, cdiv(o->N, o->N <= 1024 ? 1 : 16), o->reduction == NK_REDUCE_MEAN, reduced);
        NK_CHECK_LAUNCH("k_xent_reduce");
    }
    return NK_OK;
}

template <typename T>
int backward(const nk_xent_opts* o, const Plan& p, const void* hidden, const void* weight, const int64_t* target, const float* lse, const float* d_loss,
             void* d_hidden, void* d_weight, char* ws, hipStream_t st) {
    const int es = sizeof(T);
    const float unscale = 1.0f / Op<T>::SCALE;
    float* c = (float*)(ws + p.c);
    float* rest = (float*)(ws + p.rest);
    int rc;
    constexpr bool BOTH = BOTH_ORDERS<T>;
    Mat h = {(const char*)hidden, o->N, o->hidden_stride * es, o->D * es};
    const bool one = p.piece >= o->V, copy_h = p.copy_h && (p.pad_h || d_weight);
    FactorArgs f = {target, o->N, o->V, o->ignore_index, o->reduction, (int)cdiv(o->N, TALLY_TOKENS), d_loss, nullptr, c, rest};
    const CopyArgs clean = pad_of<T>(hidden, o->hidden_stride, o->N, o->D, target, o->ignore_index, ws + p.h, p.Dp);
    const CopyArgs ht = transpose_of<T>(hidden, o->hidden_stride, o->N, o->D, target, o->ignore_index, ws + p.ht, p.Np);
    const bool few = o->N <= 2048 && (BOTH ? one && d_weight && d_hidden : copy_h);        // factors and copies in one launch
    if (few) {
        CopyArgs wt = {};
        if (BOTH) wt = transpose_of<T>(weight, o->weight_stride, o->V, o->D, nullptr, 0, ws + p.wt, up(o->V, 128 / es));
        const CopyArgs& a = BOTH ? ht : clean;
        if ((rc = start<k_xent_prepare<T>>(1 + a.blocks + wt.blocks, 256, st, "k_xent_prepare", f, a, wt)) < 0) return rc;
    } else {
        if (f.n_parts > 2) {                // up to two: less than another launch
            f.parts = (const Tally*)(ws + p.tally);
            hipLaunchKernelGGL(k_xent_tally, dim3(f.n_parts), dim3(1024), 0, st, target, o->N, o->ignore_index, o->reduction, d_loss, (Tally*)(ws + p.tally));
            NK_CHECK_LAUNCH("k_xent_tally");
        }
        hipLaunchKernelGGL(k_xent_factors, dim3(f.parts ? f.n_parts : 1), dim3(1024), 0, st, f);
        NK_CHECK_LAUNCH("k_xent_factors");
    }
    if (copy_h) {
        if ((!few || BOTH) && (rc = pad<T>(clean, st)) < 0) return rc;
        h = Mat{ws + p.h, o->N, p.Dp * es, p.Dp * es};
    }
    if constexpr (BOTH) { if (d_weight && !few && (rc = transpose<T>(ht, st)) < 0) return rc; }
    const int64_t slice = up(cdiv(p.piece, p.slices), 128 / es) * es;
    const bool direct = p.slices == 1 && one;      // d_hidden in one product: no sums to keep
    for (int64_t v0 = 0; v0 < o->V; v0 += p.piece) {
        const int64_t rows = o->V - v0 < p.piece ? o->V - v0 : p.piece;
        const char* src = (const char*)weight + v0 * o->weight_stride * es;
        Mat w = {src, rows, o->weight_stride * es, o->D * es};
        if (p.pad_w) {
            if ((rc = pad<T>(pad_of<T>(src, o->weight_stride, rows, o->D, nullptr, 0, ws + p.w, p.Dp), st)) < 0) return rc;
            w = Mat{ws + p.w, rows, p.Dp * es, p.Dp * es};
        }
        const int64_t kv = up(rows, 128 / es);          // columns of dz that the product takes: zeros behind `rows`
        const DzArgs g = {w, h, o->D * es, v0, o->N, target, lse, c, ws + p.dz, kv, ws + p.dzt, p.Np};
        if ((rc = dz_launch<T>(tile_kind(rows, o->N), g, st)) < 0) return rc;
        ProductArgs qw = {}, qh = {};
        char* out_w = (char*)d_weight + v0 * o->D * es;
        const int cut = d_weight ? (int)cut_of(o->D, rows, p.Np, 128 / es) : 1;
        if (d_weight) {
            if (BOTH) { qw.a = Mat{ws + p.ht, o->D, p.Np * es, 0}; qw.b = Mat{ws + p.dzt, rows, p.Np * es, 0}; }
            else { qw.a = h; qw.b = Mat{ws + p.dz, o->N, kv * es, kv * es}; }
            qw.kbytes = qw.kslice = p.Np * es; qw.M = o->D; qw.N = rows; qw.slices = cut;
            if (cut == 1) { qw.out = out_w; qw.ld = o->D; qw.rest = rest; qw.scale = unscale; }
            else { qw.kslice = up(cdiv(p.Np, cut), 128 / es) * es; qw.sums = (float*)(ws + p.wsums); }
        }
        if (d_hidden) {
            if constexpr (BOTH) {
                if (!few && (rc = transpose<T>(transpose_of<T>(src, o->weight_stride, rows, o->D, nullptr, 0, ws + p.wt, kv), st)) < 0) return rc;
                qh.a = Mat{ws + p.wt, o->D, kv * es, 0};
            } else {
                qh.a = w;
            }
            qh.b = Mat{ws + p.dz, o->N, kv * es, kv * es};
            qh.kbytes = kv * es; qh.kslice = slice; qh.M = o->D; qh.N = o->N; qh.slices = p.slices;
            if (direct) { qh.out = d_hidden; qh.ld = o->D; qh.rest = rest; qh.scale = unscale; qh.row_on = c; }
            else { qh.sums = (float*)(ws + p.sums); qh.add = v0 > 0; }
        }
        if (d_weight && d_hidden && one && direct == (cut == 1) && tile_kind(o->D, rows, cut) == SMALL && tile_kind(o->D, o->N, p.slices) == SMALL) {
            const PairArgs pair = {{qw, qh}};
            if (direct) return pair_start<T, false>(pair, st);
            if ((rc = pair_start<T, true>(pair, st)) < 0) return rc;
            return finish<T>(finish_of<T>(qw.sums, cut, rows, o->D, nullptr, rest, out_w), finish_of<T>(qh.sums, p.slices, o->N, o->D, c, rest, d_hidden), st);
        }
        if (d_weight) {
            if (cut == 1) {
                if ((rc = product_launch<T, false, !BOTH, !BOTH>(qw, 1, st)) < 0) return rc;
            } else {
                if ((rc = product_launch<T, true, !BOTH, !BOTH>(qw, cut, st)) < 0) return rc;
                if ((rc = finish<T>(finish_of<T>(qw.sums, cut, rows, o->D, nullptr, rest, out_w), FinishArgs{}, st)) < 0) return rc;
            }
        }
        if (d_hidden) {
            if (direct) { if ((rc = product_launch<T, false, !BOTH, false>(qh, 1, st)) < 0) return rc; }
            else if ((rc = product_launch<T, true, !BOTH, false>(qh, p.slices, st)) < 0) return rc;
        }
    }
    if (d_hidden && !direct) return finish<T>(finish_of<T>((const float*)(ws + p.sums), p.slices, o->N, o->D, c, rest, d_hidden), FinishArgs{}, st);
    return NK_OK;
}

int check_ws(const Plan& p, const void* ws, int64_t bytes, const char* who) {
    if (bytes < p.total || (p.total > 0 && (!ws || ((uintptr_t)ws & 255))))
        NK_FAIL(NK_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed (256-byte aligned)", who, (long long)bytes, (long long)p.total);
    return NK_OK;
}

}  // namespace

extern "C" int64_t nk_linear_xent_workspace_bytes(const nk_xent_opts* o, const void* hidden, const void* weight, int backward) {
    Plan p;
    const int rc = plan_of(o, hidden, weight, backward, &p, "nk_linear_xent_workspace_bytes");
    return rc < 0 ? rc : p.total;
}

extern "C" int64_t nk_linear_xent_cuts(const nk_xent_opts* o, const void* hidden, const void* weight, int64_t piece, int32_t* cuts) {
    Plan f, b;
    int rc = plan_of(o, hidden, weight, 0, &f, "nk_linear_xent_cuts");
    if (rc < 0 || (rc = plan_of(o, hidden, weight, 1, &b, "nk_linear_xent_cuts")) < 0) return rc;
    const int64_t pieces = cdiv(o->V, b.piece);
    if (!cuts || o->N < 1 || piece < 0 || piece >= pieces) NK_FAIL(NK_ERR_ARG, "nk_linear_xent_cuts: no tokens, or no piece %lld of %lld", (long long)piece, (long long)pieces);
    const int64_t v0 = piece * b.piece, rows = o->V - v0 < b.piece ? o->V - v0 : b.piece;
    const int cut = (int)cut_of(o->D, rows, b.Np, 128 / elem(o->dtype));
    cuts[0] = f.kind;
    cuts[1] = tile_kind(rows, o->N);
    cuts[2] = tile_kind(o->D, rows, cut) + 16 * (cut > 1 ? cut : 0);
    cuts[3] = tile_kind(o->D, o->N, b.slices) + 16 * (b.slices > 1 || pieces > 1 ? b.slices : 0);
    return pieces;
}

extern "C" int nk_linear_xent_fwd(const nk_xent_opts* o, const void* hidden, const void* weight, const int64_t* target, float* loss, float* lse,
                                  float* reduced, void* workspace, int64_t workspace_bytes, void* stream) {
    Plan p;
    int rc = plan_of(o, hidden, weight, 0, &p, "nk_linear_xent_fwd");
    if (rc < 0) return rc;
    if (o->reduction != NK_REDUCE_NONE && !reduced) NK_FAIL(NK_ERR_ARG, "nk_linear_xent_fwd: the reduction needs `reduced`");
    if (o->N > 0 && (!hidden || !weight || !target || !loss || !lse)) NK_FAIL(NK_ERR_ARG, "nk_linear_xent_fwd: null pointer");
    if ((rc = check_ws(p, workspace, workspace_bytes, "nk_linear_xent_fwd")) < 0) return rc;
    const hipStream_t st = nk_stream(stream);
    if (o->N == 0) {
        if (o->reduction != NK_REDUCE_NONE) {
            hipLaunchKernelGGL(k_xent_reduce, dim3(1), dim3(1024), 0, st, (const double2*)nullptr, (int64_t)0, 0, reduced);
            NK_CHECK_LAUNCH("k_xent_reduce");
        }
        return NK_OK;
    }
    char* ws = (char*)workspace;
    if (o->dtype == NK_BF16) return forward<__bf16>(o, p, hidden, weight, target, loss, lse, reduced, ws, st);
    if (o->dtype == NK_F16) return forward<_Float16>(o, p, hidden, weight, target, loss, lse, reduced, ws, st);
    return forward<float>(o, p, hidden, weight, target, loss, lse, reduced, ws, st);
}

extern "C" int nk_linear_xent_bwd(const nk_xent_opts* o, const void* hidden, const void* weight, const int64_t* target, const float* lse,
                                  const float* d_loss, void* d_hidden, void* d_weight, void* workspace, int64_t workspace_bytes, void* stream) {
    Plan p;
    int rc = plan_of(o, hidden, weight, 1, &p, "nk_linear_xent_bwd");
    if (rc < 0) return rc;
    if (o->N < 1) NK_FAIL(NK_ERR_ARG, "nk_linear_xent_bwd: no tokens");
    if (!hidden || !weight || !target || !lse || !d_loss || (!d_hidden && !d_weight)) NK_FAIL(NK_ERR_ARG, "nk_linear_xent_bwd: null pointer");
    if ((rc = check_ws(p, workspace, workspace_bytes, "nk_linear_xent_bwd")) < 0) return rc;
    const hipStream_t st = nk_stream(stream);
    char* ws = (char*)workspace;
    if (o->dtype == NK_BF16) return backward<__bf16>(o, p, hidden, weight, target, lse, d_loss, d_hidden, d_weight, ws, st);
    if (o->dtype == NK_F16) return backward<_Float16>(o, p, hidden, weight, target, lse, d_loss, d_hidden, d_weight, ws, st);
    return backward<float>(o, p, hidden, weight, target, lse, d_loss, d_hidden, d_weight, ws, st);
}
