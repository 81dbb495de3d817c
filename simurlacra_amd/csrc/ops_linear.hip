// Layers of a population of networks: y[r] = f(W_g x[r] + b_g) for the rows r of group g, with ragged groups, and its
// gradients (psh_grouped_linear, psh_grouped_linear_grad of include/pysimhip.h).
//
// One tiled matrix product serves the three of them, D[i, j] = sum_c P[i, c] Q[j, c] per group:
//   forward  i = output unit,  j = row,          c = input unit     P = W_g          Q = x
//   dx       i = input unit,   j = row,          c = output unit    P = W_g^T        Q = dp
//   dW       i = output unit,  j = input unit,   c = row            P = dp^T         Q = x^T
// with dp = dy f'(y).  Rows are the SECOND index of the matrix instruction: its result then holds four consecutive
// units of one row per lane, which is what a row-major store wants.
//
// In LDS both operands lie as [index][128 bytes of c], whichever way they are laid out in memory; a lane's fragment is 16
// bytes along c, so 8 bf16 are one operand of v_mfma_f32_16x16x32_bf16, 4 floats those of four v_mfma_f32_16x16x4_f32 and 2
// doubles those of two v_mfma_f64_16x16x4_f64 (c is summed over, so which c meets in which instruction is free as long as
// P and Q agree).  The 16-byte units of an index are permuted, see unit_of.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "psh_linear_plan.h"
#include "psh_ops.h"

namespace {

PSH_OP int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// Part k of the product of two fragments.  The parts of one fragment pair all add to the same accumulator, so the parts are the outer
// loop: an instruction that waits for the one before it would leave the matrix pipe idle.
template <class T> struct Mfma;
template <> struct Mfma<bf16_t> {
    typedef v4f acc;
    static constexpr int PARTS = 1;
    static constexpr int row(int q, int r) { return 4 * q + r; }   // index i of accumulator register r in lane group q
    template <int> static PSH_OP void step(const v4u& p, const v4u& q, acc& d) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, p), __builtin_bit_cast(v8bf, q), d, 0, 0, 0);
    }
};
template <> struct Mfma<float> {
    typedef v4f acc;
    static constexpr int PARTS = 4;
    static constexpr int row(int q, int r) { return 4 * q + r; }
    template <int K> static PSH_OP void step(const v4u& p, const v4u& q, acc& d) {
        d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(p[K]), __uint_as_float(q[K]), d, 0, 0, 0);
    }
};
template <> struct Mfma<double> {
    typedef v4d acc;
    static constexpr int PARTS = 2;
    static constexpr int row(int q, int r) { return 4 * r + q; }
    template <int K> static PSH_OP void step(const v4u& p, const v4u& q, acc& d) {
        d = __builtin_amdgcn_mfma_f64_16x16x4f64(__hiloint2double((int)p[2 * K + 1], (int)p[2 * K]),
                                                 __hiloint2double((int)q[2 * K + 1], (int)q[2 * K]), d, 0, 0, 0);
    }
};

// an operand: element (index i, c) at p[i * ld + c], or at p[c * ld + i] if it is read transposed
template <class T> struct Operand {
    const T* p;
    long ld;
    int n, nc;      // valid indices and valid c
};

// 16 bytes at any element: the hardware takes unaligned global loads
template <class T> PSH_OP v4u load16(const T* p) {
    v4u v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// The 16-byte units of an index are permuted: 16 neighbouring indices, which a fragment read takes at a time, lie two to a row of 64 banks
// in 8 different units, and so do indices V apart, which the transposing writes take.
PSH_OP int unit_of(int i, int u) { return u ^ (((i >> 1) ^ (i >> 4)) & 7); }

// One thread's part of a tile of N indices x 8 units of 16 bytes: loaded into registers while the previous tile is being
// multiplied, stored to LDS afterwards.  Indices past the operand's end are read as whatever lies there within the operand (their results
// are not stored); c past its end are zeros.
template <class T, int N, int THREADS, bool TR> struct Stager {
    static constexpr int V = 16 / (int)sizeof(T), KC = 128 / (int)sizeof(T);
    static constexpr int WORK = TR ? (N / V) * 8 : N * 8;                 // V x V blocks, or units
    static constexpr int PER = (WORK + THREADS - 1) / THREADS;
    static constexpr int REGS = TR ? PER * V : PER;
    v4u r[REGS];
    const T* at[PER];   // line (block) of c = 0

    PSH_OP explicit Stager(const Operand<T>& o) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int id = (int)threadIdx.x + k * THREADS;
            if constexpr (!TR) at[k] = o.p + (long)min(id >> 3, o.n - 1) * o.ld + (id & 7) * V;
            else at[k] = o.p + (long)(id / (N / V) * V) * o.ld + min(id % (N / V) * V, (o.n - 1) / V * V);
        }
    }
    // whether the tile from c0 can be read in whole units.  A transposed operand's last unit may run over its line's end, by up to V - 1
    // elements: that many have to follow in the operand.
    static PSH_OP bool whole(const Operand<T>& o, int c0) {
        return c0 + KC <= o.nc && (!TR || o.n % V == 0 || (long)(o.nc - c0 - KC) * o.ld >= V - 1);
    }
    PSH_OP void fetch(const Operand<T>& o, int c0) {
        if (whole(o, c0)) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                if (WORK % THREADS != 0 && (int)threadIdx.x + k * THREADS >= WORK) break;
                if constexpr (!TR) {
                    r[k] = load16(at[k] + c0);
                } else {
                    const T* const q = at[k] + (long)c0 * o.ld;
#pragma unroll
                    for (int j = 0; j < V; ++j) r[k * V + j] = load16(q + j * o.ld);
                }
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int id = (int)threadIdx.x + k * THREADS;
            if constexpr (!TR) {
                r[k] = piece(o.p + (long)min(id >> 3, o.n - 1) * o.ld, c0 + (id & 7) * V, o.nc);
            } else {
                const int ib = id % (N / V), u = id / (N / V);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int c = c0 + u * V + j;
                    r[k * V + j] = c < o.nc && id < WORK ? piece(o.p + (long)c * o.ld, ib * V, o.n) : v4u{0, 0, 0, 0};
                }
            }
        }
    }
    // elements [first, first + V) of a line with `limit` valid ones
    static PSH_OP v4u piece(const T* line, int first, int limit) {
        T e[V];
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = first + k < limit ? line[first + k] : T(0);
        return __builtin_bit_cast(v4u, e);
    }
    PSH_OP void store(unsigned char* lds) const {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int id = (int)threadIdx.x + k * THREADS;
            if (WORK % THREADS != 0 && id >= WORK) break;
            if constexpr (!TR) {
                const int i = id >> 3, u = id & 7;
                *reinterpret_cast<v4u*>(lds + i * 128 + unit_of(i, u) * 16) = r[k];
            } else {
                const int ib = id % (N / V), u = id / (N / V);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    T e[V];
#pragma unroll
                    for (int m = 0; m < V; ++m) {
                        T line[V];
                        __builtin_memcpy(line, &r[k * V + m], 16);
                        e[m] = line[j];
                    }
                    const int i = ib * V + j;
                    *reinterpret_cast<v4u*>(lds + i * 128 + unit_of(i, u) * 16) = __builtin_bit_cast(v4u, e);
                }
            }
        }
    }
};

// This lane's number, counted anew: what is computed from it is not kept in registers for a whole loop, where 128 accumulators and 96
// registers of fragments leave room for little else.
PSH_OP int lane_now() {
    int lane;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(lane));
    return lane;
}
// A bf16 operand's tiles by loads that go to LDS directly: no registers, no transposing on the way in.  The tile lies as it is in memory, [index][64 c]
// or, for a transposed operand, [64 c][index], where ds_read_b64_tr_b16 does the transposing: 16 lanes, four to a row of 16 indices, read 4
// rows, and lane i gets column i.  The loads go to LDS in lane order, so the permutation that spreads the banks is applied
// to the addresses they read from: 16-byte units by the index as in Stager, or 32-byte chunks of a row by c, so that the 8
// rows that half a wave reads at a time are in different banks.
// Rows past the operand's end are read as its last one (their results are not stored); only whole tiles of c come this way.
template <int N, int THREADS, bool TR> struct Direct {
    static constexpr int KC = 32, BYTES = N * 2 * KC, WAVES = THREADS / 64, PER = BYTES / 1024 / WAVES;   // 1-KiB loads of a wave
    static constexpr int ROW = N * 2, STEP = WAVES * 1024 / ROW;                                          // transposed: bytes of a row, rows between a thread's loads
    static PSH_OP int swz_i(int i) { return (i >> 2) & 3; }
    static PSH_OP int swz_c(int c) { return ((c & 3) | ((c >> 1) & 4)) << 1; }
    // this wave's loads of the tile from c0 to the LDS address `lds`, one by one
    struct Loads {
        const bf16_t* line;
        long ld;
        unsigned lds;
        int i0, last, unit;
        PSH_OP Loads(const Operand<bf16_t>& o, int c0, unsigned to, int wave) : ld(o.ld), lds(to + wave * 1024) {
            const int lane = lane_now(), at = wave * 1024 + lane * 16, c = at / ROW;
            i0 = at >> 6;
            last = o.n - 1;
            unit = TR ? (at % ROW / 16) ^ swz_c(c) : (lane & 3) ^ swz_i(i0);
            line = TR ? o.p + (long)(c0 + c) * ld : o.p + c0;
        }
        PSH_OP void issue(int k) const {
            static_assert(STEP % 8 == 0, "the permutations of a thread's loads differ by constants");
            const bf16_t* g;
            if constexpr (!TR) {
                g = line + (long)min(i0 + k * 16 * WAVES, last) * ld + unit * 8;
            } else {
                g = line + (long)(k * STEP) * ld + min((unit ^ swz_c(k * STEP)) * 8, last - 7);
            }
            // (by hand, because the compiler would wait for a builtin's load before the next read of any part of LDS; the
            // waits are in front of the barriers)
            // One wait state has to lie between a write of m0 and a load to LDS.
            // (m0 is a reserved register, which the compiler warns of on a clobber list; it keeps nothing there across the statement, but it is
            // told of the write, so that it does not take a value of its own in front of the statement for the one behind it)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds + k * WAVES * 1024), "v"(g) : "memory", "m0");
#pragma clang diagnostic pop
        }
    };
    // the last, partial tile of c through registers, zero where there is none
    static PSH_OP void fetch_tail(const Operand<bf16_t>& o, int c0, unsigned char* lds, int wave) {
#pragma unroll 1
        for (int at = (wave * 64 + lane_now()) * 16; at < BYTES; at += THREADS * 16) {
            v4u v = {0, 0, 0, 0};
            if constexpr (!TR) {
                const int i = at >> 6;
                v = Stager<bf16_t, N, THREADS, false>::piece(o.p + (long)min(i, o.n - 1) * o.ld, c0 + ((at >> 4 & 3) ^ swz_i(i)) * 8, o.nc);
            } else {
                const int c = at / ROW, u = (at % ROW / 16) ^ swz_c(c);
                if (c0 + c < o.nc) v = load16(o.p + (long)(c0 + c) * o.ld + min(u * 8, o.n - 8));
            }
            *reinterpret_cast<v4u*>(lds + at) = v;
        }
    }
    // Fragments of blocks of 16 indices from i0 (a multiple of 16 times their number): 16 bytes along c for the index i0 + 16 m + (lane & 15),
    // c from s * 32 + (lane / 16) * 8
    struct Reads {
        unsigned char* lds;
        int at;
        PSH_OP Reads(unsigned char* tile, int i0) : lds(tile) {
            const int lane = lane_now(), l = lane & 15, g = lane >> 4, c = g * 8 + (l >> 2);
            at = TR ? c * ROW + ((i0 >> 4) * 32 ^ swz_c(c) * 16) + (l & 3) * 8 : (i0 + l) * 64 + (g ^ swz_i(l)) * 16;
        }
        PSH_OP v4u block(int m) const {
            if constexpr (!TR) return *reinterpret_cast<const v4u*>(lds + at + m * 1024);
            typedef short v4s __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) v4s* at_t;
            unsigned char* const q = lds + (at ^ (m * 32));
            const uint2 h0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)q));
            const uint2 h1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_t)(q + 4 * ROW)));
            return v4u{h0.x, h0.y, h1.x, h1.y};
        }
    };
};

template <class T, int BI, int BJ, int WI, int WJ> struct Tile {
    static constexpr int THREADS = 64 * WI * WJ, MI = BI / WI / 16, MJ = BJ / WJ / 16;
    typedef typename Mfma<T>::acc acc_t;
    acc_t acc[MI][MJ];
    // sums of P over c, in every column (the bias gradient), if asked for: a block of 16 indices i is summed by one of the WJ waves that have it
    static constexpr int OWN = MI / WJ > 0 ? MI / WJ : 1;
    acc_t ones[OWN];
    acc_t block[sizeof(T) == 4 ? OWN : 1];   // those of the last few steps, see fold()
    int wave_j;

    template <int K, bool SUMS> PSH_OP void part(const v4u (&fp)[MI], const v4u (&fq)[MJ], const v4u& unit) {
#pragma unroll
        for (int a = 0; a < MI; ++a) {
#pragma unroll
            for (int b = 0; b < MJ; ++b) Mfma<T>::template step<K>(fp[a], fq[b], acc[a][b]);
        }
        if constexpr (SUMS) sums<K>(fp, unit);
    }
    template <int K> PSH_OP void sums(const v4u (&fp)[MI], const v4u& unit) {
#pragma unroll
        for (int w = 0; w < WJ; ++w)
            if (w == wave_j)
#pragma unroll
                for (int k = 0; k < OWN; ++k) Mfma<T>::template step<K>(fp[w * OWN + k], unit, sizeof(T) == 4 ? block[sizeof(T) == 4 ? k : 0] : ones[k]);
    }

    template <bool SUMS> PSH_OP void clear(v4u& unit) {
#pragma unroll
        for (int a = 0; a < MI; ++a)
#pragma unroll
            for (int b = 0; b < MJ; ++b) acc[a][b] = acc_t{0, 0, 0, 0};
        if constexpr (SUMS) {
            static_assert(OWN * WJ == MI, "the waves share the blocks evenly");
            wave_j = wave_id() / WI;
#pragma unroll
            for (int k = 0; k < OWN; ++k) ones[k] = acc_t{0, 0, 0, 0};
            if constexpr (sizeof(T) == 4)
#pragma unroll
                for (int k = 0; k < OWN; ++k) block[k] = acc_t{0, 0, 0, 0};
            T e[16 / sizeof(T)];
#pragma unroll
            for (int k = 0; k < (int)(16 / sizeof(T)); ++k) e[k] = to_elem<T>(1);
            unit = __builtin_bit_cast(v4u, e);
        }
    }
    // A sum of n numbers one after the other in fp32 is off by about sqrt(n / 2) roundings of itself, one of blocks' sums by that of a block.  The sums of
    // products have library products of the same kind beside them; those of the rows themselves, which are usually summed in a tree,
    // are kept in blocks of 128 rows (2500 rows: 4.8e-7 in one go, 2.7e-7 in blocks).
    PSH_OP void fold() {
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            ones[k] += block[k];
            block[k] = acc_t{0, 0, 0, 0};
        }
    }
    template <bool SUMS> PSH_OP void parts(const v4u (&fp)[MI], const v4u (&fq)[MJ], const v4u& unit) {
        part<0, SUMS>(fp, fq, unit);
        if constexpr (Mfma<T>::PARTS > 1) part<1, SUMS>(fp, fq, unit);
        if constexpr (Mfma<T>::PARTS > 2) {
            part<2, SUMS>(fp, fq, unit);
            part<3, SUMS>(fp, fq, unit);
        }
    }

    // D += P Q^T over all c, in steps of 128 bytes of c.  LDS: two buffers of (BI + BJ) * 128 bytes.
    // A step's fragments are read in two halves, each while the half before it is being multiplied: the second half in front of the
    // step's barrier, the next step's first one behind it.  The barrier says that the next step's tile is in LDS and that nobody
    // reads this step's any more.
    template <bool TP, bool TQ, bool SUMS> PSH_OP void multiply(const Operand<T>& p, const Operand<T>& q, unsigned char* lds) {
        constexpr int KC = 128 / (int)sizeof(T);
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int wi = (wave % WI) * (BI / WI), wj = (wave / WI) * (BJ / WJ);
        const int l = lane & 15, g = lane >> 4;
        v4u unit = {0, 0, 0, 0};
        clear<SUMS>(unit);
        const int nc = p.nc, tiles = (nc + KC - 1) / KC;
        if (tiles <= 0) return;
        Stager<T, BI, THREADS, TP> sp(p);
        Stager<T, BJ, THREADS, TQ> sq(q);
        v4u fp[2][MI], fq[2][MJ];
        const auto read = [&](int s, const unsigned char* at) {
#pragma unroll
            for (int a = 0; a < MI; ++a) {
                const int i = wi + a * 16 + l;
                fp[s][a] = *reinterpret_cast<const v4u*>(at + i * 128 + unit_of(i, s * 4 + g) * 16);
            }
#pragma unroll
            for (int b = 0; b < MJ; ++b) {
                const int j = wj + b * 16 + l;
                fq[s][b] = *reinterpret_cast<const v4u*>(at + BI * 128 + j * 128 + unit_of(j, s * 4 + g) * 16);
            }
        };
        const auto fetch = [&](int t) {
            sp.fetch(p, t * KC);
            sq.fetch(q, t * KC);
        };
        const auto store = [&](unsigned char* at) {
            sp.store(at);
            sq.store(at + BI * 128);
        };
        fetch(0);
        store(lds);
        if (tiles > 1) fetch(1);
        __syncthreads();
        read(0, lds);
        // (two steps a turn, in which the buffer is a constant of the code and goes into the offsets of the LDS instructions: 115 us for 122 us in 12
        // groups of 2500 rows, 513 -> 257, fp32; not where both operands are transposed, V lines a thread: their registers do not suffice, 350 us for 298 us)
        constexpr bool TWO = sizeof(T) == 8 || !TQ;
        const auto step = [&](auto buffer, int t) {
            unsigned char* const cur = lds + (int)buffer * (BI + BJ) * 128;
            unsigned char* const nxt = lds + (1 - (int)buffer) * (BI + BJ) * 128;
            const bool second = nc - t * KC > KC / 2;   // (else nothing but zeros there)
            if (second) read(1, cur);
            __builtin_amdgcn_sched_barrier(0);
            parts<SUMS>(fp[0], fq[0], unit);
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < tiles) store(nxt);
            if (t + 2 < tiles) fetch(t + 2);
            __syncthreads();
            if (t + 1 < tiles) read(0, nxt);
            __builtin_amdgcn_sched_barrier(0);
            if (second) parts<SUMS>(fp[1], fq[1], unit);
            if constexpr (SUMS && sizeof(T) == 4)
                if ((t & 3) == 3 || t + 1 == tiles) fold();
        };
        if constexpr (TWO) {
            for (int t = 0; t < tiles; t += 2) {
                step(std::integral_constant<int, 0>(), t);
                if (t + 1 < tiles) step(std::integral_constant<int, 1>(), t + 1);
            }
        } else {
            for (int t = 0; t < tiles; ++t) step(t & 1, t);
        }
    }

    // The same for bf16 by direct loads, in steps of 64 bytes of c.  LDS: three buffers of (BI + BJ) * 64 bytes, so that the loads of two
    // steps are in flight while one is being multiplied.  A step's fragments are read while the step before it is being multiplied; its
    // barrier says that they are in everyone's registers, so that their buffer can be filled again, and that the next step's tile is in LDS.
    // Reads of LDS and loads are issued between the matrix instructions, a few behind each block of rows: in one go they would hold the wave up
    // until the queues have taken them, with its matrix instructions behind them.
    template <bool TP, bool TQ, bool SUMS> PSH_OP void multiply_direct(const Operand<bf16_t>& p, const Operand<bf16_t>& q, unsigned char* lds, unsigned block_x) {
        typedef Direct<BI, THREADS, TP> DP;
        typedef Direct<BJ, THREADS, TQ> DQ;
        constexpr int KC = DP::KC, LOADS = DP::PER + DQ::PER;
        constexpr unsigned BUF = DP::BYTES + DQ::BYTES;
        const int wave = wave_id();
        const int wi = (wave % WI) * (BI / WI), wj = (wave / WI) * (BJ / WJ);
        v4u unit = {0, 0, 0, 0};
        clear<SUMS>(unit);
        const int nc = p.nc, tiles = (nc + KC - 1) / KC, whole = nc / KC;
        if (tiles <= 0) return;
        const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
        v4u fp[2][MI], fq[2][MJ];
        // Rows of c are often powers of two apart, and then one step's reads of all rows lie in one or two of the 16 channels of an L2, 256
        // bytes each.  So every workgroup of an XCD begins elsewhere, two steps from the one before it.
        const int turn = whole > 0 ? (int)((block_x >> 3) * 2 % whole) : 0;
        const auto at = [&](int t) { return (t + turn < whole ? t + turn : t + turn - whole) * KC; };
        const auto bring = [&](int t, unsigned buf) {
            if (t < whole) {
                const typename DP::Loads lp(p, at(t), base + buf, wave);
                const typename DQ::Loads lq(q, at(t), base + buf + DP::BYTES, wave);
#pragma unroll
                for (int k = 0; k < DP::PER; ++k) lp.issue(k);
#pragma unroll
                for (int k = 0; k < DQ::PER; ++k) lq.issue(k);
            } else if (t < tiles) {
                DP::fetch_tail(p, t * KC, lds + buf, wave);
                DQ::fetch_tail(q, t * KC, lds + buf + DP::BYTES, wave);
            }
        };
        // multiplies a step's fragments, set H, reads the next one's from `from` into the other set, and with LOAD issues the loads of step t
        const auto step = [&](auto h, auto load, unsigned from, int t, unsigned to) {
            constexpr int H = decltype(h)::value, READS = MI + MJ, AT_A_TIME = (READS * 4 + 3 * MI - 1) / (3 * MI);
            const typename DP::Reads rp(lds + from, wi);
            const typename DQ::Reads rq(lds + from + DP::BYTES, wj);
            const typename DP::Loads lp(p, at(t), base + to, wave);
            const typename DQ::Loads lq(q, at(t), base + to + DP::BYTES, wave);
#pragma unroll
            for (int a = 0; a < MI; ++a) {
#pragma unroll
                for (int r = a * AT_A_TIME; r < (a + 1) * AT_A_TIME && r < READS; ++r) {
                    if (r < MJ) fq[1 - H][r] = rq.block(r);
                    else fp[1 - H][r - MJ] = rp.block(r - MJ);
                }
                if constexpr (decltype(load)::value) {
#pragma unroll
                    for (int k = a * LOADS / MI; k < (a + 1) * LOADS / MI; ++k) {
                        if (k < DP::PER) lp.issue(k);
                        else lq.issue(k - DP::PER);
                    }
                }
#pragma unroll
                for (int b = 0; b < MJ; ++b) Mfma<T>::template step<0>(fp[H][a], fq[H][b], acc[a][b]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (SUMS) sums<0>(fp[H], unit);
        };
        constexpr std::integral_constant<int, 0> even{};
        constexpr std::integral_constant<int, 1> odd{};
        // all loads have landed but those of the `later` newest steps
        const auto wait = [&](auto later) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(LOADS * decltype(later)::value) : "memory");
            __syncthreads();
        };
        bring(0, 0);
        bring(1, BUF);
        bring(2, 2 * BUF);
        if (2 < whole) wait(std::integral_constant<int, 2>());
        else wait(std::integral_constant<int, 0>());
        {
            const typename DP::Reads rp(lds, wi);
            const typename DQ::Reads rq(lds + DP::BYTES, wj);
#pragma unroll
            for (int b = 0; b < MJ; ++b) fq[0][b] = rq.block(b);
#pragma unroll
            for (int a = 0; a < MI; ++a) fp[0][a] = rp.block(a);
        }
        unsigned cur = 0, nxt = BUF;   // buffers of steps t and t + 1
        const auto on = [&]() {
            cur = nxt;
            nxt = nxt == 2 * BUF ? 0 : nxt + BUF;
        };
        int t = 0;
        for (; t + 4 < whole; t += 2) {
            wait(odd);
            step(even, std::true_type(), nxt, t + 3, cur);
            on();
            wait(odd);
            step(odd, std::true_type(), nxt, t + 4, cur);
            on();
        }
        for (; t < tiles; t += 2) {
            if (t + 2 < whole) wait(odd);
            else wait(even);
            bring(t + 3, cur);
            step(even, std::false_type(), nxt, 0, 0);   // (behind the last step it reads what nobody uses)
            on();
            if (t + 1 < tiles) {
                if (t + 3 < whole) wait(odd);
                else wait(even);
                bring(t + 4, cur);
                step(odd, std::false_type(), nxt, 0, 0);
                on();
            }
        }
    }

    // f(i, j, v[4]) for the results of this lane: units i .. i + 3 of row j for fp32 accumulators; for fp64 ones the
    // four units are i, i + 4, i + 8, i + 12
    template <class F> PSH_OP void each(F f) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int wi = (wave % WI) * (BI / WI), wj = (wave / WI) * (BJ / WJ);
#pragma unroll
        for (int a = 0; a < MI; ++a)
#pragma unroll
            for (int b = 0; b < MJ; ++b)
                f(wi + a * 16 + Mfma<T>::row(lane >> 4, 0), wj + b * 16 + (lane & 15), acc[a][b]);
    }
};

constexpr int lds_bytes(int bi, int bj, bool direct) { return (bi + bj) * (direct ? 3 * 64 : 2 * 128); }

// consecutive tiles on one XCD: workgroups go to the 8 XCDs in turn, each of which has an L2 of its own
PSH_OP long xcd_order(long b, long total) {
    const long per = (total + 7) / 8;
    return (b & 7) * per + (b >> 3);
}

template <class T> struct RowsArgs {   // forward and dx
    Parts parts;
    const T* rows_in; long ld_in;      // x, or dp
    const T* weight; long ld_w, stride_w;
    const T* bias; long stride_b;
    T* out;                            // [rows, n_out] contiguous
    float* wide;                       // the same before its rounding, or NULL (bf16 only)
    int n_in, n_out, nonlin;
    long slots, tiles_i;
};

// A result tile goes to memory through LDS (a lane holds four units of one row, and neighbouring lanes neighbouring rows, so stores
// from registers would be pieces of 8 to 32 bytes): rows of COLS elements, 16-byte units permuted within a row by XOR with swz(row).
template <class T, int COLS> PSH_OP T* tile_at(unsigned char* lds, int row, int col, int swz) {
    const int byte = col * (int)sizeof(T);
    return reinterpret_cast<T*>(lds + row * COLS * (int)sizeof(T) + (((byte >> 4) ^ swz) << 4) + (byte & 15));
}
template <class T, int COLS, class S> PSH_OP void store_tile(unsigned char* lds, T* out, long ld, int rows, int cols, S swz) {
    constexpr int V = 16 / (int)sizeof(T), UNITS = COLS / V;
    for (int id = threadIdx.x; id < rows * UNITS; id += blockDim.x) {
        const int r = id / UNITS, c = id % UNITS * V;
        if (c >= cols) continue;
        const v4u v = *reinterpret_cast<const v4u*>(tile_at<T, COLS>(lds, r, c, swz(r)));
        T* const o = out + r * ld + c;
        if (c + V <= cols) {
            __builtin_memcpy(o, &v, 16);
        } else {
            T e[V];
            __builtin_memcpy(e, &v, 16);
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (c + k < cols) o[k] = e[k];
        }
    }
}

template <class T, int BI, int BJ, int WI, int WJ, bool TW, bool DIRECT> PSH_OP void rows_tile(const RowsArgs<T>& a, unsigned block_x, unsigned char* lds) {
    const long id = xcd_order(block_x, a.slots * a.tiles_i);
    if (id >= a.slots * a.tiles_i) return;
    // blocks of 8 tiles of units for all rows, one after the other: what the workgroups of an XCD read at a time stays in its L2
    const long block = id / (a.slots * 8), in_block = id - block * a.slots * 8, wide = a.tiles_i - block * 8 < 8 ? a.tiles_i - block * 8 : 8;
    const Piece q = find_piece(a.parts, (int)(in_block / wide));
    const int i0 = (int)(block * 8 + in_block % wide) * BI;
    const int nj = q.end - q.begin, ni = min(BI, a.n_out - i0);
    if (nj <= 0) return;
    if (q.part >= a.parts.n) {   // rows behind the last group
        for (int k = threadIdx.x; k < nj * ni; k += blockDim.x) {
            const long at = (long)(q.begin + k / ni) * a.n_out + i0 + k % ni;
            a.out[at] = T(0);
            if (a.wide) a.wide[at] = 0;
        }
        return;
    }
    const T* const w = a.weight + (long)q.part * a.stride_w;
    const Operand<T> p{TW ? w + i0 : w + (long)i0 * a.ld_w, a.ld_w, ni, a.n_in};
    const Operand<T> x{a.rows_in + (long)q.begin * a.ld_in, a.ld_in, nj, a.n_in};
    Tile<T, BI, BJ, WI, WJ> tile;
    if constexpr (DIRECT) tile.template multiply_direct<TW, false, false>(p, x, lds, block_x);
    else tile.template multiply<TW, false, false>(p, x, lds);
    typedef typename Wide<T>::type W;
    const T* const b = a.bias ? a.bias + (long)q.part * a.stride_b + i0 : nullptr;
    const auto swz = [](int j) { return j & (BI * (int)sizeof(T) / 16 - 1) & 15; };
    constexpr int step = sizeof(T) == 8 ? 4 : 1;
    const auto finish = [&](auto f) {
        W bias[4];
        int bias_of = -1;
        tile.each([&](int i, int j, auto v) {
            if (i != bias_of) {   // (the units change in the outer loop of each())
#pragma unroll
                for (int r = 0; r < 4; ++r) bias[r] = b ? to_wide(b[min(i + step * r, ni - 1)]) : W(0);
                bias_of = i;
            }
            T e[4];
            W y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[r] = f((W)(v[r] + bias[r]));
                e[r] = to_elem<T>(y[r]);
            }
            if constexpr (sizeof(T) == 2) {
                if (a.wide && j < nj) {
                    float* const o = a.wide + (long)(q.begin + j) * a.n_out + i0 + i;
                    if (i + 4 <= ni) {
                        __builtin_memcpy(o, y, 16);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (i + r < ni) o[r] = y[r];
                    }
                }
            }
            if constexpr (sizeof(T) == 8) {
#pragma unroll
                for (int r = 0; r < 4; ++r) *tile_at<T, BI>(lds, j, i + 4 * r, swz(j)) = e[r];
            } else {
                __builtin_memcpy(__builtin_assume_aligned(tile_at<T, BI>(lds, j, i, swz(j)), 4 * sizeof(T)), e, 4 * sizeof(T));
            }
        });
    };
    if (a.nonlin == PSH_NL_TANH) finish([](W x) { return tanh_w(x); });
    else if (a.nonlin == PSH_NL_SIGMOID) finish([](W x) { return sigmoid_w(x); });
    else if (a.nonlin == PSH_NL_RELU) finish([](W x) { return x <= W(0) ? W(0) : x; });   // a NaN stays one
    else finish([](W x) { return x; });
    __syncthreads();
    store_tile<T, BI>(lds, a.out + (long)q.begin * a.n_out + i0, a.n_out, nj, ni, swz);
}
template <class T, int BI, int BJ, int WI, int WJ, bool TW, bool DIRECT>
__global__ __launch_bounds__(64 * WI * WJ, BI * BJ > 4096 || (sizeof(T) == 2 && TW) ? 2 : TW ? 3 : 4) void k_rows(const RowsArgs<T> a) {
    extern __shared__ __align__(16) unsigned char lds[];
    rows_tile<T, BI, BJ, WI, WJ, TW, DIRECT>(a, blockIdx.x, lds);
}

// dp = dy f'(y), rounded to the element type as the gradient that reaches a layer's product in any composition of
// layers is.  Rows behind the last group have no part in any sum.  Bound by bytes: 76800 x 64 fp64 in 19 us (6.2 TB/s, two reads and a write).
// A thread takes V neighbouring elements, which lie in one row (V divides its length, or the rows follow one another).
template <class T, class Y, int V> __global__ __launch_bounds__(256) void k_preact(long n, int cols, const T* dy, long ld, const Y* y, int nonlin, T* dp) {
    for (long k = ((long)blockIdx.x * 256 + threadIdx.x) * V; k < n; k += (long)gridDim.x * 256 * V) {
        long at = k;
        if (ld != cols) {
            const long r = k / cols;
            at = r * ld + (k - r * cols);
        }
        const int live = (int)min((long)V, n - k);
        T up[V], e[V];
        Y value[V];
        if (live == V) {
            __builtin_memcpy(up, dy + at, sizeof(up));
            __builtin_memcpy(value, y + k, sizeof(value));
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                up[i] = i < live ? dy[at + i] : T(0);
                value[i] = i < live ? y[k + i] : Y(0);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = to_elem<T>(to_wide(up[i]) * nonlin_slope_w(nonlin, to_wide(value[i])));
        if (live == V) {
            __builtin_memcpy(dp + k, e, sizeof(e));
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < live) dp[k + i] = e[i];
        }
    }
}
template <class T, class Y> void launch_preact(const psh_linear_desc* d, const Y* y, T* dp, hipStream_t st) {
    const long n = (long)d->rows * d->out_dim;
    constexpr int V = 16 / (int)sizeof(T);
    const bool wide = d->ld_dy == d->out_dim || d->out_dim % V == 0;
    const long blocks = (n + 1023) / 1024;
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    if (wide) hipLaunchKernelGGL((k_preact<T, Y, V>), grid, dim3(256), 0, st, n, (int)d->out_dim, (const T*)d->dy, (long)d->ld_dy, y, (int)d->nonlin, dp);
    else hipLaunchKernelGGL((k_preact<T, Y, 1>), grid, dim3(256), 0, st, n, (int)d->out_dim, (const T*)d->dy, (long)d->ld_dy, y, (int)d->nonlin, dp);
}

template <class T> struct GradArgs {   // dW, db
    Parts parts;                       // pieces of the contraction
    const T* dp; long ld_dp;
    const T* x; long ld_x;
    T* dw; T* db;                      // [G, n, k], [G, n]
    CutPlaces places;
    typename Wide<T>::type* part_w;    // [places, n, k] and [places, n]: sums of groups that are cut into several pieces
    typename Wide<T>::type* part_b;
    int n, k;
    long slots, tiles_i, tiles_j;
};

template <class T, int BI, int BJ, int WI, int WJ, bool DIRECT> PSH_OP void weights_tile(const GradArgs<T>& a, unsigned block_x, unsigned char* lds) {
    const long tiles = a.tiles_i * a.tiles_j, total = a.slots * tiles;
    const long id = xcd_order(block_x, total);
    if (id >= total) return;
    const int slot = (int)(id / tiles);
    const Piece q = find_piece(a.parts, slot);
    if (q.part >= a.parts.n || (q.j > 0 && q.begin >= q.end)) return;
    const int i0 = (int)(id % tiles / a.tiles_j) * BI, j0 = (int)(id % a.tiles_j) * BJ;
    const int ni = min(BI, a.n - i0), nj = min(BJ, a.k - j0), rows = max(0, q.end - q.begin);
    const Operand<T> p{a.dp + (long)q.begin * a.ld_dp + i0, a.ld_dp, ni, rows};
    const Operand<T> x{a.x + (long)q.begin * a.ld_x + j0, a.ld_x, nj, rows};
    Tile<T, BI, BJ, WI, WJ> tile;
    const bool whole = q.part_end - q.part_begin <= a.parts.L;   // no other piece: the result itself
    const bool sums = j0 == 0 && a.db;
    if constexpr (DIRECT) {
        if (sums) tile.template multiply_direct<true, true, true>(p, x, lds, block_x);
        else tile.template multiply_direct<true, true, false>(p, x, lds, block_x);
    } else {
        if (sums) tile.template multiply<true, true, true>(p, x, lds);
        else tile.template multiply<true, true, false>(p, x, lds);
    }
    constexpr int step = sizeof(T) == 8 ? 4 : 1;
    const long at = (whole ? q.part : a.places.first(a.parts, q.part, q.part_begin) + q.j) * a.n;
    if (a.dw) {
        // rows of the tile are output units here
        const auto put = [&](auto* out) {
            typedef typename std::remove_pointer<decltype(out)>::type O;
            const auto swz = [](int i) { return ((i >> 2) & 3) * (int)sizeof(O); };
            // as many rows at a time as the operands' buffers hold
            constexpr int ROOM = lds_bytes(BI, BJ, DIRECT) / (BJ * (int)sizeof(O)), ROWS = ROOM >= BI ? BI : ROOM >= BI / 2 ? BI / 2 : BI / 4;
            static_assert(ROWS <= ROOM && ROWS % 16 == 0, "whole blocks of a matrix instruction's rows");
            for (int first = 0; first < BI; first += ROWS) {
                if (first > 0) __syncthreads();
                tile.each([&](int i, int j, auto v) {
                    if (ROWS < BI && (i < first || i >= first + ROWS)) return;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        *tile_at<O, BJ>(lds, i - first + step * r, j, swz(i + step * r)) = to_elem<O>(v[r]);
                });
                __syncthreads();
                if (first < ni)
                    store_tile<O, BJ>(lds, out + (at + i0 + first) * a.k + j0, a.k, min(ROWS, ni - first), nj, swz);
            }
        };
        if (whole) put(a.dw);
        else put(a.part_w);
    }
    if (sums && (threadIdx.x & 15) == 0) {
        const int wave = threadIdx.x >> 6, wi = (wave % WI) * (BI / WI) + wave / WI * tile.OWN * 16;
#pragma unroll
        for (int m = 0; m < tile.OWN; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = wi + m * 16 + Mfma<T>::row((threadIdx.x & 63) >> 4, r);
                if (i >= ni) continue;
                if (whole) a.db[at + i0 + i] = to_elem<T>(tile.ones[m][r]);
                else a.part_b[at + i0 + i] = tile.ones[m][r];
            }
    }
}

template <class T, int BI, int BJ, int WI, int WJ, bool DIRECT>
__global__ __launch_bounds__(64 * WI * WJ, BI * BJ > 4096 || sizeof(T) == 2 ? 2 : 3) void k_weights(const GradArgs<T> a) {
    extern __shared__ __align__(16) unsigned char lds[];
    weights_tile<T, BI, BJ, WI, WJ, DIRECT>(a, blockIdx.x, lds);
}

// dW, db and dx in one launch, where both go by tiles of one kind: the first workgroups of dx begin while the last ones of dW run.
// Together and one after the other: 64 groups of 1200 rows, 64 -> 64, fp64: 50 and 57 us; 12 of 2500, 513 -> 257, fp32: 299 and 317 us (53
// TFLOP/s); 8 of 4096, 1024 -> 2048, bf16: 396 and 448 us (694 TFLOP/s).
template <class T, int BIG, int SMALL, int WI, int WJ, bool DIRECT>
__global__ __launch_bounds__(64 * WI * WJ, BIG * SMALL > 4096 || sizeof(T) == 2 ? 2 : 3) void k_both(const GradArgs<T> w, const RowsArgs<T> r, unsigned first) {
    extern __shared__ __align__(16) unsigned char lds[];
    if (blockIdx.x < first) weights_tile<T, SMALL, BIG, WI, WJ, DIRECT>(w, blockIdx.x, lds);
    else rows_tile<T, BIG, SMALL, WI, WJ, true, DIRECT>(r, blockIdx.x - first, lds);
}

// sums of the pieces of the groups that have several, in the order of the rows; V elements a thread (V divides n k), their loads of all
// pieces in flight together
template <class T, int V> __global__ __launch_bounds__(256) void k_join(const GradArgs<T> a) {
    typedef typename Wide<T>::type W;
    const long nw = a.dw ? (long)a.n * a.k : 0, nb = a.db ? a.n : 0;
    for (int g = blockIdx.y; g < a.parts.n; g += gridDim.y) {
        const int begin = a.parts.at(g), end = a.parts.at(g + 1);
        if (end - begin <= a.parts.L) continue;
        const int pieces = piece_count(begin, end, a.parts.L);
        const long first = a.places.first(a.parts, g, begin);
        const long threads = (long)gridDim.x * 256, me = (long)blockIdx.x * 256 + threadIdx.x;
        for (long e = me * V; e < nw; e += threads * V) {
            const W* const src = a.part_w + first * nw + e;
            W s[V] = {};
            T out[V];
            for (int j0 = 0; j0 < pieces; j0 += 32) {   // (in blocks, for the same reason as in fold())
                W p[V] = {};
#pragma unroll 4
                for (int j = j0; j < min(pieces, j0 + 32); ++j) {
                    W v[V];
                    __builtin_memcpy(v, src + j * nw, sizeof(v));
#pragma unroll
                    for (int i = 0; i < V; ++i) p[i] += v[i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) s[i] += p[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = to_elem<T>(s[i]);
            __builtin_memcpy(a.dw + (long)g * nw + e, out, sizeof(out));
        }
        for (long e = me; e < nb; e += threads) {
            const W* const src = a.part_b + first * nb + e;
            W s = 0;
            for (int j0 = 0; j0 < pieces; j0 += 32) {
                W p = 0;
                for (int j = j0; j < min(pieces, j0 + 32); ++j) p += src[j * nb];
                s += p;
            }
            a.db[(long)g * nb + e] = to_elem<T>(s);
        }
    }
}

template <class K> int allow_lds(psh_ctx* c, K kernel, int bytes) {
    if (bytes > 64 * 1024) PSH_HIP(c, hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return PSH_OK;
}

constexpr int TOO_MANY = -1;   // (workgroups of a launch)

// the grid of a call by such tiles, as a multiple of the 8 XCDs
template <class T> long rows_grid(RowsArgs<T>& a, int rows, int bi, int bj) {
    a.parts.L = bj;
    a.slots = parts_slots(rows, a.parts.n, bj);
    a.tiles_i = (a.n_out + bi - 1) / bi;
    const long total = (a.slots * a.tiles_i + 7) / 8 * 8;
    return total > 0x3fffffffL ? TOO_MANY : total;
}
int too_many_tiles(psh_ctx* c) {
    set_err(c, "grouped_linear: too many tiles for one launch");
    return PSH_ERR_UNSUPPORTED;
}

template <class T, int BI, int BJ, int WI, int WJ, bool TW, bool DIRECT> int launch_rows(psh_ctx* c, RowsArgs<T>& a, int rows, hipStream_t st) {
    const long total = rows_grid(a, rows, BI, BJ);
    if (total == TOO_MANY) return too_many_tiles(c);
    constexpr int lds = lds_bytes(BI, BJ, DIRECT);
    static_assert(lds >= BI * BJ * (int)sizeof(T), "a result tile goes through it");
    const auto kernel = k_rows<T, BI, BJ, WI, WJ, TW, DIRECT>;
    const int rc = allow_lds(c, kernel, lds);
    if (rc != PSH_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)total), dim3(64 * WI * WJ), lds, st, a);
    PSH_HIP(c, hipGetLastError());
    return PSH_OK;
}

template <class T, bool TW> int run_rows(psh_ctx* c, RowsArgs<T>& a, TileKind kind, int rows, hipStream_t st) {
    if (kind == TILE_ROWS16) return launch_rows<T, 64, 16, 4, 1, TW, false>(c, a, rows, st);
    if constexpr (sizeof(T) == 2) {
        if (kind == TILE_128) return launch_rows<T, 128, 128, 2, 4, TW, false>(c, a, rows, st);
        if (kind == TILE_128_DIRECT) return launch_rows<T, 128, 128, 2, 2, TW, true>(c, a, rows, st);
        if (kind == TILE_256_DIRECT) return launch_rows<T, 256, 128, 2, 2, TW, true>(c, a, rows, st);
    }
    return launch_rows<T, 64, 64, 2, 2, TW, false>(c, a, rows, st);
}

int check(psh_ctx* c, const psh_linear_desc* d, bool grad) {
    if (!c || !d) return PSH_ERR_ARG;
    if (d->dtype < PSH_F64 || d->dtype > PSH_BF16 || d->nonlin < PSH_NL_NONE || d->nonlin > PSH_NL_SIGMOID) {
        set_err(c, "grouped_linear: unknown dtype or nonlinearity");
        return PSH_ERR_ARG;
    }
    if (d->n_groups < 1 || d->rows < 0 || d->in_dim < 1 || d->out_dim < 1) { set_err(c, "grouped_linear: invalid sizes"); return PSH_ERR_ARG; }
    if (d->n_groups > (1 << 30) || d->rows > (1 << 30)) { set_err(c, "grouped_linear: at most 2^30 rows and groups"); return PSH_ERR_UNSUPPORTED; }
    if (d->y_wide && d->dtype != PSH_BF16) { set_err(c, "grouped_linear: y_wide is for PSH_BF16"); return PSH_ERR_ARG; }
    if (!d->offsets || (d->rows > 0 && !d->x) || !d->weight || d->ld_x < d->in_dim || d->ld_w < d->in_dim || d->stride_w < 0 || d->stride_b < 0) {
        set_err(c, "grouped_linear: NULL array or a row stride below the row's length");
        return PSH_ERR_ARG;
    }
    if (!grad) {
        if (d->rows > 0 && !d->y) { set_err(c, "grouped_linear: y is NULL"); return PSH_ERR_ARG; }
        return PSH_OK;
    }
    if (d->rows > 0 && (!d->dy || d->ld_dy < d->out_dim || (d->nonlin != PSH_NL_NONE && !d->y && !d->y_wide))) {
        set_err(c, "grouped_linear_grad: dy (and y, with a nonlinearity) must be given");
        return PSH_ERR_ARG;
    }
    const GradSpace s = grad_space(d);
    if (s.total > 0 && (!d->workspace || d->workspace_bytes < s.total || ((uintptr_t)d->workspace & 255))) {
        set_err(c, "grouped_linear_grad: the workspace is too small or not 256-byte aligned");
        return PSH_ERR_ARG;
    }
    return PSH_OK;
}

// the weight gradient, with the input gradient in the same launch if `r` is given
template <class T, int BIG, int SMALL, int WI, int WJ, bool DIRECT> int launch_weights(psh_ctx* c, GradArgs<T>& a, RowsArgs<T>* r, int rows, hipStream_t st) {
    a.slots = parts_slots(rows, a.parts.n, a.parts.L);
    a.tiles_i = (a.n + SMALL - 1) / SMALL;
    a.tiles_j = a.dw ? (a.k + BIG - 1) / BIG : 1;
    const long total = (a.slots * a.tiles_i * a.tiles_j + 7) / 8 * 8, also = r ? rows_grid(*r, rows, BIG, SMALL) : 0;
    if (total > 0x3fffffffL || also == TOO_MANY) return too_many_tiles(c);
    constexpr int lds = lds_bytes(BIG, SMALL, DIRECT);
    const auto alone = k_weights<T, SMALL, BIG, WI, WJ, DIRECT>;
    const auto both = k_both<T, BIG, SMALL, WI, WJ, DIRECT>;
    const int rc = r ? allow_lds(c, both, lds) : allow_lds(c, alone, lds);
    if (rc != PSH_OK) return rc;
    if (r) hipLaunchKernelGGL(both, dim3((unsigned)(total + also)), dim3(64 * WI * WJ), lds, st, a, *r, (unsigned)total);
    else hipLaunchKernelGGL(alone, dim3((unsigned)total), dim3(64 * WI * WJ), lds, st, a);
    PSH_HIP(c, hipGetLastError());
    return PSH_OK;
}

template <class T> int forward(psh_ctx* c, const psh_linear_desc* d) {
    RowsArgs<T> a{};
    a.parts = Parts{d->offsets, d->n_groups, d->rows, 0};
    a.rows_in = (const T*)d->x; a.ld_in = d->ld_x;
    a.weight = (const T*)d->weight; a.ld_w = d->ld_w; a.stride_w = d->stride_w;
    a.bias = (const T*)d->bias; a.stride_b = d->stride_b;
    a.out = (T*)d->y;
    a.wide = d->y_wide;
    a.n_in = d->in_dim; a.n_out = d->out_dim; a.nonlin = d->nonlin;
    return run_rows<T, false>(c, a, forward_kind(d), d->rows, (hipStream_t)d->stream);
}

template <class T> int backward(psh_ctx* c, const psh_linear_desc* d) {
    typedef typename Wide<T>::type W;
    hipStream_t st = (hipStream_t)d->stream;
    const GradSpace s = grad_space(d);
    unsigned char* const space = (unsigned char*)d->workspace;
    const T* dp = (const T*)d->dy;
    long ld_dp = d->ld_dy;
    if (d->nonlin != PSH_NL_NONE && d->rows > 0) {
        if (sizeof(T) == 2 && d->y_wide) launch_preact(d, (const float*)d->y_wide, (T*)space, st);
        else launch_preact(d, (const T*)d->y, (T*)space, st);
        PSH_HIP(c, hipGetLastError());
        dp = (const T*)space;
        ld_dp = d->out_dim;
    }
    RowsArgs<T> r{};
    const GradPlan plan = grad_plan(d);
    if (d->dx && d->rows > 0) {
        r.parts = Parts{d->offsets, d->n_groups, d->rows, 0};
        r.rows_in = dp; r.ld_in = ld_dp;
        r.weight = (const T*)d->weight; r.ld_w = d->ld_w; r.stride_w = d->stride_w;
        r.out = (T*)d->dx;
        r.n_in = d->out_dim; r.n_out = d->in_dim; r.nonlin = PSH_NL_NONE;
        if (!plan.joint) {
            const int rc = run_rows<T, true>(c, r, plan.rows, d->rows, st);
            if (rc != PSH_OK) return rc;
        }
    }
    if (d->dweight || d->dbias) {
        GradArgs<T> a{};
        a.parts = Parts{d->offsets, d->n_groups, d->rows, (int)grad_piece(d, grad_direct(d))};
        a.places = cut_places(d->rows, d->n_groups, a.parts.L);
        a.dp = dp; a.ld_dp = ld_dp;
        a.x = (const T*)d->x; a.ld_x = d->ld_x;
        a.dw = (T*)d->dweight; a.db = (T*)d->dbias;
        a.part_w = (W*)(space + s.dp); a.part_b = (W*)(space + s.dp + s.part_w);
        a.n = d->out_dim; a.k = d->in_dim;
        RowsArgs<T>* const also = plan.joint ? &r : nullptr;
        const TileKind kind = plan.weights;
        int rc;
        if constexpr (sizeof(T) == 2) {
            if (kind == TILE_64) rc = launch_weights<T, 64, 64, 2, 2, false>(c, a, also, d->rows, st);
            else if (kind == TILE_128) rc = launch_weights<T, 128, 128, 2, 4, false>(c, a, also, d->rows, st);
            else if (kind == TILE_128_DIRECT) rc = launch_weights<T, 128, 128, 2, 2, true>(c, a, also, d->rows, st);
            else rc = launch_weights<T, 256, 128, 2, 2, true>(c, a, also, d->rows, st);
        } else {
            rc = launch_weights<T, 64, 64, 2, 2, false>(c, a, also, d->rows, st);
        }
        if (rc != PSH_OK) return rc;
        if (d->rows > a.parts.L) {
            const long n = (long)a.n * (a.k + 1);
            // 16 bytes a thread once there are threads enough for four workgroups a CU: 37 us for 56 us where 24 pieces of 2048 x 1024 are summed, 10 us
            // for 7.6 us with 64 groups of 64 x 64
            const bool wide = (long)a.n * a.k % 4 == 0 && (int64_t)d->n_groups * n >= (1 << 20);
            const long blocks = (n + (wide ? 1023 : 255)) / (wide ? 1024 : 256);
            const unsigned bx = (unsigned)(blocks < 1024 ? blocks : 1024);
            const unsigned gy = (unsigned)(d->n_groups < 65535 ? d->n_groups : 65535);
            if (wide) hipLaunchKernelGGL((k_join<T, 4>), dim3(bx, gy), dim3(256), 0, st, a);
            else hipLaunchKernelGGL((k_join<T, 1>), dim3(bx, gy), dim3(256), 0, st, a);
            PSH_HIP(c, hipGetLastError());
        }
    }
    return PSH_OK;
}

}  // namespace

extern "C" int64_t psh_grouped_linear_grad_workspace(const psh_linear_desc* d) {
    if (!d || d->n_groups < 1 || d->rows < 0 || d->in_dim < 1 || d->out_dim < 1) return PSH_ERR_ARG;
    return grad_space(d).total;
}

extern "C" int psh_grouped_linear(psh_ctx* c, const psh_linear_desc* d) {
    const int rc = check(c, d, false);
    if (rc != PSH_OK || d->rows == 0) return rc;
    PSH_ON_DEVICE(c);
    if (d->dtype == PSH_F64) return forward<double>(c, d);
    if (d->dtype == PSH_F32) return forward<float>(c, d);
    return forward<bf16_t>(c, d);
}

extern "C" int psh_grouped_linear_grad(psh_ctx* c, const psh_linear_desc* d) {
    const int rc = check(c, d, true);
    if (rc != PSH_OK) return rc;
    PSH_ON_DEVICE(c);
    if (d->dtype == PSH_F64) return backward<double>(c, d);
    if (d->dtype == PSH_F32) return backward<float>(c, d);
    return backward<bf16_t>(c, d);
}
