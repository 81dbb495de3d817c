// The recurrence of a policy with memory: the causal convolution and the selective state-space scan over recorded
// sequences and for single steps, with their gradients (psh_causal_conv*, psh_selective_scan* of include/pysimhip.h).
#include <hip/hip_runtime.h>

#include <utility>

#include "psh_ops.h"

namespace {

struct Policies : Shares {
    PSH_OP int of(int seq) const { return n == 1 || !groups ? 0 : wave_search(n - 1, seq, [&](int p) { return at(p); }); }
};

// (vectors and not arrays in a struct: those the compiler keeps in memory once a branch writes them)
template <class T, int E> struct Vec { typedef T type __attribute__((ext_vector_type(E))); };

// E elements of a line with n valid ones starting at c; elements behind it are zero
template <int E, class T> PSH_OP void load_line(typename Wide<T>::type (&out)[E], const T* line, int c, int n, bool vec) {
    if (vec && c + E <= n) {
        const typename Vec<T, E>::type p = *reinterpret_cast<const typename Vec<T, E>::type*>(line + c);
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = to_wide((T)p[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = c + e < n ? to_wide(line[c + e]) : typename Wide<T>::type(0);
    }
}
template <int E, class T> PSH_OP void store_line(T* line, const typename Wide<T>::type (&in)[E], int c, int n, bool vec) {
    if (vec && c + E <= n) {
        typename Vec<T, E>::type p;
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = to_elem<T>(in[e]);
        *reinterpret_cast<typename Vec<T, E>::type*>(line + c) = p;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (c + e < n) line[c + e] = to_elem<T>(in[e]);
    }
}

template <int E, class T> PSH_OP typename Vec<T, E>::type load_raw(const T* line, int c, int n, bool vec) {
    if (vec && c + E <= n) return *reinterpret_cast<const typename Vec<T, E>::type*>(line + c);
    typename Vec<T, E>::type out;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = c + e < n ? line[c + e] : T(0);
    return out;
}

// ====================================================================================================== convolution
// y[t, d] = f(b[d] + sum_k w[d, k] x[t - (K - 1) + k, d]).  A lane holds V neighbouring channels (16 bytes) and walks down a run of rows with
// the last K inputs in registers, so every input is read once (K - 1 rows of a run again at its start).  One wave: one piece
// of a sequence, its lanes split over the channels first and over runs with what is left of the 64.
// Bound by the bytes of x and y: 120000 x 128 fp32 in 32 us (3.9 TB/s; a copy reaches 4.7).  131072 x 256 bf16 in 42 us (3.2 TB/s) is bound by
// neither: the vector pipes are busy for half of it (18 instructions an element, two of them an exponential and a reciprocal), and the
// waves wait for the other half, with the loads of four rows each in flight.
template <class T> struct ConvArgs {
    Parts parts;
    Policies pol;
    const T* x; long ld_x;
    const typename Wide<T>::type *w, *b;
    const T* state; long stride_state;
    T* y;
    T* last; long stride_last;
    int D, silu, lanes_c;   // lanes across channels (a power of two)
    int run;                // rows of one lane's run
    bool vec;
    // gradients
    const T* dy; long ld_dy;
    const T* dlast;
    T* dx; T* dstate;
    typename Wide<T>::type* part;   // [slots, D, K + 1]: weight and bias gradients of a piece
};
constexpr int CONV_BATCH = 4;        // rows whose loads are in flight together

template <class T, int K> PSH_OP void conv_params(typename Wide<T>::type (&w)[K], typename Wide<T>::type& b, const ConvArgs<T>& a, int p, int c) {
    const bool in = c < a.D;
#pragma unroll
    for (int k = 0; k < K; ++k) w[k] = in ? a.w[((long)p * a.D + c) * K + k] : 0;
    b = in && a.b ? a.b[(long)p * a.D + c] : 0;
}

// input of sequence `part` at row `row` (carried ones before its first row) for V channels from c
template <int V, int K, class T> PSH_OP void conv_input(typename Wide<T>::type (&out)[V], const ConvArgs<T>& a, const Piece& q, int row, int c) {
    if (row >= q.part_begin) {
        load_line<V>(out, a.x + (long)row * a.ld_x, c, a.D, a.vec);
        return;
    }
    const int k = row - q.part_begin + K - 1;
#pragma unroll
    for (int e = 0; e < V; ++e)
        out[e] = a.state && k >= 0 && c + e < a.D ? to_wide(a.state[q.part * a.stride_state + (long)(c + e) * (K - 1) + k]) : typename Wide<T>::type(0);
}

template <class T, int V, int K> __global__ __launch_bounds__(256) void k_conv(const ConvArgs<T> a, long slots) {
    typedef typename Wide<T>::type W;
    const long slot = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (slot >= slots) return;
    const Piece q = find_piece(a.parts, (int)slot);
    const int lane = threadIdx.x & 63, sub = lane / a.lanes_c;
    const int c = ((int)blockIdx.y * a.lanes_c + lane % a.lanes_c) * V;
    const int r0 = q.begin + sub * a.run, r1 = min(q.end, r0 + a.run);
    if (q.part >= a.parts.n) {
        const W zero[V] = {};
        if (c < a.D)
            for (int r = r0; r < r1; ++r) store_line<V>(a.y + (long)r * a.D, zero, c, a.D, a.vec);
        return;
    }
    if (q.j > 0 && q.begin >= q.end) return;
    const int p = a.pol.of(q.part);
    if (c >= a.D) return;
    if (q.j == 0 && sub == 0 && a.last) {   // the K - 1 newest inputs
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            W v[V];
            conv_input<V, K>(v, a, q, q.part_end - (K - 1) + k, c);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < a.D) a.last[q.part * a.stride_last + (long)(c + e) * (K - 1) + k] = to_elem<T>(v[e]);
        }
    }
    if (r0 >= r1) return;
    W w[V][K], b[V], win[K][V];
#pragma unroll
    for (int e = 0; e < V; ++e) conv_params<T, K>(w[e], b[e], a, p, c + e);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) conv_input<V, K>(win[k], a, q, r0 - (K - 1) + k, c);
    for (int r = r0; r < r1; r += CONV_BATCH) {
        typename Vec<T, V>::type in[CONV_BATCH];
#pragma unroll
        for (int i = 0; i < CONV_BATCH; ++i) in[i] = load_raw<V>(a.x + (long)min(r + i, r1 - 1) * a.ld_x, c, a.D, a.vec);
#pragma unroll
        for (int i = 0; i < CONV_BATCH; ++i) {
            if (r + i >= r1) break;
            W y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                win[K - 1][e] = to_wide((T)in[i][e]);
                W s = b[e];
#pragma unroll
                for (int k = 0; k < K; ++k) s += w[e][k] * win[k][e];
                y[e] = a.silu ? silu_w(s) : s;
            }
            store_line<V>(a.y + (long)(r + i) * a.D, y, c, a.D, a.vec);
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) win[k][e] = win[k + 1][e];
        }
    }
}

// One row per sequence: 16384 sequences of 128 channels in fp32 take 11.4 us (5.9 TB/s, nothing but the carried inputs, x and y).
// A wave takes step_seqs() neighbouring sequences and 64 channels: with one policy (ONE) their parameters are read
// once.  A thread reads its carried inputs before it writes the new ones, which may be in the same place.
template <class T> constexpr int step_seqs() { return sizeof(T) == 8 ? 2 : 4; }
template <class T, int K, bool ONE> __global__ __launch_bounds__(256) void k_conv_step(const ConvArgs<T> a, int n_seqs, int per_row) {
    typedef typename Wide<T>::type W;
    constexpr int STEP_SEQS = step_seqs<T>();
    const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int s0 = (int)(id / per_row) * STEP_SEQS, c = (int)(id % per_row) * 64 + (threadIdx.x & 63);
    if (s0 >= n_seqs) return;
    const int live = min(STEP_SEQS, n_seqs - s0), cc = min(c, a.D - 1);
    W w[K], b;
    if constexpr (ONE) conv_params<T, K>(w, b, a, 0, cc);
    T in[STEP_SEQS][K];
#pragma unroll
    for (int i = 0; i < STEP_SEQS; ++i) {
        const long s = s0 + min(i, live - 1);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) in[i][k] = a.state ? a.state[s * a.stride_state + (long)cc * (K - 1) + k] : T(0);
        in[i][K - 1] = a.x[s * a.ld_x + cc];
    }
#pragma unroll
    for (int i = 0; i < STEP_SEQS; ++i) {
        if (i >= live) break;
        const long s = s0 + i;
        if constexpr (!ONE) conv_params<T, K>(w, b, a, a.pol.of((int)s), cc);
        if (c >= a.D) continue;
        W sum = b;
#pragma unroll
        for (int k = 0; k < K; ++k) sum += w[k] * to_wide(in[i][k]);
        a.y[s * a.D + c] = to_elem<T>(a.silu ? silu_w(sum) : sum);
        if (a.last)
#pragma unroll
            for (int k = 0; k < K - 1; ++k) a.last[s * a.stride_last + (long)c * (K - 1) + k] = in[i][k + 1];
    }
}

// dx[t] = sum_k w[k] dpre[t + K-1-k],  dw[k] = sum_t dpre[t] x[t - (K-1) + k],  db = sum_t dpre[t],  dpre = dy f'(pre).
// A run of rows needs dpre of K - 1 rows behind it, which it computes itself from the inputs (again): nothing but x and dy is read.
// Rows t < 0 of a sequence are its carried inputs: the first run of a sequence computes their gradients too.
// 131072 x 256 bf16: 82 us (2.5 TB/s); the vector pipes are busy for 71 % of that, with 47 instructions an element.
template <class T, int V, int K> __global__ __launch_bounds__(256) void k_conv_grad(const ConvArgs<T> a, long slots) {
    typedef typename Wide<T>::type W;
    const long slot = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (slot >= slots) return;
    const Piece q = find_piece(a.parts, (int)slot);
    const int lane = threadIdx.x & 63, sub = lane / a.lanes_c;
    const int c = ((int)blockIdx.y * a.lanes_c + lane % a.lanes_c) * V;
    const int r0 = q.begin + sub * a.run, r1 = min(q.end, r0 + a.run);
    if (q.part >= a.parts.n) {
        const W zero[V] = {};
        if (c < a.D && a.dx)
            for (int r = r0; r < r1; ++r) store_line<V>(a.dx + (long)r * a.D, zero, c, a.D, a.vec);
        return;
    }
    const int p = a.pol.of(q.part);
    const bool live = c < a.D;
    W w[V][K], b[V], dw[V][K], db[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        conv_params<T, K>(w[e], b[e], a, p, c + e);
        db[e] = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[e][k] = 0;
    }
    const bool head = q.j == 0 && sub == 0;   // also the carried inputs' run
    const int first = head ? q.part_begin - (K - 1) : r0;
    if (live && (r0 < r1 || head)) {
        // win: inputs up to row t, dpre: its gradients up to row t; the result of row t - (K - 1) is complete with row t
        W win[K][V], dp[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) dp[k][e] = 0;
        const int start = head ? q.part_begin : r0, stop = head && r0 >= r1 ? q.part_begin : r1;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) conv_input<V, K>(win[k], a, q, start - (K - 1) + k, c);
        // rows start .. stop + K - 2; those behind the run only for dpre, those behind the sequence not at all
        for (int t0 = start; t0 < stop + K - 1; t0 += CONV_BATCH) {
        typename Vec<T, V>::type in[CONV_BATCH], up[CONV_BATCH];
#pragma unroll
        for (int i = 0; i < CONV_BATCH; ++i) {
            const int t = t0 + i;
            in[i] = up[i] = T(0);
            if (t < q.part_end && t < stop + K - 1) {
                in[i] = load_raw<V>(a.x + (long)t * a.ld_x, c, a.D, a.vec);
                up[i] = load_raw<V>(a.dy + (long)t * a.ld_dy, c, a.D, a.vec);
            }
        }
#pragma unroll
        for (int i = 0; i < CONV_BATCH; ++i) {
            const int t = t0 + i;
            if (t >= stop + K - 1) break;
            if (t < q.part_end) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    win[K - 1][e] = to_wide((T)in[i][e]);
                    const W dy = to_wide((T)up[i][e]);
                    W s = b[e];
#pragma unroll
                    for (int k = 0; k < K; ++k) s += w[e][k] * win[k][e];
                    dp[K - 1][e] = a.silu ? dy * silu_slope_w(s, sigmoid_w(s)) : dy;
                    if (t < stop) {
                        db[e] += dp[K - 1][e];
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[e][k] += dp[K - 1][e] * win[k][e];
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) dp[K - 1][e] = 0;
            }
            const int row = t - (K - 1);   // dx[row] = sum_k w[k] dpre[row + K-1-k], dp[m] = dpre of row + m
            if (row >= first && row < max(stop, start)) {
                W g[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    g[e] = 0;
#pragma unroll
                    for (int k = 0; k < K; ++k) g[e] += w[e][k] * dp[K - 1 - k][e];
                }
                const int newest = row - (q.part_end - (K - 1));   // which of the K - 1 newest inputs it is, if any
                if (a.dlast && newest >= 0 && newest < K - 1)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (c + e < a.D) g[e] += to_wide(a.dlast[((long)q.part * a.D + c + e) * (K - 1) + newest]);
                if (row >= q.part_begin) {
                    if (a.dx) store_line<V>(a.dx + (long)row * a.D, g, c, a.D, a.vec);
                } else if (a.dstate) {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (c + e < a.D) a.dstate[((long)q.part * a.D + c + e) * (K - 1) + row - q.part_begin + K - 1] = to_elem<T>(g[e]);
                }
            }
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    win[k][e] = win[k + 1][e];
                    dp[k][e] = dp[k + 1][e];
                }
        }
        }
    }
    if (!a.part) return;
    // runs of the piece: lanes with equal channels, lanes_c apart
#pragma unroll
    for (int e = 0; e < V; ++e) {
        for (int m = a.lanes_c; m < 64; m *= 2) {
            db[e] += __shfl_xor(db[e], m);
#pragma unroll
            for (int k = 0; k < K; ++k) dw[e][k] += __shfl_xor(dw[e][k], m);
        }
        if (sub == 0 && c + e < a.D) {
            W* const o = a.part + (slot * a.D + c + e) * (K + 1);
#pragma unroll
            for (int k = 0; k < K; ++k) o[k] = dw[e][k];
            o[K] = db[e];
        }
    }
}

// ============================================================================== sums over the pieces of a policy
// out[p, m] = sum of part[slot, m] over the slots of policy p's sequences, in two passes of about the square root of their
// number, in the order of the slots: 4 to 9 us each, the time of a few dependent loads.  `slot_of(p)`: the first slot of policy p.
template <class W> struct JoinArgs : PolicySlots {   // (seg = 0: few enough slots for one pass over `part`)
    const W* part; W* mid;
    W *out0, *out1, *out2;    // columns [0, n0) -> out0, then n1 -> out1, then n2 -> out2 (NULL: not wanted)
    long n0, n1, n2, split;   // split: column layout [.., split + 1] with the last of each row going to out1 (0: plain)
};
template <class W> __global__ __launch_bounds__(256) void k_join_mid(const JoinArgs<W> a) {
    const int seg = blockIdx.x;
    const int p = a.pol.n == 1 ? 0 : wave_search(a.pol.n - 1, seg, [&](int i) { return a.seg_of(i); });
    const long m = (long)blockIdx.y * 256 + threadIdx.x, cols = a.n0 + a.n1 + a.n2;
    if (m >= cols) return;
    int64_t begin, stop;
    if (!a.segment(seg, p, begin, stop)) return;
    W s = 0;
    long k = begin;
    for (; k + 8 <= stop; k += 8) {
        W v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = a.part[(k + i) * cols + m];
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; k < stop; ++k) s += a.part[k * cols + m];
    a.mid[(long)seg * cols + m] = s;
}
template <class W> __global__ __launch_bounds__(256) void k_join_out(const JoinArgs<W> a) {
    const int p = blockIdx.x;
    const long m = (long)blockIdx.y * 256 + threadIdx.x, cols = a.n0 + a.n1 + a.n2;
    if (m >= cols) return;
    int first, n;
    a.of_policy(p, first, n);
    const W* const mid = a.seg ? a.mid : a.part;
    W s = 0;
    int k0 = 0;
    for (; k0 + 8 <= n; k0 += 8) {
        W v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mid[(long)(first + k0 + i) * cols + m];
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; k0 < n; ++k0) s += mid[(long)(first + k0) * cols + m];
    if (a.split) {   // convolution: [D, K + 1] rows of weights and a bias
        const long d = m / (a.split + 1), k = m - d * (a.split + 1);
        if (k < a.split) { if (a.out0) a.out0[(long)p * (cols / (a.split + 1)) * a.split + d * a.split + k] = s; }
        else if (a.out1) a.out1[(long)p * (cols / (a.split + 1)) + d] = s;
    } else if (m < a.n0) {
        if (a.out0) a.out0[p * a.n0 + m] = s;
    } else if (m < a.n0 + a.n1) {
        if (a.out1) a.out1[p * a.n1 + m - a.n0] = s;
    } else if (a.out2) {
        a.out2[p * a.n2 + m - a.n0 - a.n1] = s;
    }
}
int join_seg(long slots) {
    int seg = 32;
    while ((long)seg * seg < slots) seg *= 2;
    return seg;
}
long join_segs(long slots, int policies) { return policy_segments(slots, policies, join_seg(slots)); }
template <class W> int run_join(psh_ctx* c, JoinArgs<W>& a, long slots, hipStream_t st) {
    const unsigned by = (unsigned)((a.n0 + a.n1 + a.n2 + 255) / 256);
    a.seg = 0;
    if (slots <= 96 * (long)a.pol.n) {   // one pass of a few dozen loads, eight in flight, is done before a second launch would begin
        hipLaunchKernelGGL(k_join_out<W>, dim3((unsigned)a.pol.n, by), dim3(256), 0, st, a);
        PSH_HIP(c, hipGetLastError());
        return PSH_OK;
    }
    a.seg = join_seg(slots);
    hipLaunchKernelGGL(k_join_mid<W>, dim3((unsigned)join_segs(slots, a.pol.n), by), dim3(256), 0, st, a);
    PSH_HIP(c, hipGetLastError());
    hipLaunchKernelGGL(k_join_out<W>, dim3((unsigned)a.pol.n, by), dim3(256), 0, st, a);
    PSH_HIP(c, hipGetLastError());
    return PSH_OK;
}

// ============================================================================================================= scan
// A channel's N states are spread over LPC neighbouring lanes, NP each, so that B and C of a step, which all channels
// share, are read from LDS by broadcast, the sum over the states takes log2(LPC) DPP additions, and the sum over the
// channels that the gradients of B and C need starts in registers.  A workgroup of 4 waves runs 256 / LPC channels over one
// piece of a sequence, TS steps at a time: it loads the TS x channels tiles of u, delta (and z, dy) together, one 8- or
// 16-byte load per thread and array, computes the step sizes once per element, and leaves dt and dt u in LDS for the steps.
// TS = 16 steps (8 in fp64) are also as far apart as the states that the forward pass stores for the gradient (`check`): 4 N / TS
// bytes an element, where storing every state would be 16 times as many, and computing from the beginning again impossible.
constexpr int THREADS = 256;
template <class W, int NP, int LPC> struct Shape {
    static constexpr int TS = sizeof(W) == 8 ? 8 : 16;   // steps of a tile = distance of the stored states
    static constexpr int CB = THREADS / LPC;             // channels of a workgroup
    static constexpr int NL = NP * LPC;                  // states, padded
    static constexpr int E = TS * CB >= THREADS ? TS * CB / THREADS : 1;
    static constexpr int LOADERS = TS * CB / E;          // threads that load (all but for the widest fp64 shape)
    static constexpr int CP = CB + 64 / LPC;             // stride of rows that the lanes of a channel write one each of: other banks for each
};

template <class T> struct ScanArgs {
    typedef typename Wide<T>::type W;
    Parts parts;             // pieces
    Policies pol;
    int D, N;
    const T *u, *delta, *z, *B, *C;
    long ld_u, ld_delta, ld_z, ld_B, ld_C;
    const W *A, *skip, *bias;
    const W* state; long stride_state;
    T* y;
    W* last; long stride_last;
    W* check;                // [rows / TS + n + 1, D, N] states before every tile
    W* carry;                // [slots, D, N]: states (adjoint states) at the pieces' beginnings (ends), NULL: pieces are whole sequences
    W* carry_dt;             // [slots, D]
    const int* order;        // sequences from the longest to the shortest, NULL: as they come
    int blocks;              // channel blocks
    bool vec_d, vec_n;       // wide loads of channel rows / of states
    bool vec_bc;             // and of rows of B and C (single steps)
    // gradients
    const T* dy; long ld_dy;
    const W* dlast;
    T *du, *ddelta, *dz, *dB, *dC;
    W* dstate;
    W* part;                 // [slots, D N + 2 D] parameter gradients of a piece
    W* part_bc;              // [channel blocks, rows, 2 N], NULL: one block, results go to dB and dC
};

// exp(dt A) from A prepared once per lane.  A of minus infinity (a state without memory) becomes the lowest finite number: the
// steps behind a sequence's end in a tile are steps of size 0, which must leave a state as it is.
PSH_OP float decay_rate(float a) {
    const float r = a * (float)PSH_LOG2E;
    return r < -3.4028234663852886e38f ? -3.4028234663852886e38f : r;
}
PSH_OP double decay_rate(double a) { return a < -1.7976931348623157e308 ? -1.7976931348623157e308 : a; }
PSH_OP float decay(float dt, float rate) { return exp2_w(dt * rate); }
PSH_OP double decay(double dt, double rate) { return exp_w(dt * rate); }
// sum of g a h' A from a sum with prepared rates
PSH_OP float rate_unit(float) { return (float)PSH_LN2; }
PSH_OP double rate_unit(double) { return 1.; }

template <int CTRL> PSH_OP float dpp_move(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
template <int CTRL> PSH_OP double dpp_move(double x) {
    return __hiloint2double(__builtin_amdgcn_mov_dpp(__double2hiint(x), CTRL, 0xf, 0xf, true),
                            __builtin_amdgcn_mov_dpp(__double2loint(x), CTRL, 0xf, 0xf, true));
}
// sum over the LPC lanes of a channel, in all of them
template <int LPC, class W> PSH_OP W sum_states(W x) {
    x += dpp_move<0xB1>(x);                              // quad_perm [1, 0, 3, 2]
    x += dpp_move<0x4E>(x);                              // quad_perm [2, 3, 0, 1]
    if constexpr (LPC >= 8) x += dpp_move<0x141>(x);     // row_half_mirror: the other quad of the eight
    if constexpr (LPC >= 16) x += dpp_move<0x140>(x);    // row_mirror: the other eight of the row
    return x;
}
// [a.low a.high], [b.low b.high] -> sums of a's halves in the low half, of b's in the high half
PSH_OP float halves32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
PSH_OP float halves16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
PSH_OP double halves32(double a, double b) {
    const auto l = __builtin_amdgcn_permlane32_swap((unsigned)__double2loint(a), (unsigned)__double2loint(b), false, false);
    const auto h = __builtin_amdgcn_permlane32_swap((unsigned)__double2hiint(a), (unsigned)__double2hiint(b), false, false);
    return __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
}
PSH_OP double halves16(double a, double b) {
    const auto l = __builtin_amdgcn_permlane16_swap((unsigned)__double2loint(a), (unsigned)__double2loint(b), false, false);
    const auto h = __builtin_amdgcn_permlane16_swap((unsigned)__double2hiint(a), (unsigned)__double2hiint(b), false, false);
    return __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
}

// The compiler takes x to be computed here.  (Not for what a DPP instruction reads next: the wait states it needs are not counted across this.)
PSH_OP void fixed(float& x) { asm volatile("" : "+v"(x)); }
PSH_OP void fixed(double& x) { asm volatile("" : "+v"(x)); }

// Keeps the scheduler from running several steps' exponentials side by side: in fp64 one step has enough of them to fill the
// pipe, and more do not fit into the registers.
template <class W, int NP> PSH_OP void step_fence() {
    if constexpr (sizeof(W) == 8 && NP > 1) __builtin_amdgcn_sched_barrier(0);
}

template <class W> struct alignas(2 * sizeof(W)) Pair { W dt, dtu; };

// NP states of a lane from / to [.., D, N] memory
template <int NP, class W> PSH_OP void load_states(W (&h)[NP], const W* p, int n, int N, bool vec) { load_line<NP>(h, p, n, N, vec); }

// What a thread loads of a tile: E channels of one step, as they are in memory.
template <class T, int E> struct Rows {
    typename Vec<T, E>::type u, delta, z, dy;
};
template <class T, class SH> struct Loader {
    typedef typename Wide<T>::type W;
    static constexpr int E = SH::E, TS = SH::TS, CB = SH::CB;
    int t, c, d;     // step in the tile, first channel in the block and overall
    bool on;
    W bias[E], skip[E];

    PSH_OP Loader(const ScanArgs<T>& a, int c0, int p) {
        on = (int)threadIdx.x < SH::LOADERS;
        t = (int)threadIdx.x / (CB / E) % TS;
        c = (int)threadIdx.x % (CB / E) * E;
        d = c0 + c;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool in = d + e < a.D;
            bias[e] = in && a.bias ? a.bias[(long)p * a.D + d + e] : W(0);
            skip[e] = in && a.skip ? a.skip[(long)p * a.D + d + e] : W(0);
        }
    }
    template <bool GRAD> PSH_OP void fetch(Rows<T, E>& r, const ScanArgs<T>& a, int row0, int end) const {
        const long row = row0 + t;
        if (!on || row >= end) {
            r.u = r.delta = r.z = r.dy = T(0);
            return;
        }
        r.u = load_raw<E>(a.u + row * a.ld_u, d, a.D, a.vec_d);
        r.delta = load_raw<E>(a.delta + row * a.ld_delta, d, a.D, a.vec_d);
        if (a.z) r.z = load_raw<E>(a.z + row * a.ld_z, d, a.D, a.vec_d);
        if constexpr (GRAD) r.dy = load_raw<E>(a.dy + row * a.ld_dy, d, a.D, a.vec_d);
    }
};

// B and C of a tile: TS x NL values each, zero behind the piece's end and behind N
template <class T, class SH> struct StepRows {
    typedef typename Wide<T>::type W;
    static constexpr int COUNT = SH::TS * SH::NL, PER = (COUNT + THREADS - 1) / THREADS;
    T b[PER], c[PER];
    template <bool WITH_C> PSH_OP void fetch(const ScanArgs<T>& a, int row0, int end) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int id = (int)threadIdx.x + k * THREADS, n = id % SH::NL;
            const long row = row0 + id / SH::NL;
            const bool in = id < COUNT && row < end && n < a.N;
            b[k] = in ? a.B[row * a.ld_B + n] : T(0);
            if constexpr (WITH_C) c[k] = in ? a.C[row * a.ld_C + n] : T(0);
        }
    }
    template <bool WITH_C> PSH_OP void store(W* sb, W* sc) const {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int id = (int)threadIdx.x + k * THREADS;
            if (id >= COUNT) continue;
            sb[id] = to_wide(b[k]);
            if constexpr (WITH_C) sc[id] = to_wide(c[k]);
        }
    }
};

// Sequences from the longest to the shortest (to 1/256 of the longest), for launches of whole sequences: workgroups are
// handed out in this order, so that those that run last, or that share a CU, are not by chance the long ones.  It takes 3 us; 500 sequences
// of 120000 rows, 128 channels, then take 89 us for 132 us as they come, the gradient of 256 of 131072 rows, 256 channels, 600 us for 809 us.
constexpr int ORDER_MOST = 16384;   // sequences; with more, chance evens the CUs out
__global__ __launch_bounds__(1024) void k_order(const Parts p, int* order) {
    __shared__ int count[256], most;
    const int tid = threadIdx.x;
    if (tid == 0) most = 1;
    if (tid < 256) count[tid] = 0;
    __syncthreads();
    int m = 1;
    for (int s = tid; s < p.n; s += 1024) m = max(m, p.at(s + 1) - p.at(s));
    for (int k = 32; k > 0; k /= 2) m = max(m, __shfl_xor(m, k));
    if ((tid & 63) == 0) atomicMax(&most, m);
    __syncthreads();
    const float scale = 255.f / (float)most;
    for (int s = tid; s < p.n; s += 1024) atomicAdd(&count[255 - min(255, (int)((float)max(0, p.at(s + 1) - p.at(s)) * scale))], 1);
    __syncthreads();
    if (tid < 64) {   // exclusive prefix sums of 4 buckets a lane
        int c[4], sum = 0;
        for (int i = 0; i < 4; ++i) {
            c[i] = count[tid * 4 + i];
            sum += c[i];
        }
        int before = sum;
        for (int k = 1; k < 64; k *= 2) {
            const int o = __shfl_up(before, k);
            before += tid >= k ? o : 0;
        }
        before -= sum;
        for (int i = 0; i < 4; ++i) {
            count[tid * 4 + i] = before;
            before += c[i];
        }
    }
    __syncthreads();
    for (int s = tid; s < p.n; s += 1024) order[atomicAdd(&count[255 - min(255, (int)((float)max(0, p.at(s + 1) - p.at(s)) * scale))], 1)] = s;
}

// Which slot and channel block a workgroup works on.  In an ordered launch work item k is channel block k % blocks of the (k / blocks)-th
// longest sequence, and workgroup i takes item i in even, the mirrored one in odd runs of 256: workgroups go round the
// CUs, so a CU that got the longest of one run gets the shortest of the next.
template <class T> PSH_OP void work_of(const ScanArgs<T>& a, int& slot, int& block) {
    const int blocks = a.blocks;
    unsigned i = blockIdx.x;
    const unsigned ordered = (unsigned)a.parts.n * blocks;
    if (a.order && i < ordered) {
        const unsigned run = i / 256, r = i % 256, len = min(256u, ordered - run * 256);
        i = run & 1 ? run * 256 + len - 1 - r : i;
        slot = a.order[i / blocks];
    } else {
        slot = (int)(i / blocks);
    }
    block = (int)(i % blocks);
}

// h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t and y_t = (C_t . h_t + D u_t) silu(z_t) along a piece.
// Bound by instruction issue: a state costs an exponential (16 cycles a wave) and four or five others (4 each) a step, 32 to 36 cycles; the vector
// pipes are busy all the time.  131072 x 256 x 16 states, bf16, with `check`: 164 us (2.5 TB/s); 120000 x 128 x 16, fp32, without: 89 us.
// CARRY: only the state at the piece's end from zero and the sum of its step sizes, for the joining
// of pieces; otherwise y as well, from the state at the piece's beginning.
template <class T, int NP, int LPC, bool CARRY> __global__ __launch_bounds__(THREADS) void k_scan(const ScanArgs<T> a) {
    typedef typename Wide<T>::type W;
    typedef Shape<W, NP, LPC> SH;
    constexpr int TS = SH::TS, CB = SH::CB, CP = SH::CP, E = SH::E, NL = SH::NL;
    __shared__ Pair<W> s_dt[TS][CB];
    __shared__ __align__(16) W s_b[TS * NL];
    __shared__ __align__(16) W s_c[CARRY ? 1 : TS * NL];
    __shared__ __align__(16) W s_y[CARRY ? 1 : TS][CP];
    int slot, block;
    work_of(a, slot, block);
    const int c0 = block * CB;
    const Piece q = find_piece(a.parts, slot);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ql = lane % LPC, cl = wave * (64 / LPC) + lane / LPC;     // lane of the channel, channel of the block
    const int d = c0 + cl, n0 = ql * NP;
    if (q.part >= a.parts.n) {
        if constexpr (!CARRY)
            for (int r = q.begin; r < q.end; ++r)
                for (int c = c0 + threadIdx.x; c < min(c0 + CB, a.D); c += THREADS) a.y[(long)r * a.D + c] = T(0);
        return;
    }
    const bool final = q.end >= q.part_end;
    if (q.begin >= q.end && q.j > 0) return;
    if (CARRY && q.j == 0 && final) return;                             // a sequence of one piece
    const int p = a.pol.of(q.part);
    W h[NP], rate[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) h[i] = 0;
    if (d < a.D) {
        load_states<NP>(rate, a.A + ((long)p * a.D + d) * a.N, n0, a.N, a.vec_n);
        if constexpr (!CARRY) {
            if (a.carry && !(q.j == 0 && final)) load_states<NP>(h, a.carry + ((long)slot * a.D + d) * a.N, n0, a.N, a.vec_n);
            else if (a.state) load_states<NP>(h, a.state + q.part * a.stride_state + (long)d * a.N, n0, a.N, a.vec_n);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) rate[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) rate[i] = decay_rate(rate[i]);
    W total = 0;
    const Loader<T, SH> ld(a, c0, p);
    Rows<T, E> now, next;
    StepRows<T, SH> bc;
    ld.template fetch<false>(next, a, q.begin, q.end);
    bc.template fetch<!CARRY>(a, q.begin, q.end);
    const long check0 = check_slot(q, TS);
    for (int r0 = q.begin, tile = 0; r0 < q.end; r0 += TS, ++tile) {
        now = next;
        if (ld.on) {
            const int live = r0 + ld.t < q.end ? -1 : 0;   // (a step size of 0 leaves the state as it is)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const W dt = masked(softplus_w(to_wide((T)now.delta[e]) + ld.bias[e]), live);
                s_dt[ld.t][ld.c + e] = Pair<W>{dt, dt * to_wide((T)now.u[e])};
            }
        }
        bc.template store<!CARRY>(s_b, s_c);
        __syncthreads();
        if (r0 + TS < q.end) {
            ld.template fetch<false>(next, a, r0 + TS, q.end);
            bc.template fetch<!CARRY>(a, r0 + TS, q.end);
        }
        if constexpr (!CARRY) {
            if (a.check && d < a.D) store_line<NP>(a.check + ((check0 + tile) * a.D + d) * a.N, h, n0, a.N, a.vec_n);
        }
        // (four states a lane keep a wave busy for long enough by four steps; fewer do not: 73 us rolled, 69 us unrolled for 32 policies' 256
        // rollouts of 65437 steps, 96 channels, 8 states, fp32)
#pragma unroll NP >= 4 ? 1 : TS
        for (int t1 = 0; t1 < TS; t1 += LPC < TS ? LPC : TS) {
            W keep = 0;
#pragma unroll
            for (int t2 = 0; t2 < (LPC < TS ? LPC : TS); ++t2) {
                const int t = t1 + t2;
                const Pair<W> x = s_dt[t][cl];
                W y = 0;
                const W* const bt = s_b + t * NL + n0;
                const W* const ct = s_c + (CARRY ? 0 : t * NL + n0);
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    h[i] = decay(x.dt, rate[i]) * h[i] + x.dtu * bt[i];
                    if constexpr (!CARRY) y += ct[i] * h[i];
                }
                if constexpr (CARRY) {
                    total += x.dt;
                } else {
                    y = sum_states<LPC>(y);
                    keep = ql == t2 ? y : keep;
                }
                step_fence<W, NP>();
            }
            if constexpr (!CARRY) {
                if (ql < TS) s_y[t1 + ql][cl] = keep;
            }
        }
        __syncthreads();
        if constexpr (!CARRY) {
            const long row = r0 + ld.t;
            if (ld.on && row < q.end && ld.d < a.D) {
                W out[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    W v = s_y[ld.t][ld.c + e];
                    if (a.skip) v += ld.skip[e] * to_wide((T)now.u[e]);
                    out[e] = a.z ? v * silu_w(to_wide((T)now.z[e])) : v;
                }
                store_line<E>(a.y + row * a.D, out, ld.d, a.D, a.vec_d);
            }
        }
    }
    if (d >= a.D) return;
    if constexpr (CARRY) {
        store_line<NP>(a.carry + ((long)slot * a.D + d) * a.N, h, n0, a.N, a.vec_n);
        if (ql == 0) a.carry_dt[(long)slot * a.D + d] = total;
    } else if (final && a.last) {
        store_line<NP>(a.last + q.part * a.stride_last + (long)d * a.N, h, n0, a.N, a.vec_n);
    }
}

// carry[slot]: from the end state of every piece (from zero) to the state at every piece's beginning; for the gradient
// (BACK) from the adjoint state at every piece's beginning to that at its end, from the last piece on.
// A piece maps its beginning h to P h + own with P = exp(A sum dt), and such maps compose: 8 threads take an eighth of the
// pieces of a state each, compose them, find their beginnings from the eighths before, and walk through theirs again.
// 9 us for 256 pieces of 4096 states; 52 us with one thread a state.
constexpr int JOIN_GROUPS = 8, JOIN_COLS = 256 / JOIN_GROUPS;
template <class T, bool BACK> __global__ __launch_bounds__(256) void k_scan_join(const ScanArgs<T> a) {
    typedef typename Wide<T>::type W;
    __shared__ W s_p[JOIN_GROUPS][JOIN_COLS], s_h[JOIN_GROUPS][JOIN_COLS];
    const int s = blockIdx.x, col = threadIdx.x % JOIN_COLS, grp = threadIdx.x / JOIN_COLS;
    const long cols = (long)a.D * a.N;
    const int begin = a.parts.at(s), end = a.parts.at(s + 1);
    if (end - begin <= a.parts.L) return;
    const int n = piece_count(begin, end, a.parts.L), first = a.parts.first_slot(s);
    const int p = a.pol.of(s);
    const long m = min((long)blockIdx.y * JOIN_COLS + col, cols - 1);   // (threads behind the last state repeat it, and do not store)
    const bool mine = (long)blockIdx.y * JOIN_COLS + col < cols;
    const int d = (int)(m / a.N);
    const W rate = decay_rate(a.A[p * cols + m]);
    const int per = (n + JOIN_GROUPS - 1) / JOIN_GROUPS, k0 = min(n, grp * per), k1 = min(n, k0 + per);
    const auto slot_of = [&](int k) { return (long)(BACK ? first + n - 1 - k : first + k); };
    constexpr int AHEAD = 8;   // loads in flight: the chain itself is one fma a piece
    W h = 0, total = 0;
    for (int k = k0; k < k1; k += AHEAD) {
        W own[AHEAD], dt[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const long slot = slot_of(min(k1 - 1, k + i));
            own[i] = a.carry[slot * cols + m];
            dt[i] = a.carry_dt[slot * a.D + d];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (k + i < k1) {
                h = decay(dt[i], rate) * h + own[i];
                total += dt[i];
            }
    }
    s_p[grp][col] = decay(total, rate);
    s_h[grp][col] = h;
    __syncthreads();
    if (BACK) h = a.dlast ? a.dlast[s * cols + m] : W(0);
    else h = a.state ? a.state[s * a.stride_state + m] : W(0);
    for (int g = 0; g < grp; ++g)
        if (g * per < n) h = s_p[g][col] * h + s_h[g][col];
    for (int k = k0; k < k1; k += AHEAD) {
        W own[AHEAD], dt[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const long slot = slot_of(min(k1 - 1, k + i));
            own[i] = a.carry[slot * cols + m];
            dt[i] = a.carry_dt[slot * a.D + d];
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (k + i < k1) {
                if (mine) a.carry[slot_of(k + i) * cols + m] = h;
                h = decay(dt[i], rate) * h + own[i];
            }
    }
}

// The adjoint recurrence of a piece, tiles of TS steps from its end:  g_t = C_t dy0_t + G_{t+1},  G_t = a_t g_t,  where dy0 = dy silu(z).
// Each tile first runs forward from its stored state and keeps a_t and h_{t-1} of its steps in registers (2 TS NP values
// per lane), then backward:  dA += G h_{t-1} dt,  ddt = sum_n G h_{t-1} A + u sum_n g B,  du = dt sum_n g B + D dy0,  and, summed over
// the channels, dB = g dt u and dC = dy0 h.  The sums over a wave's 16 channels swap halves and quarters of the wave, so that eight sums
// take 16 instructions; those over the waves go through LDS, those over workgroups through memory (k_sum_bc), none by atomics.
// Bound by instruction issue for three quarters of the time, by what two waves a SIMD leave uncovered of the steps' latency for the rest: 101 vector
// instructions a step for four states of 16 channels, 52 of them the formulas, 33 the sums, besides 12 reads and writes of LDS.  131072 x 256 x 16
// states, bf16: 590 us (690 cycles a step of a wave, of which the vector pipe is busy for 450); 65437 x 96 x 8, fp32, 256 sequences: 145 us,
// the time of the longest of them (vector pipes busy for 60 %).
// CARRY: only G at the piece's beginning, from zero.
template <class T, int NP, int LPC, bool CARRY> __global__ __launch_bounds__(THREADS, 2) void k_scan_grad(const ScanArgs<T> a) {
    typedef typename Wide<T>::type W;
    typedef Shape<W, NP, LPC> SH;
    constexpr int TS = SH::TS, CB = SH::CB, CP = SH::CP, E = SH::E, NL = SH::NL;
    constexpr int NV = 2 * NP < 4 ? 4 : 2 * NP;     // gradients of B and C of a step and lane, padded
    constexpr int GS = LPC < TS ? LPC : TS;         // steps whose sums the lanes of a channel collect, one each
    __shared__ Pair<W> s_dt[TS][CB];
    __shared__ __align__(16) W s_dy[TS][CB];
    __shared__ __align__(16) W s_sz[CARRY ? 1 : TS][CB], s_sd[CARRY ? 1 : TS][CB];   // sigmoids of z and of delta + bias
    __shared__ __align__(16) W s_b[TS * NL], s_c[TS * NL];
    __shared__ __align__(16) W s_1[CARRY ? 1 : TS][CP], s_2[CARRY ? 1 : TS][CP], s_y[CARRY ? 1 : TS][CP];
    __shared__ __align__(16) W s_bc[CARRY ? 1 : 4 * TS * 2 * NL];
    int slot, block;
    work_of(a, slot, block);
    const int c0 = block * CB;
    const Piece q = find_piece(a.parts, slot);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ql = lane % LPC, cl = wave * (64 / LPC) + lane / LPC;
    const int d = c0 + cl, n0 = ql * NP;
    const long cols = (long)a.D * a.N + 2 * a.D;
    if (q.part >= a.parts.n) {
        if constexpr (!CARRY)
            for (int r = q.begin; r < q.end; ++r) {
                for (int c = c0 + threadIdx.x; c < min(c0 + CB, a.D); c += THREADS) {
                    if (a.du) a.du[(long)r * a.D + c] = T(0);
                    if (a.ddelta) a.ddelta[(long)r * a.D + c] = T(0);
                    if (a.dz) a.dz[(long)r * a.D + c] = T(0);
                }
                for (int n = threadIdx.x; n < a.N && block == 0; n += THREADS) {
                    if (a.dB) a.dB[(long)r * a.N + n] = T(0);
                    if (a.dC) a.dC[(long)r * a.N + n] = T(0);
                }
            }
        return;
    }
    const bool final = q.end >= q.part_end, first = q.j == 0;
    if (CARRY && (q.begin >= q.end || (first && final))) return;
    const int p = a.pol.of(q.part);
    W g[NP], rate[NP], dA[NP];   // g: G of the step behind
#pragma unroll
    for (int i = 0; i < NP; ++i) g[i] = rate[i] = dA[i] = 0;
    if (d < a.D) {
        load_states<NP>(rate, a.A + ((long)p * a.D + d) * a.N, n0, a.N, a.vec_n);
        if constexpr (!CARRY) {
            if (a.carry && !(first && final)) {
                if (q.begin < q.end) load_states<NP>(g, a.carry + ((long)slot * a.D + d) * a.N, n0, a.N, a.vec_n);
            } else if (a.dlast && final && (first || q.begin < q.end)) {
                load_states<NP>(g, a.dlast + ((long)q.part * a.D + d) * a.N, n0, a.N, a.vec_n);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) rate[i] = decay_rate(rate[i]);
    W total = 0;
    const Loader<T, SH> ld(a, c0, p);
    W dD[E], dbias[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dD[e] = dbias[e] = 0;
    Rows<T, E> now, next;
    StepRows<T, SH> bc;
    const int tiles = q.begin < q.end ? (q.end - q.begin + TS - 1) / TS : 0;
    const long check0 = check_slot(q, TS);
    if (tiles > 0) {
        ld.template fetch<true>(next, a, q.begin + (tiles - 1) * TS, q.end);
        bc.template fetch<true>(a, q.begin + (tiles - 1) * TS, q.end);
    }
    for (int tile = tiles - 1; tile >= 0; --tile) {
        const int r0 = q.begin + tile * TS;
        now = next;
        W dt[E];
        if (ld.on) {
            const int live = r0 + ld.t < q.end ? -1 : 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                W slope;
                dt[e] = masked(softplus_w(to_wide((T)now.delta[e]) + ld.bias[e], slope), live);
                s_dt[ld.t][ld.c + e] = Pair<W>{dt[e], dt[e] * to_wide((T)now.u[e])};
                W dy = to_wide((T)now.dy[e]);
                if (a.z) {
                    const W z = to_wide((T)now.z[e]), sz = sigmoid_w(z);
                    dy *= z * sz;
                    if constexpr (!CARRY) s_sz[ld.t][ld.c + e] = sz;
                }
                s_dy[ld.t][ld.c + e] = dy;
                if constexpr (!CARRY) s_sd[ld.t][ld.c + e] = slope;
            }
        }
        bc.template store<true>(s_b, s_c);
        W h[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i) h[i] = 0;
        if constexpr (!CARRY) {
            if (d < a.D) load_states<NP>(h, a.check + ((check0 + tile) * a.D + d) * a.N, n0, a.N, a.vec_n);
        }
        __syncthreads();
        if (tile > 0) {
            ld.template fetch<true>(next, a, r0 - TS, q.end);
            bc.template fetch<true>(a, r0 - TS, q.end);
        }
        if constexpr (CARRY) {
#pragma unroll
            for (int t = TS - 1; t >= 0; --t) {
                const W step = s_dt[t][cl].dt, dy = s_dy[t][cl];
                total += step;
#pragma unroll
                for (int i = 0; i < NP; ++i) g[i] = decay(step, rate[i]) * (s_c[t * NL + n0 + i] * dy + g[i]);
                step_fence<W, NP>();
            }
        } else {
            W av[TS][NP], hv[TS][NP];   // a_t and h_{t-1}
#pragma unroll
            for (int t1 = 0; t1 < TS; t1 += GS) {
                W keep = 0;
#pragma unroll
                for (int t2 = 0; t2 < GS; ++t2) {
                    const int t = t1 + t2;
                    const Pair<W> x = s_dt[t][cl];
                    W y = 0;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        av[t][i] = decay(x.dt, rate[i]);
                        hv[t][i] = h[i];
                        h[i] = av[t][i] * h[i] + x.dtu * s_b[t * NL + n0 + i];
                        y += s_c[t * NL + n0 + i] * h[i];
                    }
                    // (only needed with z, but a branch in every step costs more than the sum: nothing would be scheduled across it)
                    y = sum_states<LPC>(y);
                    keep = ql == t2 ? y : keep;
                    step_fence<W, NP>();
                    if (t2 % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (else every LDS read of the tile is hoisted to its top, into registers that it has not got)
                }
                if (ql < GS) s_y[t1 + ql][cl] = keep;
            }
#pragma unroll
            for (int t1 = TS - GS; t1 >= 0; t1 -= GS) {
                W keep1 = 0, keep2 = 0;
#pragma unroll
                for (int t2 = GS - 1; t2 >= 0; --t2) {
                    const int t = t1 + t2;
                    const Pair<W> x = s_dt[t][cl];
                    const W dy = s_dy[t][cl];
                    W v[NV];
#pragma unroll
                    for (int i = 0; i < NV; ++i) v[i] = 0;
                    W s1 = 0, s2 = 0;
#pragma unroll
                    for (int i = 0; i < NP; ++i) {
                        const W b = s_b[t * NL + n0 + i], cc = s_c[t * NL + n0 + i];
                        v[NP + i] = dy * h[i];
                        const W gt = cc * dy + g[i];
                        v[i] = gt * x.dtu;
                        g[i] = av[t][i] * gt;
                        const W gah = g[i] * hv[t][i];
                        dA[i] += gah * x.dt;
                        s1 += gah * rate[i];
                        s2 += gt * b;
                        h[i] = hv[t][i];
                    }
                    s1 = sum_states<LPC>(s1);
                    s2 = sum_states<LPC>(s2);
                    keep1 = ql == t2 ? s1 : keep1;
                    keep2 = ql == t2 ? s2 : keep2;
                    // over the wave's channels: halves, then quarters of the wave take one value of two each
#pragma unroll
                    for (int i = 0; i < NV / 2; ++i) v[i] = halves32(v[2 * i], v[2 * i + 1]);
#pragma unroll
                    for (int i = 0; i < NV / 4; ++i) {
                        W s = halves16(v[2 * i], v[2 * i + 1]);
                        if constexpr (LPC < 16) s += dpp_move<0x128>(s);   // row_ror:8
                        if constexpr (LPC < 8) s += dpp_move<0x124>(s);    // row_ror:4
                        fixed(s);   // (else the last sum goes into the branch, and its DPP move stays outside by itself)
                        const int row = lane >> 4, k = 2 * (2 * i + (row & 1)) + (row >> 1);
                        if ((lane & 15) < LPC && k < 2 * NP)
                            s_bc[((wave * TS + t) * 2 + k / NP) * NL + n0 + k % NP] = s;
                    }
                    step_fence<W, NP>();
                    if (t2 % 4 == 0) __builtin_amdgcn_sched_barrier(0);
                }
                if (ql < GS) {
                    s_1[t1 + ql][cl] = keep1;
                    s_2[t1 + ql][cl] = keep2;
                }
            }
            __syncthreads();
            const long row = r0 + ld.t;
            if (ld.on && row < q.end && ld.d < a.D) {
                W du[E], dd[E], dz[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const W dy0 = s_dy[ld.t][ld.c + e], s2 = s_2[ld.t][ld.c + e];
                    const W ddt = s_1[ld.t][ld.c + e] * rate_unit(W(0)) + s2 * to_wide((T)now.u[e]);
                    dd[e] = ddt * s_sd[ld.t][ld.c + e];
                    du[e] = dt[e] * s2 + (a.skip ? ld.skip[e] * dy0 : W(0));
                    dbias[e] += dd[e];
                    dD[e] += dy0 * to_wide((T)now.u[e]);
                    dz[e] = 0;
                    if (a.z) {
                        const W y0 = s_y[ld.t][ld.c + e] + (a.skip ? ld.skip[e] * to_wide((T)now.u[e]) : W(0));
                        dz[e] = to_wide((T)now.dy[e]) * y0 * silu_slope_w(to_wide((T)now.z[e]), s_sz[ld.t][ld.c + e]);
                    }
                }
                if (a.du) store_line<E>(a.du + row * a.D, du, ld.d, a.D, a.vec_d);
                if (a.ddelta) store_line<E>(a.ddelta + row * a.D, dd, ld.d, a.D, a.vec_d);
                if (a.dz) store_line<E>(a.dz + row * a.D, dz, ld.d, a.D, a.vec_d);
            }
            if (a.dB || a.dC) {
                for (int k = threadIdx.x; k < TS * 2 * NL; k += THREADS) {
                    const int t = k / (2 * NL), which = k / NL % 2, n = k % NL;
                    const long r = r0 + t;
                    if (r >= q.end || n >= a.N) continue;
                    W s = 0;
#pragma unroll
                    for (int w = 0; w < 4; ++w) s += s_bc[w * TS * 2 * NL + k];
                    if (a.part_bc) a.part_bc[((long)block * a.parts.rows + r) * 2 * a.N + which * a.N + n] = s;
                    else if (which ? a.dC : a.dB) (which ? a.dC : a.dB)[r * a.N + n] = to_elem<T>(s);
                }
            }
        }
        // (what follows here is written for the next tile by the thread that has just read it, or was last read in front of the barrier above)
        if constexpr (CARRY) __syncthreads();
    }
    if constexpr (CARRY) {
        if (d >= a.D) return;
        store_line<NP>(a.carry + ((long)slot * a.D + d) * a.N, g, n0, a.N, a.vec_n);
        if (ql == 0) a.carry_dt[(long)slot * a.D + d] = total;
    } else {
        if (first && a.dstate && d < a.D) store_line<NP>(a.dstate + ((long)q.part * a.D + d) * a.N, g, n0, a.N, a.vec_n);
        if (!a.part) return;
        W* const out = a.part + (long)slot * cols;
        if (d < a.D) {
#pragma unroll
            for (int i = 0; i < NP; ++i)
                if (n0 + i < a.N) out[(long)d * a.N + n0 + i] = dA[i];
        }
        // the loaders' sums: TS threads per channel
        if (ld.on) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s_1[ld.t][ld.c + e] = dD[e];
                s_2[ld.t][ld.c + e] = dbias[e];
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < CB; c += THREADS) {
            if (c0 + c >= a.D) continue;
            W sd = 0, sb = 0;
            for (int t = 0; t < TS; ++t) {
                sd += s_1[t][c];
                sb += s_2[t][c];
            }
            out[(long)a.D * a.N + c0 + c] = sd;
            out[(long)a.D * a.N + a.D + c0 + c] = sb;
        }
    }
}

// dB and dC from the channel blocks' sums (131072 rows of 2 x 16 sums from four blocks: 23 us, 3.2 TB/s)
template <class T> __global__ __launch_bounds__(256) void k_sum_bc(const typename Wide<T>::type* part, long rows, const int* off, int n_seqs, int blocks, int N, T* dB, T* dC) {
    const Parts p{off, n_seqs, (int)rows, 1};
    const long stop = p.at(n_seqs) * 2L * N;
    for (long k = (long)blockIdx.x * 256 + threadIdx.x; k < stop; k += (long)gridDim.x * 256) {
        typename Wide<T>::type s = 0;
        for (int b = 0; b < blocks; ++b) s += part[b * rows * 2 * N + k];
        const long r = k / (2 * N);
        const int m = (int)(k - r * 2 * N);
        if (m < N) { if (dB) dB[r * N + m] = to_elem<T>(s); }
        else if (dC) dC[r * N + m - N] = to_elem<T>(s);
    }
}

// One step of every sequence: states read and written once, 4 lanes per channel with 4 neighbouring states each, 16
// states per turn of the loop, step_seqs() neighbouring sequences a wave, whose loads are in flight together.  `last` may be `state`.
// Bound by the states' bytes: 16384 sequences of 128 x 16 fp32 states take 52 us (5.5 TB/s); one sequence in fp64 takes 4.4 us, a launch's latency.
template <class T, bool ONE> __global__ __launch_bounds__(256) void k_scan_step(const ScanArgs<T> a, int n_seqs, int per_row) {
    typedef typename Wide<T>::type W;
    constexpr int STEP_SEQS = step_seqs<T>();
    const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int s0 = (int)(id / per_row) * STEP_SEQS;
    if (s0 >= n_seqs) return;
    const int lane = threadIdx.x & 63, ql = lane & 3, live = min(STEP_SEQS, n_seqs - s0);
    const int d = (int)(id % per_row) * 16 + lane / 4;
    const bool in = d < a.D;
    const int dd = min(d, a.D - 1);
    long pd[STEP_SEQS];      // the parameters' row
    W u[STEP_SEQS], dt[STEP_SEQS], y[STEP_SEQS];
    T raw_u[STEP_SEQS], raw_dt[STEP_SEQS], raw_z[STEP_SEQS];
#pragma unroll
    for (int i = 0; i < STEP_SEQS; ++i) {
        const long s = s0 + min(i, live - 1);
        pd[i] = (ONE ? 0L : (long)a.pol.of((int)s) * a.D) + dd;
        raw_u[i] = a.u[s * a.ld_u + dd];
        raw_dt[i] = a.delta[s * a.ld_delta + dd];
        raw_z[i] = a.z ? a.z[s * a.ld_z + dd] : T(0);
        y[i] = 0;
    }
    for (int n = ql * 4; n < a.N; n += 16) {
        W h[STEP_SEQS][4], A[4], b[STEP_SEQS][4], c[STEP_SEQS][4];
#pragma unroll
        for (int i = 0; i < STEP_SEQS; ++i) {
            const long s = s0 + min(i, live - 1);
#pragma unroll
            for (int k = 0; k < 4; ++k) h[i][k] = 0;
            if (a.state) load_line<4>(h[i], a.state + s * a.stride_state + (long)dd * a.N, n, a.N, a.vec_n);
            load_line<4>(b[i], a.B + s * a.ld_B, n, a.N, a.vec_bc);
            load_line<4>(c[i], a.C + s * a.ld_C, n, a.N, a.vec_bc);
        }
        if constexpr (ONE) load_line<4>(A, a.A + (long)dd * a.N, n, a.N, a.vec_n);
        if (n < 16) {
#pragma unroll
            for (int i = 0; i < STEP_SEQS; ++i) {
                u[i] = to_wide(raw_u[i]);
                dt[i] = softplus_w(to_wide(raw_dt[i]) + (a.bias ? a.bias[pd[i]] : W(0)));
            }
        }
#pragma unroll
        for (int i = 0; i < STEP_SEQS; ++i) {
            if constexpr (!ONE) load_line<4>(A, a.A + pd[i] * a.N, n, a.N, a.vec_n);
            const W dtu = dt[i] * u[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h[i][k] = decay(dt[i], decay_rate(A[k])) * h[i][k] + dtu * b[i][k];
                y[i] += c[i][k] * h[i][k];
            }
            step_fence<W, 4>();
            if (a.last && in && i < live) store_line<4>(a.last + (s0 + i) * a.stride_last + (long)d * a.N, h[i], n, a.N, a.vec_n);
        }
    }
#pragma unroll
    for (int i = 0; i < STEP_SEQS; ++i) {
        if (i >= live) break;
        W v = sum_states<4>(y[i]);
        if (ql == i % 4 && in) {
            if (a.skip) v += a.skip[pd[i]] * to_wide(raw_u[i]);
            if (a.z) v *= silu_w(to_wide(raw_z[i]));
            a.y[(long)(s0 + i) * a.D + d] = to_elem<T>(v);
        }
    }
}

// ====================================================================================================== host side
int64_t tile_steps(int dtype) { return dtype == PSH_F64 ? 8 : 16; }
// How a call's channels and rows are cut.  A step takes a wave 150 to 400 cycles however few waves there are, and a SIMD needs
// two of them to be busy.  Long sequences that are too few for that are cut into pieces, at the price of a second pass over
// the decays and of two more launches; short ones have their states spread over more lanes instead (more waves with a
// shorter step each, at the price of its fixed work).  Where sequences have more than 192 rows on average the pieces win: one
// of 16384 rows, 256 channels, 16 states, bf16, takes 1536 us spread and 55 us in 256 pieces; 64 of 300 rows, 64 x 16, fp64, 147 and 87 us
// (gradient 265 and 133 us).
// The limit of 512 workgroups, by sequences of 256 rows on average, forward (gradient) in us, in pieces and whole:
//   fp32, 96 x 8, two workgroups a sequence:    64: 30, 60 (69, 130)    192: 64, 64 (155, 136)   255: 80, 65 (205, 139)   257: 78, 65 (202, 138)
//   bf16, 256 x 16, four workgroups a sequence: 64: 67, 65 (134, 134)   100: 96, 65 (214, 141)   127: 113, 65 (251, 170)  129: 112, 65 (246, 163)
//   fp64, 64 x 16, one workgroup (two) a sequence: 128: 118, 248 (201, 255)   256: 216, 250 (403, 279)   480: 396, 264 (735, 392)   513: 436, 267 (820, 440)
// So pieces win to about 256 workgroups there, and between that and the limit calls are up to twice as long as they would be whole; with
// longer sequences the pieces gain (one of 16384 rows, above).  Sequences of 100 rows, which are spread there, take 27 us for 30 (fp32) and 72 us
// for 105 (fp64).
struct ScanPlan {
    int np, lpc, blocks;   // states a lane, lanes a channel, channel blocks
    int64_t piece;         // rows
};
ScanPlan scan_plan(const psh_scan_desc* d, bool grad) {
    const int N = d->states, padded = N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64;
    // the gradient's registers hold a tile's decays and states; in fp64 that is two states a lane
    const int most = grad && d->dtype == PSH_F64 ? 2 : 4;
    const int64_t ts = tile_steps(d->dtype), whole = ((int64_t)d->rows + ts) / ts * ts;
    ScanPlan p;
    const auto with = [&](int lpc) {
        p.lpc = lpc;
        p.np = padded / lpc;
        p.blocks = (d->channels + THREADS / lpc - 1) / (THREADS / lpc);
        return (int64_t)d->n_seqs * p.blocks;
    };
    int least = 4;
    while (least < 16 && padded / least > most) least *= 2;
    const int widest = padded < 16 ? padded : 16;
    p.piece = whole;
    int lpc = least;
    if (with(least) < 512 && d->n_seqs > 0) {
        if (d->rows > 192 * (int64_t)d->n_seqs) {
            p.piece = (int64_t)d->rows * p.blocks / 1024 / ts * ts;
            if (p.piece < 32) p.piece = 32;
            if (p.piece > whole) p.piece = whole;
        } else {
            while (lpc < widest && with(lpc) < 512) lpc *= 2;
        }
    } else if (grad && d->dtype != PSH_F64 && with(least) < 1024 && lpc < widest) {
        // a gradient step has twice the latency for the same bytes: 256 to 511 sequences of 256 rows, 96 x 8, fp32, two workgroups each, take 161 to 272 us on
        // 4 lanes and 138 to 241 us on 8 (512: 270 and 243; 640: 313 and 286); bf16, 256 x 16, four each, 128: 195 and 169, 255: 318 and 314.  Not fp64,
        // which begins on 8 lanes: 64 x 16, two each, 256: 279 us on 8 and 348 on 16, 480: 392 and 599, of 100 rows 167 and 252
        lpc *= 2;
    }
    with(lpc);
    return p;
}
int64_t scan_piece(const psh_scan_desc* d, bool grad) { return scan_plan(d, grad).piece; }
int channel_blocks(const psh_scan_desc* d, bool grad) { return scan_plan(d, grad).blocks; }
// the most there can be, whatever the plan
int64_t most_blocks(const psh_scan_desc* d) { return (d->channels + 15) / 16; }
bool scan_split(const psh_scan_desc* d, bool grad) { return scan_piece(d, grad) < d->rows; }
bool scan_ordered(const psh_scan_desc* d, bool grad) { return !d->step && !scan_split(d, grad) && d->n_seqs > 1 && d->n_seqs <= ORDER_MOST && d->rows > 64 * (int64_t)d->n_seqs; }

// (the order of the launch, if any, lies first)
struct ScanSpace { int64_t order, carry, carry_dt, part, mid, bc, total; };
ScanSpace scan_space(const psh_scan_desc* d, bool grad) {
    ScanSpace s{};
    const int64_t slots = parts_slots(d->rows, d->n_seqs, scan_piece(d, grad)), w = wide_size(d->dtype), D = d->channels, N = d->states;
    if (scan_ordered(d, grad)) s.order = align256((int64_t)d->n_seqs * 4);
    if (scan_split(d, grad)) {
        s.carry = align256(slots * D * N * w);
        s.carry_dt = align256(slots * D * w);
    }
    if (grad) {
        if (d->dA || d->dD || d->ddelta_bias) {
            s.part = align256(slots * (D * N + 2 * D) * w);
            s.mid = align256(join_segs(slots, d->n_policies) * (D * N + 2 * D) * w);
        }
        if ((d->dB || d->dC) && channel_blocks(d, true) > 1) s.bc = align256((int64_t)channel_blocks(d, true) * d->rows * 2 * N * w);
    }
    s.total = s.order + s.carry + s.carry_dt + s.part + s.mid + s.bc;
    return s;
}

bool aligned(const void* p, int64_t bytes, int64_t stride_bytes) { return ((uintptr_t)p % bytes) == 0 && stride_bytes % bytes == 0; }

int bad(psh_ctx* c, const char* what) {
    set_err(c, "%s", what);
    return PSH_ERR_ARG;
}
// limits that keep 32-bit row and slot numbers and grids in range
int too_large(psh_ctx* c, const char* what) {
    set_err(c, "%s: too many rows, sequences or policies for one launch", what);
    return PSH_ERR_UNSUPPORTED;
}

template <class T> ScanArgs<T> scan_args(const psh_scan_desc* d, bool grad) {
    typedef typename Wide<T>::type W;
    ScanArgs<T> a{};
    a.parts = Parts{d->offsets, d->n_seqs, d->rows, (int)scan_piece(d, grad)};
    a.pol = Policies{{d->groups, d->groups ? d->n_policies : 1, d->n_seqs}};
    a.D = d->channels; a.N = d->states;
    a.u = (const T*)d->u; a.delta = (const T*)d->delta; a.z = (const T*)d->z; a.B = (const T*)d->B; a.C = (const T*)d->C;
    a.ld_u = d->ld_u; a.ld_delta = d->ld_delta; a.ld_z = d->ld_z; a.ld_B = d->ld_B; a.ld_C = d->ld_C;
    a.A = (const W*)d->A; a.skip = (const W*)d->D; a.bias = (const W*)d->delta_bias;
    a.state = (const W*)d->state; a.stride_state = d->stride_state;
    a.y = (T*)d->y; a.last = (W*)d->last; a.stride_last = d->stride_last;
    a.check = (W*)d->check;
    a.dy = (const T*)d->dy; a.ld_dy = d->ld_dy; a.dlast = (const W*)d->dlast;
    a.du = (T*)d->du; a.ddelta = (T*)d->ddelta; a.dz = (T*)d->dz; a.dB = (T*)d->dB; a.dC = (T*)d->dC;
    a.dstate = (W*)d->dstate;
    return a;
}
// the widest element runs of a lane: 4 states, and Shape::E channels
template <class T> void scan_alignment(ScanArgs<T>& a, bool grad) {
    const int64_t e = 4 * sizeof(T), n = 4 * sizeof(typename Wide<T>::type), w = sizeof(typename Wide<T>::type);
    a.vec_d = a.D % 4 == 0 && aligned(a.u, e, a.ld_u * sizeof(T)) && aligned(a.delta, e, a.ld_delta * sizeof(T)) &&
              aligned(a.z, e, a.z ? a.ld_z * sizeof(T) : 0);
    a.vec_n = a.N % 4 == 0 && aligned(a.A, n, 0) && aligned(a.state, n, a.state ? a.stride_state * w : 0) &&
              aligned(a.last, n, a.last ? a.stride_last * w : 0) && aligned(a.check, n, 0) && aligned(a.carry, n, 0);
    if (grad) {
        a.vec_d = a.vec_d && aligned(a.dy, e, a.ld_dy * sizeof(T)) && aligned(a.du, e, 0) && aligned(a.ddelta, e, 0) && aligned(a.dz, e, 0);
        a.vec_n = a.vec_n && aligned(a.dlast, n, 0) && aligned(a.dstate, n, 0);
    } else {
        a.vec_d = a.vec_d && aligned(a.y, e, 0);
    }
}

template <class T, int NP, int LPC> int scan_forward(psh_ctx* c, const psh_scan_desc* d, ScanArgs<T>& a) {
    hipStream_t st = (hipStream_t)d->stream;
    const long slots = parts_slots(d->rows, d->n_seqs, a.parts.L);
    a.blocks = channel_blocks(d, false);
    const dim3 grid((unsigned)(slots * a.blocks));
    if (a.order) {
        hipLaunchKernelGGL(k_order, dim3(1), dim3(1024), 0, st, a.parts, const_cast<int*>(a.order));
        PSH_HIP(c, hipGetLastError());
    }
    if (a.carry) {
        hipLaunchKernelGGL((k_scan<T, NP, LPC, true>), grid, dim3(THREADS), 0, st, a);
        PSH_HIP(c, hipGetLastError());
        hipLaunchKernelGGL((k_scan_join<T, false>), dim3(d->n_seqs, (unsigned)(((long)a.D * a.N + JOIN_COLS - 1) / JOIN_COLS)), dim3(256), 0, st, a);
        PSH_HIP(c, hipGetLastError());
    }
    hipLaunchKernelGGL((k_scan<T, NP, LPC, false>), grid, dim3(THREADS), 0, st, a);
    PSH_HIP(c, hipGetLastError());
    return PSH_OK;
}
template <class T, int NP, int LPC> int scan_backward(psh_ctx* c, const psh_scan_desc* d, ScanArgs<T>& a) {
    hipStream_t st = (hipStream_t)d->stream;
    const long slots = parts_slots(d->rows, d->n_seqs, a.parts.L);
    a.blocks = channel_blocks(d, true);
    const dim3 grid((unsigned)(slots * a.blocks));
    if (a.order) {
        hipLaunchKernelGGL(k_order, dim3(1), dim3(1024), 0, st, a.parts, const_cast<int*>(a.order));
        PSH_HIP(c, hipGetLastError());
    }
    if (a.carry) {
        hipLaunchKernelGGL((k_scan_grad<T, NP, LPC, true>), grid, dim3(THREADS), 0, st, a);
        PSH_HIP(c, hipGetLastError());
        hipLaunchKernelGGL((k_scan_join<T, true>), dim3(d->n_seqs, (unsigned)(((long)a.D * a.N + JOIN_COLS - 1) / JOIN_COLS)), dim3(256), 0, st, a);
        PSH_HIP(c, hipGetLastError());
    }
    hipLaunchKernelGGL((k_scan_grad<T, NP, LPC, false>), grid, dim3(THREADS), 0, st, a);
    PSH_HIP(c, hipGetLastError());
    return PSH_OK;
}
// calls f<NP, LPC>() of the plan
#define PSH_SHAPE(plan, f)                                                                                                       \
    ((plan).lpc == 4 ? ((plan).np == 1 ? f(1, 4) : (plan).np == 2 ? f(2, 4) : f(4, 4))                                           \
                     : (plan).lpc == 8 ? ((plan).np == 1 ? f(1, 8) : (plan).np == 2 ? f(2, 8) : f(4, 8))                         \
                                       : ((plan).np == 1 ? f(1, 16) : (plan).np == 2 ? f(2, 16) : f(4, 16)))

template <class T> int run_scan(psh_ctx* c, const psh_scan_desc* d) {
    typedef typename Wide<T>::type W;
    hipStream_t st = (hipStream_t)d->stream;
    ScanArgs<T> a = scan_args<T>(d, false);
    if (d->step) {
        a.check = nullptr;
        scan_alignment(a, false);
        const int per_row = (a.D + 15) / 16;
        const int64_t e = 4 * sizeof(T);
        a.vec_bc = a.N % 4 == 0 && aligned(a.B, e, a.ld_B * sizeof(T)) && aligned(a.C, e, a.ld_C * sizeof(T));
        const long blocks = (((long)d->n_seqs + step_seqs<T>() - 1) / step_seqs<T>() * per_row + 3) / 4;
        if (blocks > 0x7fffffffL) return too_large(c, "selective_scan");
        if (a.pol.n == 1) hipLaunchKernelGGL((k_scan_step<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, a, (int)d->n_seqs, per_row);
        else hipLaunchKernelGGL((k_scan_step<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, a, (int)d->n_seqs, per_row);
        PSH_HIP(c, hipGetLastError());
        return PSH_OK;
    }
    const ScanSpace s = scan_space(d, false);
    unsigned char* const at = (unsigned char*)d->workspace + s.order;
    if (s.order) a.order = (const int*)d->workspace;
    if (s.carry) {
        a.carry = (W*)at;
        a.carry_dt = (W*)(at + s.carry);
    }
    scan_alignment(a, false);
#define PSH_CALL(NP, LPC) scan_forward<T, NP, LPC>(c, d, a)
    const ScanPlan plan = scan_plan(d, false);
    return PSH_SHAPE(plan, PSH_CALL);
#undef PSH_CALL
}
template <class T> int run_scan_grad(psh_ctx* c, const psh_scan_desc* d) {
    typedef typename Wide<T>::type W;
    hipStream_t st = (hipStream_t)d->stream;
    ScanArgs<T> a = scan_args<T>(d, true);
    const ScanSpace s = scan_space(d, true);
    unsigned char* at = (unsigned char*)d->workspace + s.order;
    if (s.order) a.order = (const int*)d->workspace;
    if (s.carry) {
        a.carry = (W*)at;
        a.carry_dt = (W*)(at + s.carry);
    }
    at += s.carry + s.carry_dt;
    if (s.part) a.part = (W*)at;
    at += s.part;
    W* const mid = (W*)at;
    at += s.mid;
    if (s.bc) a.part_bc = (W*)at;
    scan_alignment(a, true);
#define PSH_CALL(NP, LPC) scan_backward<T, NP, LPC>(c, d, a)
    const ScanPlan plan = scan_plan(d, true);
    const int rc = PSH_SHAPE(plan, PSH_CALL);
#undef PSH_CALL
    if (rc != PSH_OK) return rc;
    if (a.part_bc && d->rows > 0) {
        const long n = ((long)d->rows * 2 * a.N + 255) / 256;
        hipLaunchKernelGGL(k_sum_bc<T>, dim3((unsigned)(n < 4096 ? n : 4096)), dim3(256), 0, st, (const W*)a.part_bc, (long)d->rows,
                           d->offsets, (int)d->n_seqs, a.blocks, (int)a.N, a.dB, a.dC);
        PSH_HIP(c, hipGetLastError());
        // rows behind the last sequence: the grad kernel's first channel block has written their zeros
    }
    if (a.part) {
        JoinArgs<W> j{};
        j.parts = a.parts; j.pol = a.pol;
        j.part = a.part; j.mid = mid;
        j.out0 = (W*)d->dA; j.out1 = (W*)d->dD; j.out2 = (W*)d->ddelta_bias;
        j.n0 = (long)a.D * a.N; j.n1 = j.n2 = a.D;
        return run_join(c, j, parts_slots(d->rows, d->n_seqs, a.parts.L), st);
    }
    return PSH_OK;
}

int check_scan(psh_ctx* c, const psh_scan_desc* d, bool grad) {
    if (!c || !d) return PSH_ERR_ARG;
    if (d->dtype < PSH_F64 || d->dtype > PSH_BF16) return bad(c, "selective_scan: unknown dtype");
    if (d->n_policies < 1 || d->n_seqs < 0 || d->rows < 0 || d->channels < 1 || d->states < 1 || d->states > PSH_MAX_MEM_STATES)
        return bad(c, "selective_scan: invalid sizes (1..PSH_MAX_MEM_STATES states)");
    if (d->rows > (1 << 30) || d->n_seqs > (1 << 30) || (d->rows / 64 + (int64_t)d->n_seqs + 2) * most_blocks(d) > 0x7fffffffLL || ((int64_t)d->channels * d->states + 2 * (int64_t)d->channels + 31) / 32 > 65535)
        return too_large(c, "selective_scan");
    if (d->n_policies > 1 && !d->groups) return bad(c, "selective_scan: several policies need groups");
    if (d->step ? d->rows != d->n_seqs : !d->offsets) return bad(c, "selective_scan: offsets are NULL, or a step call has not one row per sequence");
    if (!d->A || (d->rows > 0 && (!d->u || !d->delta || !d->B || !d->C))) return bad(c, "selective_scan: NULL array");
    if (d->ld_u < d->channels || d->ld_delta < d->channels || (d->z && d->ld_z < d->channels) || d->ld_B < d->states || d->ld_C < d->states)
        return bad(c, "selective_scan: a row stride is below the row's length");
    const int64_t DN = (int64_t)d->channels * d->states;
    if ((d->state && d->stride_state < DN) || (d->last && d->stride_last < DN)) return bad(c, "selective_scan: a state's stride is below its size");
    if (grad) {
        if (d->step) return bad(c, "selective_scan_grad: single steps have no gradient call");
        if (d->rows > 0 && (!d->dy || d->ld_dy < d->channels || !d->check)) return bad(c, "selective_scan_grad: dy or check is NULL, or dy's stride is below its length");
    } else if (d->rows > 0 && !d->y) {
        return bad(c, "selective_scan: y is NULL");
    }
    if (!d->step) {
        const ScanSpace s = scan_space(d, grad);
        if (s.total > 0 && (!d->workspace || d->workspace_bytes < s.total || ((uintptr_t)d->workspace & 255)))
            return bad(c, "selective_scan: the workspace is too small or not 256-byte aligned");
    }
    return PSH_OK;
}

// ---- convolution
int lanes_for(int D, int V) {
    int n = 1;
    while (n < 64 && n * V < D) n *= 2;
    return n;
}
// channels of a lane: 16 bytes, for bf16 gradients 8 (8 channels' windows, sums and weights take 174 registers, 4 channels' 98)
constexpr int conv_wide(int elem, bool grad) { return grad && elem == 2 ? 4 : 16 / elem; }
int conv_vec(const psh_conv_desc* d, bool grad) {
    const int e = elem_size(d->dtype), V = conv_wide(e, grad);
    const bool ok = d->channels % V == 0 && aligned(d->x, V * e, d->ld_x * e) &&
                    (grad ? aligned(d->dy, V * e, d->ld_dy * e) && aligned(d->dx, V * e, 0) : aligned(d->y, V * e, 0));
    return ok ? V : 1;
}
// Rows of a run: a run reads K - 1 rows (the gradient computes as many) that the next one reads again, so they are as long as leaves
// two waves a SIMD.  One episode of 16384 steps, 256 channels, bf16: 14 us in runs of 16, 11 us in runs of 4.
int conv_run(const psh_conv_desc* d, int V, bool grad) {
    const int lanes = lanes_for(d->channels, V);
    const int64_t across = (d->channels + lanes * V - 1) / (lanes * V);
    int run = grad ? 32 : 16;
    while (run > 4 && (int64_t)d->rows * lanes / (64 * run) * across < 2048) run /= 2;
    return run;
}
int64_t conv_piece(const psh_conv_desc* d, int V, bool grad) {
    return (int64_t)conv_run(d, V, grad) * (64 / lanes_for(d->channels, V));
}
struct ConvSpace { int64_t part, mid, total; };
ConvSpace conv_space(const psh_conv_desc* d) {
    ConvSpace s{};
    if (d->dweight || d->dbias) {
        // the wide and the one-element lane layouts cut pieces of different lengths: room for either
        for (int k = 0; k < 2; ++k) {
            const int64_t slots = parts_slots(d->rows, d->n_seqs, conv_piece(d, k ? 1 : conv_wide(elem_size(d->dtype), true), true));
            const int64_t cols = (int64_t)d->channels * (d->taps + 1) * wide_size(d->dtype);
            const int64_t part = align256(slots * cols), mid = align256(join_segs(slots, d->n_policies) * cols);
            if (part > s.part) s.part = part;
            if (mid > s.mid) s.mid = mid;
        }
    }
    s.total = s.part + s.mid;
    return s;
}

template <class T, int K> int run_conv(psh_ctx* c, const psh_conv_desc* d, bool grad) {
    typedef typename Wide<T>::type W;
    constexpr int VW = conv_wide(sizeof(T), false), VG = conv_wide(sizeof(T), true);
    hipStream_t st = (hipStream_t)d->stream;
    ConvArgs<T> a{};
    a.pol = Policies{{d->groups, d->groups ? d->n_policies : 1, d->n_seqs}};
    a.x = (const T*)d->x; a.ld_x = d->ld_x;
    a.w = (const W*)d->weight; a.b = (const W*)d->bias;
    a.state = K > 1 ? (const T*)d->state : nullptr; a.stride_state = d->stride_state;
    a.y = (T*)d->y;
    a.last = K > 1 ? (T*)d->last : nullptr; a.stride_last = d->stride_last;
    a.D = d->channels; a.silu = d->silu;
    if (d->step) {
        const int per_row = (a.D + 63) / 64;
        const long blocks = (((long)d->n_seqs + step_seqs<T>() - 1) / step_seqs<T>() * per_row + 3) / 4;
        if (blocks > 0x7fffffffL) return too_large(c, "causal_conv");
        if (a.pol.n == 1) hipLaunchKernelGGL((k_conv_step<T, K, true>), dim3((unsigned)blocks), dim3(256), 0, st, a, (int)d->n_seqs, per_row);
        else hipLaunchKernelGGL((k_conv_step<T, K, false>), dim3((unsigned)blocks), dim3(256), 0, st, a, (int)d->n_seqs, per_row);
        PSH_HIP(c, hipGetLastError());
        return PSH_OK;
    }
    const int V = conv_vec(d, grad);
    a.vec = V > 1;
    a.lanes_c = lanes_for(a.D, V);
    a.run = conv_run(d, V, grad);
    a.parts = Parts{d->offsets, d->n_seqs, d->rows, (int)conv_piece(d, V, grad)};
    const long slots = parts_slots(d->rows, d->n_seqs, a.parts.L);
    const int by = (a.D + a.lanes_c * V - 1) / (a.lanes_c * V);
    const dim3 grid((unsigned)((slots + 3) / 4), (unsigned)by);
    if (!grad) {
        if (V > 1) hipLaunchKernelGGL((k_conv<T, VW, K>), grid, dim3(256), 0, st, a, slots);
        else hipLaunchKernelGGL((k_conv<T, 1, K>), grid, dim3(256), 0, st, a, slots);
        PSH_HIP(c, hipGetLastError());
        return PSH_OK;
    }
    a.dy = (const T*)d->dy; a.ld_dy = d->ld_dy;
    a.dlast = K > 1 ? (const T*)d->dlast : nullptr;
    a.dx = (T*)d->dx; a.dstate = K > 1 ? (T*)d->dstate : nullptr;
    const ConvSpace s = conv_space(d);
    if (s.part) a.part = (W*)d->workspace;
    if (V > 1) hipLaunchKernelGGL((k_conv_grad<T, VG, K>), grid, dim3(256), 0, st, a, slots);
    else hipLaunchKernelGGL((k_conv_grad<T, 1, K>), grid, dim3(256), 0, st, a, slots);
    PSH_HIP(c, hipGetLastError());
    if (a.part) {
        JoinArgs<W> j{};
        j.parts = a.parts; j.pol = a.pol;
        j.part = a.part; j.mid = (W*)((unsigned char*)d->workspace + s.part);
        j.out0 = (W*)d->dweight; j.out1 = (W*)d->dbias;
        j.n0 = (long)a.D * (K + 1); j.split = K;
        return run_join(c, j, slots, st);
    }
    return PSH_OK;
}
template <class T> int conv_taps(psh_ctx* c, const psh_conv_desc* d, bool grad) {
    switch (d->taps) {
        case 1: return run_conv<T, 1>(c, d, grad);
        case 2: return run_conv<T, 2>(c, d, grad);
        case 3: return run_conv<T, 3>(c, d, grad);
        case 4: return run_conv<T, 4>(c, d, grad);
        case 5: return run_conv<T, 5>(c, d, grad);
        case 6: return run_conv<T, 6>(c, d, grad);
        case 7: return run_conv<T, 7>(c, d, grad);
        default: return run_conv<T, 8>(c, d, grad);
    }
}
int check_conv(psh_ctx* c, const psh_conv_desc* d, bool grad) {
    if (!c || !d) return PSH_ERR_ARG;
    if (d->dtype < PSH_F64 || d->dtype > PSH_BF16) return bad(c, "causal_conv: unknown dtype");
    if (d->n_policies < 1 || d->n_seqs < 0 || d->rows < 0 || d->channels < 1 || d->taps < 1 || d->taps > PSH_MAX_TAPS)
        return bad(c, "causal_conv: invalid sizes (1..PSH_MAX_TAPS taps)");
    if (d->rows > (1 << 30) || d->n_seqs > (1 << 30) || ((int64_t)d->channels * (d->taps + 1) + 255) / 256 > 65535) return too_large(c, "causal_conv");
    if (d->n_policies > 1 && !d->groups) return bad(c, "causal_conv: several policies need groups");
    if (d->step ? d->rows != d->n_seqs : !d->offsets) return bad(c, "causal_conv: offsets are NULL, or a step call has not one row per sequence");
    if (!d->weight || (d->rows > 0 && !d->x) || d->ld_x < d->channels) return bad(c, "causal_conv: NULL array or a row stride below the row's length");
    const int64_t DK = (int64_t)d->channels * (d->taps - 1);
    if ((d->state && d->stride_state < DK) || (d->last && d->stride_last < DK)) return bad(c, "causal_conv: a state's stride is below its size");
    if (grad) {
        if (d->step) return bad(c, "causal_conv_grad: single steps have no gradient call");
        if (d->rows > 0 && (!d->dy || d->ld_dy < d->channels)) return bad(c, "causal_conv_grad: dy is NULL or its stride is below its length");
        const ConvSpace s = conv_space(d);
        if (s.total > 0 && (!d->workspace || d->workspace_bytes < s.total || ((uintptr_t)d->workspace & 255)))
            return bad(c, "causal_conv_grad: the workspace is too small or not 256-byte aligned");
    } else if (d->rows > 0 && !d->y) {
        return bad(c, "causal_conv: y is NULL");
    }
    return PSH_OK;
}
bool valid_sizes(const psh_scan_desc* d) {
    return d && d->n_policies >= 1 && d->n_seqs >= 0 && d->rows >= 0 && d->channels >= 1 && d->states >= 1 && d->states <= PSH_MAX_MEM_STATES;
}

}  // namespace

extern "C" int64_t psh_causal_conv_grad_workspace(const psh_conv_desc* d) {
    if (!d || d->n_policies < 1 || d->n_seqs < 0 || d->rows < 0 || d->channels < 1 || d->taps < 1 || d->taps > PSH_MAX_TAPS) return PSH_ERR_ARG;
    return conv_space(d).total;
}
extern "C" int psh_causal_conv(psh_ctx* c, const psh_conv_desc* d) {
    const int rc = check_conv(c, d, false);
    if (rc != PSH_OK || (d->rows == 0 && d->n_seqs == 0)) return rc;
    PSH_ON_DEVICE(c);
    return d->dtype == PSH_F64 ? conv_taps<double>(c, d, false) : d->dtype == PSH_F32 ? conv_taps<float>(c, d, false) : conv_taps<bf16_t>(c, d, false);
}
extern "C" int psh_causal_conv_grad(psh_ctx* c, const psh_conv_desc* d) {
    const int rc = check_conv(c, d, true);
    if (rc != PSH_OK) return rc;
    PSH_ON_DEVICE(c);
    return d->dtype == PSH_F64 ? conv_taps<double>(c, d, true) : d->dtype == PSH_F32 ? conv_taps<float>(c, d, true) : conv_taps<bf16_t>(c, d, true);
}

extern "C" int64_t psh_selective_scan_check(const psh_scan_desc* d) {
    if (!valid_sizes(d)) return PSH_ERR_ARG;
    return parts_slots(d->rows, d->n_seqs, tile_steps(d->dtype)) * (int64_t)d->channels * d->states * wide_size(d->dtype);
}
extern "C" int64_t psh_selective_scan_workspace(const psh_scan_desc* d) { return valid_sizes(d) ? (d->step ? 0 : scan_space(d, false).total) : PSH_ERR_ARG; }
extern "C" int64_t psh_selective_scan_grad_workspace(const psh_scan_desc* d) { return valid_sizes(d) ? scan_space(d, true).total : PSH_ERR_ARG; }
extern "C" int psh_selective_scan(psh_ctx* c, const psh_scan_desc* d) {
    const int rc = check_scan(c, d, false);
    if (rc != PSH_OK || (d->rows == 0 && d->n_seqs == 0)) return rc;
    PSH_ON_DEVICE(c);
    return d->dtype == PSH_F64 ? run_scan<double>(c, d) : d->dtype == PSH_F32 ? run_scan<float>(c, d) : run_scan<bf16_t>(c, d);
}
extern "C" int psh_selective_scan_grad(psh_ctx* c, const psh_scan_desc* d) {
    const int rc = check_scan(c, d, true);
    if (rc != PSH_OK) return rc;
    PSH_ON_DEVICE(c);
    return d->dtype == PSH_F64 ? run_scan_grad<double>(c, d) : d->dtype == PSH_F32 ? run_scan_grad<float>(c, d) : run_scan_grad<bf16_t>(c, d);
}
