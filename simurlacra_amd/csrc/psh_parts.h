// How the policy operators cut rows into parts and pieces: which rows, which entries of the stored states and which
// partial sums a workgroup works on.  Plain arithmetic on what the offsets hold, for the device, and for the CPU, where it is
// tested with offsets of any kind.
#pragma once

#include <cstdint>

#include "../../include/pysimhip.h"

#define PSH_BOTH __host__ __device__ __forceinline__

// Rows are cut into n parts by offsets (device memory, so the host cannot count tiles) and a launch works in pieces of L
// rows.  Piece j of part i gets the slot  floor(off[i] / L) + i + j.  Two parts never share a slot: with off[i] = a L + r
// and off[i+1] = b L + r', part i has ceil((b - a) + (r' - r) / L) <= b - a + 1 pieces, exactly the distance of the two
// parts' first slots.  So slots are found without a prefix sum or a second launch, there are at most rows / L + n + 1 of
// them, and every part owns at least one, empty parts too.  Part n stands for the rows behind the last offset.
struct Parts {
    const int* off;
    int n, rows, L;
    PSH_BOTH int at(int i) const {
        if (i <= 0) return 0;
        if (i > n) return rows;
        const int o = off[i];
        return o < 0 ? 0 : (o > rows ? rows : o);
    }
    PSH_BOTH int first_slot(int i) const { return at(i) / L + i; }
};
PSH_BOTH int64_t parts_slots(int64_t rows, int64_t n, int64_t L) { return rows / L + n + 1; }
// pieces of a part of these rows that has more than L of them
PSH_BOTH int piece_count(int begin, int end, int L) { return (int)(((int64_t)end - begin + L - 1) / L); }

struct Piece {
    int part, j;      // piece j of the part
    int begin, end;   // its rows (begin >= end: none)
    int part_begin, part_end;
};
PSH_BOTH Piece piece_of(const Parts& p, int part, int part_begin, int part_end, int slot) {
    Piece q;
    q.part = part;
    q.part_begin = part_begin;
    q.part_end = part_end;
    q.j = slot - (part_begin / p.L + part);
    const int64_t b = (int64_t)part_begin + (int64_t)q.j * p.L, e = b + p.L;
    q.begin = (int)(b < p.rows ? b : p.rows);
    q.end = (int)(e < part_end ? e : part_end);
    return q;
}
// Room for partial results of the parts of more than L rows, which are cut; the others have none.  Piece j of a part from row b has the
// place floor(2 b / L) + j: a part of x L rows has ceil(x) pieces, no more than floor(2 x) for x > 1, and the next part's places begin
// at least floor(2 x) further on.  These are at most 2 rows / L + 1 places however many parts there are; with few parts there are
// fewer slots than that, and a piece's place is its slot.
struct CutPlaces {
    bool by_rows;
    PSH_BOTH int64_t first(const Parts& p, int part, int part_begin) const { return by_rows ? 2 * (int64_t)part_begin / p.L : part_begin / p.L + part; }
};
PSH_BOTH int64_t places_by_rows(int64_t rows, int64_t L) { return 2 * rows / L + 1; }
PSH_BOTH CutPlaces cut_places(int64_t rows, int64_t n, int64_t L) { return CutPlaces{places_by_rows(rows, L) < parts_slots(rows, n, L)}; }
PSH_BOTH int64_t cut_places_count(int64_t rows, int64_t n, int64_t L) {
    return cut_places(rows, n, L).by_rows ? places_by_rows(rows, L) : parts_slots(rows, n, L);
}
// where the states stored before every tile of TS steps of a piece begin (TS divides L)
PSH_BOTH int64_t check_slot(const Piece& q, int TS) { return (int64_t)q.part_begin / TS + q.part + (q.begin - q.part_begin) / TS; }

// The largest i in [0, n] with key(i) <= slot, for ascending keys with key(0) <= slot: 64 lanes probe one candidate each, so 4096
// parts take two rounds of loads where a binary search takes twelve.  One round: lane l probes candidate(l) if probes(l), and
// `below` has the bits of those whose key is not above the slot.
struct Search {
    int lo, count;
    PSH_BOTH int step() const { return (count + 63) / 64; }
    PSH_BOTH bool probes(int lane) const { return lane * step() < count; }
    PSH_BOTH int candidate(int lane) const { return lo + lane * step(); }
    PSH_BOTH void narrow(uint64_t below) {
        const int s = step(), next = lo + (63 - __builtin_clzll(below | 1)) * s;   // (lane 0 probes lo itself: key(lo) <= slot)
        const int left = lo + count - next;
        count = s < left ? s : left;
        lo = next;
    }
};

// which policy's parameters a sequence uses: the part of the sequences it lies in (the last part ends with the last
// sequence, whatever groups[P] says)
struct Shares {
    const int* groups;
    int n, n_seqs;
    PSH_BOTH int at(int p) const {
        if (p <= 0) return 0;
        if (p >= n) return n_seqs;
        const int o = groups[p];
        return o < 0 ? 0 : (o > n_seqs ? n_seqs : o);
    }
};

// Sums over the slots of a policy's sequences, in segments of `seg` slots: segment k of policy p is number slot_of(p) / seg + p + k, by
// the reasoning of Parts.
struct PolicySlots {
    Parts parts;
    Shares pol;
    int seg;
    PSH_BOTH int slot_of(int p) const { return p >= pol.n ? parts.first_slot(parts.n) : parts.first_slot(pol.at(p)); }
    PSH_BOTH int seg_of(int p) const { return slot_of(p) / seg + p; }
    // the slots of segment number k, which is one of policy p's; whether there are any, or it is the policy's first
    PSH_BOTH bool segment(int k, int p, int64_t& begin, int64_t& stop) const {
        const int first = slot_of(p), end = slot_of(p + 1), own = seg_of(p);
        begin = (int64_t)first + (int64_t)(k - own) * seg;
        stop = begin + seg < end ? begin + seg : end;
        return begin < end || k == own;
    }
    // the policy's segments (seg > 0) or slots (seg = 0)
    PSH_BOTH void of_policy(int p, int& first, int& n) const {
        const int a = slot_of(p), slots = slot_of(p + 1) - a;
        first = seg ? seg_of(p) : a;
        n = slots <= 0 ? 0 : seg ? (slots + seg - 1) / seg : slots;
    }
};
PSH_BOTH int64_t policy_segments(int64_t slots, int policies, int seg) { return slots / seg + policies + 1; }

static inline int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }
static inline int elem_size(int dtype) { return dtype == PSH_F64 ? 8 : dtype == PSH_F32 ? 4 : 2; }
static inline int wide_size(int dtype) { return dtype == PSH_F64 ? 8 : 4; }
