// ecu_draft.h -- the lists of sequences of a step with drafted tokens, shared by
// the translation units that launch its kernels.
#pragma once
#include "ecu_kv4.cuh"
#include "ecu_kv4.h"

inline int number_of(int first, const int *seq, int i) { return seq ? seq[i] : first + i; }

// What append_rope and attend_tree ask of their lists: slots that exist, none
// twice, at most `most` new rows of each and no more than it holds.  The rows
// in all, or -1.
inline long long rows_ok(const ecu_kv *kv, const int *seq, const int *n_new, int n, int most, const char *what)
{
    if (slots_ok(kv, seq, n, what) != 0) return -1;
    long long         rows = 0;
    std::vector<bool> seen((size_t)kv->book.n_seq, false);
    for (int i = 0; i < n; i++) {
        const int s = number_of(0, seq, i);
        if (seen[s]) {
            ecu_set_error(nullptr, 0, "%s: sequence %d comes twice", what, s);
            return -1;
        }
        seen[s] = true;
        if (n_new[i] < 0 || n_new[i] > kv->book.seq[s].len || n_new[i] > most) {
            ecu_set_error(nullptr, 0, "%s: %d rows for sequence %d of %d positions%s", what, n_new[i], s, kv->book.seq[s].len,
                          n_new[i] > most ? " (64 drafted rows at most)" : "");
            return -1;
        }
        rows += n_new[i];
    }
    return rows;
}

template <int N> void fill_rows(KvRows<N> &r, const int *seq, int first, const int *n_new, int n)
{
    r.n = n;
    r.row0[0] = 0;
    for (int i = 0; i < n; i++) {
        r.seq[i] = (uint16_t)number_of(first, seq, i);
        r.row0[i + 1] = r.row0[i] + n_new[i];
    }
}
