// spt_kv_seq.h -- a sequence's rows and positions, from what the batch's
// arrays say.  Plain C++, so that it is checked on the host too.
#pragma once

namespace spt {

// A sequence of the batch: its rows [r0, r0 + n) (cut to the buffers'), the
// position of the first, and the position behind the last (first may be below
// 0, and no position >= end is any row's); ok: within the batch's declared
// bounds (else n is cut to them).
struct KvSeq {
    int r0, n, first, end;
    bool ok;
};

// lo, hi, len: any ints.  n_rows >= 0; max_len, max_new >= 1.
constexpr KvSeq kv_seq_of(int lo, int hi, int len, int n_rows, int max_len, int max_new) {
    // both ends into the buffers before their difference: hi - lo of any two
    // ints passes 32 bits
    const int r0 = lo < 0 ? 0 : lo < n_rows ? lo : n_rows;
    const int r1 = hi < r0 ? r0 : hi < n_rows ? hi : n_rows;
    KvSeq q{r0, r1 - r0, 0, 0, false};
    const int positions = len < 0 ? 0 : len;
    q.ok = positions <= max_len && (long long)hi - lo <= max_new;
    if (!q.ok) {
        q.n = q.n < max_new ? q.n : max_new;
    } else if (q.n > 0) {
        // row hi - 1 is the last position, in the buffers or not: row r is
        // len - (hi - r) (lo <= r < hi <= lo + max_new: no overflow)
        q.first = positions - (hi - r0);
        q.end = q.first + q.n;
    }
    return q;
}

}  // namespace spt
