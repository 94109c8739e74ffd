// spt_kv_seq.h -- a sequence's rows and positions, from what the batch's
// arrays say.  Plain C++, so that it is checked on the host too.
#pragma once

namespace spt {

// A sequence of the batch: its rows [r0, r0 + n) (cut to the buffers') and
// the position of the first; ok: within the batch's declared bounds (else n
// is cut to them).
struct KvSeq {
    int r0, n, len, first;
    bool ok;
};

// lo, hi, len: any ints.  n_rows >= 0; max_len, max_new >= 1.
constexpr KvSeq kv_seq_of(int lo, int hi, int len, int n_rows, int max_len, int max_new) {
    // both ends into the buffers before their difference: hi - lo of any two
    // ints passes 32 bits
    const int r0 = lo < 0 ? 0 : lo < n_rows ? lo : n_rows;
    const int r1 = hi < r0 ? r0 : hi < n_rows ? hi : n_rows;
    KvSeq q{r0, r1 - r0, len < 0 ? 0 : len, 0, false};
    q.first = q.len - q.n;
    q.ok = q.len <= max_len && q.n <= max_new;
    if (!q.ok) {
        q.n = q.n < max_new ? q.n : max_new;
        q.first = 0;
    }
    return q;
}

}  // namespace spt
