// ecu_kvbook.cpp -- the page pool's bookkeeping (host only).
//
// Free pages are a bitmap and taken lowest id first, so that the same calls
// always give the same tables and the pool stays packed towards its start.
// An operation logs what it changes and is undone from the log when a later
// part of it cannot be done, here or on the device.  Memory for a step and its
// log is taken before the step, so that one that runs out leaves a log that
// matches what was done.
#include "ecu_kv4.h"
#include "ecu_model.h"

#include <algorithm>

static int pages_of(long long n) { return (int)((n + ECU_KV4_PAGE - 1) / ECU_KV4_PAGE); }

enum { U_HOLD, U_DROP, U_PUSH, U_POP, U_CELL, U_LEN };

template <typename T> static void room(std::vector<T> &v, size_t n)
{
    if (v.capacity() - v.size() < n) v.reserve(std::max(2 * v.capacity(), v.size() + n));
}

void KvBook::init(int pages, int seqs, int per_seq)
{
    n_pages = pages;
    n_seq = seqs;
    max_pages = per_seq;
    seq.assign((size_t)seqs, Seq());
    ref.assign((size_t)pages, 0);
    taken.assign(((size_t)pages + 63) / 64, 0);
}

void KvBook::hold(int p)
{
    if (ref[p]++ == 0) {
        taken[p >> 6] |= 1ull << (p & 63);
        used++;
    }
}

void KvBook::drop(int p)
{
    if (--ref[p] == 0) {
        taken[p >> 6] &= ~(1ull << (p & 63));
        hint = std::min(hint, (size_t)p >> 6);
        used--;
    }
}

// The lowest free page, held once; -1: none.
int KvBook::take()
{
    for (; hint < taken.size(); hint++)
        if (~taken[hint]) {
            const int p = (int)(hint * 64) + __builtin_ctzll(~taken[hint]);
            if (p >= n_pages) return -1;
            room(log_, 1);
            hold(p);
            log_.push_back({U_HOLD, p, 0});
            return p;
        }
    return -1;
}

void KvBook::begin()
{
    log_.clear();
    cell_.clear();
    length_.clear();
    copies.clear();
    sets.clear();
    compacted_ = false;
}

// Pages `from` become pages `to` in every table.
void KvBook::move_pages(bool back)
{
    std::vector<int> &to = move_;
    for (const Copy &c : copies) to[back ? c.to : c.from] = back ? c.from : c.to;
    for (Seq &q : seq)
        for (int &p : q.page)
            if (to[p] >= 0) p = to[p];
    for (const Copy &c : copies) to[back ? c.to : c.from] = -1;
    for (const Copy &c : copies) std::swap(ref[c.to], ref[c.from]);
    std::fill(taken.begin(), taken.end(), 0ull);
    for (int p = 0; p < n_pages; p++)
        if (ref[p]) taken[p >> 6] |= 1ull << (p & 63);
    hint = back ? 0 : (size_t)used >> 6;
}

int KvBook::fail()
{
    if (compacted_) move_pages(true);
    for (size_t i = log_.size(); i-- > 0;) {
        const Undo u = log_[i];
        switch (u.kind) {
        case U_HOLD: drop(u.a); break;
        case U_DROP: hold(u.a); break;
        case U_PUSH: seq[u.a].page.pop_back(); break;
        case U_POP:  seq[u.a].page.push_back(u.b); break;
        case U_CELL: seq[u.a].page.back() = u.b; break;
        case U_LEN:  seq[u.a].len = u.b; break;
        }
    }
    begin();
    return -1;
}

// The device words that the operation changed, each once, with their last values.
void KvBook::finish()
{
    std::sort(cell_.begin(), cell_.end());
    cell_.erase(std::unique(cell_.begin(), cell_.end()), cell_.end());
    std::sort(length_.begin(), length_.end());
    length_.erase(std::unique(length_.begin(), length_.end()), length_.end());
    for (auto &c : cell_) {
        const Seq &q = seq[c.first];
        sets.push_back({c.first * max_pages + c.second, c.second < (int)q.page.size() ? q.page[c.second] : -1});
    }
    for (int s : length_) sets.push_back({n_seq * max_pages + s, seq[s].len});
}

bool KvBook::slot(int s, const char *what)
{
    if (s >= 0 && s < n_seq) return true;
    ecu_set_error(nullptr, 0, "%s: no sequence %d (%d slots)", what, s, n_seq);
    return false;
}

int KvBook::extend(const int *s, const int *n_new, int n)
{
    begin();
    for (int i = 0; i < n; i++) {
        if (!slot(s[i], "ecu_kv_extend")) return fail();
        Seq &q = seq[s[i]];
        const long long want = (long long)q.len + n_new[i];
        if (n_new[i] < 0 || want > (long long)max_pages * ECU_KV4_PAGE) {
            ecu_set_error(nullptr, 0, "ecu_kv_extend: sequence %d cannot grow by %d (%d of %lld positions)", s[i], n_new[i],
                          q.len, (long long)max_pages * ECU_KV4_PAGE);
            return fail();
        }
        if (n_new[i] == 0) continue;
        auto none = [&] {
            ecu_set_error(nullptr, 0, "ecu_kv_extend: no free page for sequence %d (all %d in use or taken by this call)",
                          s[i], n_pages);
            return fail();
        };
        // a partly filled last page that others hold too: a copy of its own
        if (q.len % ECU_KV4_PAGE && ref[q.page.back()] > 1) {
            const int old = q.page.back(), p = take();
            if (p < 0) return none();
            copies.push_back({old, p});
            cell_.push_back({s[i], (int)q.page.size() - 1});
            room(log_, 2);
            drop(old);
            log_.push_back({U_DROP, old, 0});
            log_.push_back({U_CELL, s[i], old});
            q.page.back() = p;
        }
        while ((int)q.page.size() < pages_of(want)) {
            const int p = take();
            if (p < 0) return none();
            cell_.push_back({s[i], (int)q.page.size()});
            room(q.page, 1);
            room(log_, 1);
            q.page.push_back(p);
            log_.push_back({U_PUSH, s[i], 0});
        }
        length_.push_back(s[i]);
        room(log_, 1);
        log_.push_back({U_LEN, s[i], q.len});
        q.len = (int)want;
    }
    finish();
    return 0;
}

int KvBook::fork(const int *src, const int *dst, int n)
{
    begin();
    for (int i = 0; i < n; i++) {
        if (!slot(src[i], "ecu_kv_fork") || !slot(dst[i], "ecu_kv_fork")) return fail();
        if (src[i] == dst[i] || seq[dst[i]].len != 0) {
            ecu_set_error(nullptr, 0, "ecu_kv_fork: slot %d is not empty", dst[i]);
            return fail();
        }
        Seq &d = seq[dst[i]];
        const std::vector<int> &from = seq[src[i]].page;
        room(d.page, from.size());
        room(log_, 2 * from.size() + 1);
        room(cell_, from.size());
        room(length_, 1);
        for (int p : from) {
            hold(p);
            log_.push_back({U_HOLD, p, 0});
            d.page.push_back(p);
            log_.push_back({U_PUSH, dst[i], 0});
            cell_.push_back({dst[i], (int)d.page.size() - 1});
        }
        log_.push_back({U_LEN, dst[i], d.len});
        d.len = seq[src[i]].len;
        length_.push_back(dst[i]);
    }
    finish();
    return 0;
}

int KvBook::truncate(const int *s, const int *len, int n)
{
    begin();
    for (int i = 0; i < n; i++) {
        if (!slot(s[i], "ecu_kv_truncate")) return fail();
        Seq      &q = seq[s[i]];
        const int keep = len ? len[i] : 0;
        if (keep < 0 || keep > q.len) {
            ecu_set_error(nullptr, 0, "ecu_kv_truncate: sequence %d has %d positions, not %d", s[i], q.len, keep);
            return fail();
        }
        if (keep == q.len) continue;
        const size_t gone = q.page.size() - pages_of(keep);
        room(log_, 2 * gone + 1);
        room(cell_, gone);
        room(length_, 1);
        while ((int)q.page.size() > pages_of(keep)) {
            const int p = q.page.back();
            drop(p);
            log_.push_back({U_DROP, p, 0});
            q.page.pop_back();
            log_.push_back({U_POP, s[i], p});
            cell_.push_back({s[i], (int)q.page.size()});
        }
        log_.push_back({U_LEN, s[i], q.len});
        q.len = keep;
        length_.push_back(s[i]);
    }
    finish();
    return 0;
}

int KvBook::compact()
{
    begin();
    int hole = 0;
    for (int p = used; p < n_pages; p++) {
        if (!ref[p]) continue;
        while (ref[hole]) hole++;
        copies.push_back({p, hole});
        hole++;
    }
    if (copies.empty()) return 0;
    for (int s = 0; s < n_seq; s++)
        for (size_t j = 0; j < seq[s].page.size(); j++)
            if (seq[s].page[j] >= used) cell_.push_back({s, (int)j});
    room(sets, cell_.size());
    move_.resize((size_t)n_pages, -1);
    move_pages(false);
    compacted_ = true;
    finish();
    return (int)copies.size();
}
