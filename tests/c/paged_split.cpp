// The split of an attention call over the paged KV cache (paged_attn.h,
// paged_split.h), followed on the host piece by piece: where every (token, head)
// row's partial results are put, and where the join looks for them.
//
// Reads batches from stdin, one a line of whole numbers:
//   kv_type n_head n_kv hd page max_len n_prefix window n_seq n_tok table_stride has_off,
//   n_seq lengths, and with has_off n_seq + 1 offsets.
// Prints a line a batch: "ok" and counts, or what is wrong with the split.  The
// workspace starts with notes that lead out of it: what the join reads has to have
// been noted by the call, for rows of no sequence too.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../g4run_amd/csrc/paged_split.h"

using namespace g4;

namespace {

struct Error {
    std::string text;
};
[[noreturn]] void wrong(const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    throw Error{buf};
}

struct Part {
    size_t row;
    bool pre;
    int step, n, all;
};
struct Run {
    PagedAttn a;
    PagedLayout y;
    PagedPlan pl;
    std::vector<uint2> own, pre;
    std::unordered_map<size_t, Part> places;                 // byte offset in the workspace
    std::vector<int> out;                                    // times a row was written out
    long pieces = 0;
    int n_seq = 0;                                           // before the first torn one
};

template <bool MANY>
void follow(Run &r) {
    const PagedAttn &a = r.a;
    const PagedPlan &pl = r.pl;
    const PagedList &y = pa_list<MANY>(pl);
    std::vector<int64_t> upto(1, 0);                         // steps before each sequence
    for (int s = 0; s < r.n_seq; s++) upto.push_back(upto.back() + (int64_t)pa_steps<MANY>(a, pl, paged_seq(a.p, a.b, s)) * a.p.n_kv);
    const int64_t all = upto.back() + (int64_t)y.pre_tiles * y.pre_steps * a.p.n_kv;
    if (all > 0x7fffffff) wrong("%lld steps do not fit 32 bits", (long long)all);
    const int total = (int)all, share = pa_share(y, total);
    auto find = [&](int u, int &seq, int &before) {
        int lo = 0, hi = r.n_seq;                          // the last with upto <= u
        while (hi - lo > 1) (upto[(lo + hi) / 2] <= u ? lo : hi) = (lo + hi) / 2;
        seq = lo;
        before = (int)upto[lo];
    };
    for (int wg = 0; wg < y.wgs; wg++) {
        const int first = wg * share, stop = std::min(first + share, total);
        for (int u = first; u < stop;) {
            const PaPiece x = pa_piece_by<MANY>(a, pl, r.n_seq, wg, u, first, stop, find);
            if (x.took <= 0) wrong("a piece of no steps at %d", u);
            u += x.took;
            if (x.n == 0) {
                if (u != stop) wrong("a share ends early at %d", u);
                break;
            }
            r.pieces++;
            if (x.kvh >= a.p.n_kv || x.step < 0 || x.step + x.n > x.all) wrong("steps %d + %d of %d of head %d", x.step, x.n, x.all, x.kvh);
            if (x.end > x.start && (x.start < 0 || x.end > x.seglen)) wrong("positions %d .. %d of %d", x.start, x.end, x.seglen);
            if (!x.pre && !x.sq.bad) {                       // lowest position of the tile's first token: this piece's start, but for its steps
                const int64_t p0 = (int64_t)x.sq.len - x.sq.nq + (MANY ? (int64_t)x.tile * y.toks : 0), lo = std::max<int64_t>(0, a.window ? p0 + 1 - a.window : 0);
                if (x.start != (lo & ~31) + ((int64_t)x.step << y.shift)) wrong("a piece starts at %d, its tile at %lld", x.start, (long long)lo);
            }
            const int G = a.grp, r0 = MANY ? x.tile * y.rows : 0, r1 = MANY ? std::min(x.sq.nq * G, r0 + y.rows) : x.sq.nq * G;
            if (!MANY && r1 > y.rows) wrong("%d rows of a tile of %d", r1, y.rows);
            for (int i = r0; i < r1; i++) {
                const int tok = x.sq.t0 + i / G, head = x.kvh * G + i % G;
                if (tok < 0 || tok >= a.b.n_tok) wrong("token %d", tok);
                const size_t row = (size_t)tok * a.n_head + head;
                const PaSink to = pa_sink<MANY>(a, pl, x, share, i - r0, tok, head, !x.sq.bad && x.sq.len - x.sq.nq + i / G < 0, true);
                if (to.out) {
                    r.out[row]++;
                    continue;
                }
                const size_t at = (uint8_t *)to.o - a.ws, ml = (uint8_t *)to.ml - a.ws;
                if (at + a.p.hd * 4 > r.y.total || ml + sizeof(float2) > r.y.total) wrong("row %zu past the workspace", row);
                if (!r.places.emplace(at, Part{row, x.pre, x.step, x.n, x.all}).second) wrong("place %zu given to rows %zu and %zu", at, r.places[at].row, row);
                if (!r.places.emplace(ml, Part{row, x.pre, x.step, x.n, x.all}).second) wrong("sums %zu given to rows %zu and %zu", ml, r.places[ml].row, row);
            }
        }
    }
}

void joined(Run &r) {
    const PagedAttn &a = r.a;
    const int all = a.b.n_tok * a.n_head;
    std::vector<char> held(a.b.n_tok, 0), none(a.b.n_tok, 0);
    for (int s = 0; s < r.n_seq; s++) {
        const PagedSeq q = paged_seq(a.p, a.b, s);
        for (int i = 0; i < q.nq; i++) {
            if (held[q.t0 + i]++) wrong("token %d is two sequences'", q.t0 + i);
            none[q.t0 + i] = !q.bad && q.len - q.nq + i < 0;
        }
    }
    for (int row = 0; row < all; row++) {
        if (!held[row / a.n_head]) {
            if (r.out[row]) wrong("row %d without a sequence is written", row);
            if (r.y.join && r.own[row].x >> 2) wrong("row %d without a sequence is joined", row);
            continue;
        }
        if (!r.y.join) {
            if (r.out[row] != 1) wrong("row %d is written %d times", row, r.out[row]);
            continue;
        }
        const uint2 own = r.own[row], pre = a.b.n_prefix > 0 ? r.pre[row] : make_uint2(0, 0);
        const int n_pre = pre.x >> 2, n_own = own.x >> 2;
        if (n_own == 0) {
            if (r.out[row] != 1) wrong("row %d is written %d times", row, r.out[row]);
            continue;
        }
        if (r.out[row]) wrong("row %d is written and joined", row);
        if ((own.x >> 1 & 1) != (none[row / a.n_head])) wrong("row %d is noted as %s a position", row, own.x & 2 ? "without" : "with");
        if (n_pre > 4096 || n_own > 4096) wrong("row %d of %d + %d pieces", row, n_pre, n_own);
        int at = 0;                                          // steps so far, of the prefix's tile, then of the own one
        bool in_pre = n_pre > 0;
        for (int k = 0; k < n_pre + n_own; k++) {
            const PaPart p = pa_part(a, r.pl, row, pre, own, k);
            const size_t o = (uint8_t *)p.o - a.ws, ml = (uint8_t *)p.ml - a.ws;
            if (o + a.p.hd * 4 > r.y.total || ml + sizeof(float2) > r.y.total) wrong("piece %d of row %d lies past the workspace", k, row);
            if (k == n_pre) {
                in_pre = false;
                at = 0;
            }
            const auto x = r.places.find(o), z = r.places.find(ml);
            if (x == r.places.end() || z == r.places.end()) wrong("piece %d of row %d was not written", k, row);
            if (x->second.row != (size_t)row || z->second.row != (size_t)row) wrong("piece %d of row %d is row %zu's", k, row, x->second.row);
            if (x->second.pre != in_pre || x->second.step != at) wrong("piece %d of row %d is at step %d, not %d", k, row, x->second.step, at);
            at += x->second.n;
            if (k == (in_pre ? n_pre : n_pre + n_own) - 1 && at != x->second.all) wrong("row %d has %d of %d steps", row, at, x->second.all);
        }
        if (a.b.n_prefix && !n_pre) wrong("row %d without its prefix", row);
    }
}

}  // namespace

int main() {
    int t, n_head, n_kv, hd, page, max_len, n_prefix, window, n_seq, n_tok, stride, has_off;
    while (scanf("%d %d %d %d %d %d %d %d %d %d %d %d", &t, &n_head, &n_kv, &hd, &page, &max_len, &n_prefix, &window, &n_seq, &n_tok, &stride, &has_off) == 12) {
        std::vector<int> len(n_seq), off(has_off ? n_seq + 1 : 0);
        for (int &x : len) if (scanf("%d", &x) != 1) return 1;
        for (int &x : off) if (scanf("%d", &x) != 1) return 1;
        Run r;
        memset((void *)&r.a, 0, sizeof r.a);
        PagedAttn &a = r.a;
        a.p.type = t;
        a.p.n_kv = n_kv;
        a.p.hd = hd;
        a.p.page = page;
        a.b.n_seq = n_seq;
        a.b.n_tok = n_tok;
        a.b.q_off = has_off ? off.data() : nullptr;
        a.b.len = len.data();
        a.b.table_stride = stride;
        a.b.max_len = max_len;
        a.b.n_prefix = n_prefix;
        a.n_head = n_head;
        a.grp = n_head / n_kv;
        a.os = (size_t)n_head * hd;
        a.window = paged_window(a.b, window);
        a.ws = (uint8_t *)0x100000000;                       // never read or written
        r.y = paged_layout(a.p, a.b, a.grp, a.window);
        if (r.y.total > paged_layout(a.p, a.b, a.grp, 0).total) {
            printf("a window needs more workspace\n");
            continue;
        }
        r.pl = paged_places(r.y, a.ws);
        // what a call finds in its workspace: anything
        r.own.assign((size_t)n_tok * n_head, make_uint2(~0u, 0x7fffffffu));
        r.pre = r.own;
        r.out.assign((size_t)n_tok * n_head, 0);
        if (r.y.join) r.pl.own = r.own.data();
        r.pl.pre = r.pre.data();
        // the batch ends at its first torn sequence, behind which rows become NaN
        while (r.n_seq < n_seq && !paged_seq(a.p, a.b, r.n_seq).torn) r.n_seq++;
        std::vector<float> out(r.n_seq < n_seq ? (size_t)n_tok * n_head * hd : 0, 1.0f);
        a.out = out.data();
        try {
            pa_outside(a, r.pl, r.n_seq, 0, 1);
            for (size_t i = 0; i < out.size(); i++)
                if (std::isnan(out[i]) != (i >= (size_t)pa_tokens(a.b, r.n_seq) * n_head * hd)) wrong("element %zu behind a torn sequence", i);
            if (r.pl.many.rows) follow<true>(r);
            if (r.pl.few.rows) follow<false>(r);
            joined(r);
            printf("ok %ld pieces, %zu places\n", r.pieces, r.places.size() / 2);
        } catch (const Error &e) {
            printf("%s\n", e.text.c_str());
        }
        fflush(stdout);
    }
    return 0;
}
