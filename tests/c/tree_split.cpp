// The split of an attention call over trees of new tokens (paged_attn.h,
// paged_split.h), followed as paged_split.cpp follows the other calls': the same
// batches on stdin, the same lines.  A tree's tiles all reach to the sequence's last
// token, and a share may begin behind the last step of a tile that is not its own.
#define main paged_split_main
#include "paged_split.cpp"
#undef main

namespace {

template <bool MANY>
void follow_trees(Run &r) {
    const PagedAttn &a = r.a;
    const PagedPlan &pl = r.pl;
    const PagedList &y = pa_list<MANY>(pl);
    std::vector<int64_t> upto(1, 0);                         // costs before each sequence
    int dearest = y.pre_tiles ? y.toks : 0;                  // tokens of a tile
    for (int s = 0; s < r.n_seq; s++) {
        const PagedSeq q = paged_seq(a.p, a.b, s);
        upto.push_back(upto.back() + (int64_t)pa_steps<MANY, true>(a, pl, q) * a.p.n_kv);
        dearest = std::max(dearest, std::min(q.nq, y.toks));
    }
    const int64_t all = upto.back() + (int64_t)y.pre_tiles * y.pre_steps * pa_cost<MANY, true>(a, pl, y.toks) * a.p.n_kv;
    if (all > 0x7fffffff) wrong("%lld steps do not fit 32 bits", (long long)all);
    const int total = (int)all, share = MANY ? std::max(pa_share(y, total), pa_cost<MANY, true>(a, pl, dearest)) : pa_share(y, total);
    auto find = [&](int u, int &seq, int &before) {
        int lo = 0, hi = r.n_seq;                            // the last with upto <= u
        while (hi - lo > 1) (upto[(lo + hi) / 2] <= u ? lo : hi) = (lo + hi) / 2;
        seq = lo;
        before = (int)upto[lo];
    };
    for (int wg = 0; wg < y.wgs; wg++) {
        const int first = std::min<int64_t>((int64_t)wg * share, total), stop = std::min(first + share, total);
        for (int u = first; u < stop;) {
            const PaPiece x = pa_piece_by<MANY, true>(a, pl, r.n_seq, wg, u, first, stop, find);
            if (x.took <= 0) wrong("a piece of no steps at %d", u);
            const bool begins = u == first;
            u += x.took;
            if (x.n == 0) {
                if (u != stop && !(MANY && begins)) wrong("a share ends early at %d", u);
                continue;
            }
            r.pieces++;
            if (x.kvh >= a.p.n_kv || x.step < 0 || x.step + x.n > x.all) wrong("steps %d + %d of %d of head %d", x.step, x.n, x.all, x.kvh);
            if (x.end > x.start && (x.start < 0 || x.end > x.seglen)) wrong("positions %d .. %d of %d", x.start, x.end, x.seglen);
            if (!x.pre && !x.sq.bad) {                       // the tile's lowest position, but for the piece's steps
                const int64_t p0 = (int64_t)x.sq.len - x.sq.nq, lo = std::max<int64_t>(0, a.window ? p0 + 1 - a.window : 0);
                if (x.start != (lo & ~31) + ((int64_t)x.step << y.shift)) wrong("a piece starts at %d, its tile at %lld", x.start, (long long)lo);
                if (x.step + x.n == x.all && x.end != x.sq.len) wrong("the last piece ends at %d of %d", x.end, x.sq.len);
            }
            const int G = a.grp, r0 = MANY ? x.tile * y.rows : 0, r1 = MANY ? std::min(x.sq.nq * G, r0 + y.rows) : x.sq.nq * G;
            if ((r1 <= r0 && !x.pre) || r1 - r0 > y.rows) wrong("%d rows of a tile of %d", r1 - r0, y.rows);
            for (int i = r0; i < r1; i++) {
                const int tok = x.sq.t0 + i / G, head = x.kvh * G + i % G;
                if (tok < 0 || tok >= a.b.n_tok) wrong("token %d", tok);
                const size_t row = (size_t)tok * a.n_head + head;
                const PaSink to = pa_sink<MANY, true>(a, pl, x, share, i - r0, tok, head, !x.sq.bad && x.sq.len - x.sq.nq + i / G < 0, true);
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
    // all of it: a call has no workgroups behind these
    if ((int64_t)y.wgs * share < total) wrong("%lld steps of %d are taken", (long long)y.wgs * share, total);
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
        r.y = paged_layout(a.p, a.b, a.grp, a.window, true);
        if (r.y.total > paged_layout(a.p, a.b, a.grp, 0, true).total) {
            printf("a window needs more workspace\n");
            continue;
        }
        r.pl = paged_places(r.y, a.ws);
        r.own.assign((size_t)n_tok * n_head, make_uint2(~0u, 0x7fffffffu));          // what a call finds in its workspace: anything
        r.pre = r.own;
        r.out.assign((size_t)n_tok * n_head, 0);
        if (r.y.join) r.pl.own = r.own.data();
        r.pl.pre = r.pre.data();
        while (r.n_seq < n_seq && !paged_seq(a.p, a.b, r.n_seq).torn) r.n_seq++;
        std::vector<float> out(r.n_seq < n_seq ? (size_t)n_tok * n_head * hd : 0, 1.0f);
        a.out = out.data();
        try {
            pa_outside(a, r.pl, r.n_seq, 0, 1);
            if (r.pl.many.rows) follow_trees<true>(r);
            if (r.pl.few.rows) follow_trees<false>(r);
            joined(r);
            printf("ok %ld pieces, %zu places\n", r.pieces, r.places.size() / 2);
        } catch (const Error &e) {
            printf("%s\n", e.text.c_str());
        }
        fflush(stdout);
    }
    return 0;
}
