"""Block tables, paged append, page-sparse attention, adapters and logits rules against plain 64-bit restatements."""
import numpy as np
import pytest
import torch

from zeroplatform_b200 import ops
from zeroplatform_b200._lib import ZcError

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------------------------------------


class Pool:
    """The page pool's rules on the host."""

    def __init__(self, rng, max_rows, max_pages, num_pages, page):
        self.page = page
        self.table = np.full((max_rows, max_pages), -1, np.int64)
        self.lens = np.zeros(max_rows, np.int64)
        self.free = np.zeros(num_pages, np.int64)
        self.free[:] = rng.permutation(num_pages)
        self.count = num_pages

    def reserve(self, rows, new, tokens):
        start, granted, named, pages = [0], [], set(), 0
        slots = np.full(tokens, -1, np.int64)
        pos, row_of, ctx = np.zeros(tokens, np.int64), np.full(tokens, -1, np.int64), np.zeros(tokens, np.int64)
        top = self.count
        for r, n in zip(rows, new):
            n = max(int(n), 0)
            start.append(start[-1] + n)
            ok = 0 <= r < len(self.lens) and r not in named
            named.add(r)
            if ok:
                old = int(self.lens[r])
                ok = old + n <= self.table.shape[1] * self.page and start[-1] <= tokens
            if ok:
                have, need = -(-old // self.page), -(-(old + n) // self.page)
                pages += need - have
                ok = pages <= top
            granted.append(int(ok))
            if not ok:
                continue
            for c in range(have, need):
                self.count -= 1
                self.table[r, c] = self.free[self.count]
            for i in range(n):
                t, p = start[-2] + i, old + i
                slots[t] = self.table[r, p // self.page] * self.page + p % self.page
                pos[t], row_of[t], ctx[t] = p, r, p + 1
            self.lens[r] = old + n
        return np.array(start), slots, pos, row_of, ctx, np.array(granted)

    def trim(self, rows, new):
        named = set()
        use = []
        for r, n in zip(rows, new):
            use.append(0 <= r < len(self.lens) and r not in named)
            named.add(r)
        for (r, n), ok in reversed(list(zip(zip(rows, new), use))):
            if not ok:
                continue
            keep = min(max(int(n), 0), int(self.lens[r]))
            for c in range(-(-int(self.lens[r]) // self.page) - 1, -(-keep // self.page) - 1, -1):
                self.free[self.count] = self.table[r, c]
                self.count += 1
                self.table[r, c] = -1
            self.lens[r] = keep


def upload(p):
    return (dev(p.table, torch.int32), dev(p.lens, torch.int32), dev(p.free, torch.int32), ints([p.count]))


def same_pool(p, d):
    assert d[3].item() == p.count
    np.testing.assert_array_equal(d[0].cpu().numpy(), p.table)
    np.testing.assert_array_equal(d[1].cpu().numpy(), p.lens)
    np.testing.assert_array_equal(d[2].cpu().numpy(), p.free)


def same_plan(plan, want):
    for name, got, ref in zip(plan._fields, plan, want):
        np.testing.assert_array_equal(got.cpu().numpy(), ref, err_msg=name)


@pytest.mark.parametrize("batch,max_rows,max_pages,num_pages,page,hi", [
    (1, 1, 4, 4, 16, 9), (3, 7, 8, 20, 16, 40), (64, 64, 40, 1500, 16, 3), (130, 200, 33, 2100, 8, 70),
    (37, 64, 9, 200, 5, 30), (1500, 2000, 4, 3000, 16, 12)])
def test_pages_follow_the_host(batch, max_rows, max_pages, num_pages, page, hi):
    """Steps of ragged requests on a pool that runs full, each trimmed a little: every array as the host has it."""
    rng = np.random.default_rng(batch * 31 + page)
    p = Pool(rng, max_rows, max_pages, num_pages, page)
    d = upload(p)
    for step in range(6):
        rows = rng.permutation(max_rows)[:batch]
        new = rng.integers(-1, hi + 1, batch)
        tokens = int(np.maximum(new, 0).sum()) + int(rng.integers(-3, 9))
        tokens = max(tokens, 0)
        plan = ops.reserve_pages(*d, ints(new), page, rows=ints(rows), tokens=tokens)
        same_plan(plan, p.reserve(rows, new, tokens))
        same_pool(p, d)
        rows = rng.permutation(max_rows)[:batch]
        new = np.where(rng.random(batch) < 0.3, 0, p.lens[rows] - rng.integers(-2, hi // 2 + 2, batch))
        ops.trim_pages(*d, ints(new), page, rows=ints(rows))
        p.trim(rows, new)
        same_pool(p, d)


def test_pages_refuse_rows_out_of_range_and_named_twice():
    rng = np.random.default_rng(1)
    p = Pool(rng, 6, 8, 30, 4)
    d = upload(p)
    rows, new = [3, -1, 3, 6, 0, 2 ** 31 - 1, 5], [5, 2, 9, 1, 4, 1, 0]
    plan = ops.reserve_pages(*d, ints(new), 4, rows=ints(rows), tokens=22)
    same_plan(plan, p.reserve(rows, new, 22))
    assert plan.granted.tolist() == [1, 0, 0, 0, 1, 0, 1]
    ops.trim_pages(*d, ints([2, 0, 0, 0, 3, 0, 0]), 4, rows=ints(rows))
    p.trim(rows, [2, 0, 0, 0, 3, 0, 0])
    same_pool(p, d)


def test_pages_empty_steps():
    rng = np.random.default_rng(2)
    p = Pool(rng, 4, 8, 8, 16)
    d = upload(p)
    plan = ops.reserve_pages(*d, ints([]), 16, tokens=3)
    assert plan.start.tolist() == [0] and plan.slots.tolist() == [-1] * 3 and plan.ctx_len.tolist() == [0] * 3
    plan = ops.reserve_pages(*d, ints([0, 0]), 16, tokens=0)
    assert plan.granted.tolist() == [1, 1] and plan.start.tolist() == [0, 0, 0]
    ops.trim_pages(*d, ints([]), 16)
    same_pool(p, d)


def test_pages_taken_back_leave_the_stack_as_it_was():
    rng = np.random.default_rng(3)
    p = Pool(rng, 40, 30, 700, 16)
    d = upload(p)
    ops.reserve_pages(*d, ints(rng.integers(1, 60, 40)), 16, tokens=3000)
    before = [t.clone() for t in d]
    ops.reserve_pages(*d, ints(rng.integers(0, 200, 40)), 16, tokens=9000)
    ops.trim_pages(*d, before[1], 16)
    for a, b in zip(before, d):
        assert torch.equal(a, b)


def test_pages_run_out_for_a_request_and_all_behind_it():
    """A prompt larger than the stack stops whoever comes after it, with or without a page to take; put last, it stops
    nobody."""
    pool = lambda: (torch.full((3, 8), -1, dtype=torch.int32, device="cuda"), ints([5, 0, 5]), ints([3, 1, 2, 0]),  # noqa: E731
                    ints([2]))
    d = pool()
    d[0][0, 0], d[0][2, 0] = 2, 0
    plan = ops.reserve_pages(*d, ints([1, 100, 1]), 16, tokens=102)
    assert plan.granted.tolist() == [1, 0, 0] and d[1].tolist() == [6, 0, 5] and d[3].item() == 2
    assert plan.slots[0].item() == 2 * 16 + 5 and (plan.slots[1:] == -1).all()
    plan = ops.reserve_pages(*d, ints([1, 1, 100]), 16, rows=ints([0, 2, 1]), tokens=102)
    assert plan.granted.tolist() == [1, 1, 0] and d[1].tolist() == [7, 0, 6] and d[3].item() == 2


def test_pages_slots_pass_32_bits():
    """A pool of few pages that are very long: the slot is page * page_size in 64 bits."""
    page = 1 << 30
    table, lens = torch.full((1, 2), -1, dtype=torch.int32, device="cuda"), ints([0])
    free, count = ints([6, 7]), ints([2])
    plan = ops.reserve_pages(table, lens, free, count, ints([2]), page, tokens=2)
    assert plan.slots.tolist() == [7 * page, 7 * page + 1]


def test_pages_in_a_captured_graph_and_on_a_side_stream():
    rng = np.random.default_rng(4)
    p = Pool(rng, 16, 64, 1024, 16)
    d = upload(p)
    new, out = ints([3] * 16), ops.PagePlan.empty(16, 48)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.reserve_pages(*d, new, 16, out=out)
    torch.cuda.current_stream().wait_stream(s)
    p.reserve(range(16), [3] * 16, 48)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.reserve_pages(*d, new, 16, out=out)
    for _ in range(5):
        g.replay()
        want = p.reserve(range(16), [3] * 16, 48)
        same_plan(out, want)
    same_pool(p, d)


# ---------------------------------------------------------------------------------------------------------
# paged append
# ---------------------------------------------------------------------------------------------------------


def key_bounds(k):
    """k [..., tokens, hd] as stored -> (codes [..., 2, hd], scales [...]), from the definition in 64 bits."""
    k = k.astype(np.float64)
    lo, hi = k.min(-2), k.max(-2)
    s = (np.maximum(np.abs(lo), np.abs(hi)).max(-1) / 127).astype(np.float32)
    d = np.where(s > 0, s, 1).astype(np.float64)[..., None]
    c = np.stack([np.floor(lo / d), np.ceil(hi / d)], -2)
    return np.clip(c, -127, 127).astype(np.int8), s


@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("src,dst", [("float32", "float16"), ("float16", "float16"), ("float32", "float32"),
                                     ("float16", "float32")])
@pytest.mark.parametrize("hkv,hd,page,lens", [
    (2, 128, 16, [(0, 1), (5, 1), (15, 1), (16, 1), (47, 1)]), (3, 64, 16, [(0, 40), (7, 33), (31, 2), (12, 0)]),
    (1, 256, 8, [(3, 50)]), (5, 32, 5, [(4, 19), (0, 5), (9, 1)]), (8, 128, 64, [(10, 200), (64, 64), (1, 62)]),
    (12, 64, 16, [(3, 900)])])
def test_append_stores_rows_and_bounds(hkv, hd, page, lens, src, dst, head_major):
    rng = np.random.default_rng(hkv * hd + page)
    per = max(-(-(a + b) // page) for a, b in lens)
    pages = len(lens) * per + 2
    table = rng.permutation(pages)
    pool = [rng.standard_normal((pages, hkv, page, hd)).astype(dst) for _ in range(2)]
    slots, last = [], {}
    for b, (old, new) in enumerate(lens):
        for p in range(old, old + new):
            slots.append(table[b * per + p // page] * page + p % page)
            last[slots[-1] // page] = p % page + 1
        slots.append(-1)  # padding between the sequences
    slots += [pages * page, 1 << 40]
    rows = [rng.standard_normal((len(slots), hkv, hd)).astype(src) for _ in range(2)]
    # a wider activation row than the heads fill, as a slice of fused q | k | v
    wide = torch.zeros((len(slots), 2 * hkv * hd + 8), dtype=getattr(torch, src), device="cuda")
    k, v = (wide[:, i * hkv * hd:(i + 1) * hkv * hd].view(-1, hkv, hd) for i in range(2))
    k.copy_(dev(rows[0]))
    v.copy_(dev(rows[1]))

    def up(x):
        return dev(x) if head_major else dev(x.transpose(0, 2, 1, 3)).transpose(1, 2)

    kp, vp = up(pool[0]), up(pool[1])
    bounds = torch.full((pages, hkv, 2, hd), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((pages, hkv), -7.0, device="cuda")
    ops.append_kv(k, v, dev(np.array(slots, np.int64)), kp, vp, bounds, scales)
    for t, s in enumerate(slots):
        if 0 <= s < pages * page:
            pool[0][s // page, :, s % page] = rows[0][t].astype(dst)
            pool[1][s // page, :, s % page] = rows[1][t].astype(dst)
    np.testing.assert_array_equal(kp.cpu().numpy(), pool[0])
    np.testing.assert_array_equal(vp.cpu().numpy(), pool[1])
    got_b, got_s = bounds.cpu().numpy(), scales.cpu().numpy()
    for p in range(pages):
        if p in last:
            want_b, want_s = key_bounds(pool[0][p, :, :last[p]])
            np.testing.assert_array_equal(got_s[p], want_s)
            np.testing.assert_array_equal(got_b[p], want_b)
        else:  # a page that nothing was written to keeps its bounds
            assert (got_b[p] == 99).all() and (got_s[p] == -7).all()


def test_append_bounds_hold_the_keys_and_odd_values_stay_finite():
    """lo * s <= k <= hi * s up to the ulp of the largest key, for zeros, subnormals and powers of two; a page with an
    infinite key has zero codes."""
    k = torch.zeros((6, 1, 64), device="cuda")
    k[1] = 2.0 ** -24
    k[2] = torch.linspace(-1, 1, 64, device="cuda")
    k[3] = 2.0 ** torch.arange(-32, 32, device="cuda").float()
    k[4, 0, 3] = float("inf")
    k[5] = torch.randn(64, device="cuda") * 1e-42
    pools = [torch.zeros((6, 1, 16, 64), device="cuda") for _ in range(2)]
    bounds, scales = torch.zeros((6, 1, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((6, 1), device="cuda")
    ops.append_kv(k, k, torch.arange(6, device="cuda") * 16, *pools, bounds, scales)
    b, s = bounds.double().cpu()[:, 0], scales.double().cpu()[:, 0, None]
    kk = k[:, 0].double().cpu()
    for p in (0, 1, 2, 3):
        slack = kk[p].abs().max() * 2.0 ** -23
        assert (b[p, 0] * s[p] <= kk[p] + slack).all() and (b[p, 1] * s[p] >= kk[p] - slack).all(), p
        assert (b[p].abs() <= 127).all()
    assert (b[4] == 0).all() and torch.isinf(s[4]).all()
    assert (b[5].abs() <= 127).all()
    assert (pools[0][4, 0, 0] == k[4, 0]).all()


@pytest.mark.parametrize("src,dst", [("float32", "float16"), ("float16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("hkv,hd,page,pages", [(2, 128, 16, 60), (1, 256, 8, 40), (12, 64, 64, 80), (3, 32, 200, 6),
                                               (8, 128, 1, 30), (8, 256, 32, 90)])
def test_append_pages_with_gaps_and_skipped_entries(hkv, hd, page, pages, src, dst):
    """Tokens of a page in ascending slots that leave some out (which keep what they hold), with skipped entries, a few or
    hundreds, between tokens of one page and of different ones: every row and every page's bounds as the host has
    them."""
    rng = np.random.default_rng(hkv * hd + page)
    pool = [rng.standard_normal((pages, hkv, page, hd)).astype(dst) for _ in range(2)]
    slots, last = [], {}
    for p in rng.permutation(pages - 1):
        for j in np.sort(rng.choice(page, rng.integers(1, page + 1), replace=False)):
            if rng.random() < 0.25:
                skipped = int(rng.choice([-1, -2 ** 40, pages * page, 2 ** 62]))
                slots += [skipped] * int(rng.choice([1, 2, 40, 700], p=[0.6, 0.25, 0.13, 0.02]))
            slots.append(int(p) * page + int(j))
            last[p] = int(j) + 1
    rows = [rng.standard_normal((len(slots), hkv, hd)).astype(src) for _ in range(2)]
    kp, vp = dev(pool[0]), dev(pool[1])
    bounds = torch.full((pages, hkv, 2, hd), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((pages, hkv), -7.0, device="cuda")
    ops.append_kv(dev(rows[0]), dev(rows[1]), dev(np.array(slots, np.int64)), kp, vp, bounds, scales)
    for t, s in enumerate(slots):
        if 0 <= s < pages * page:
            pool[0][s // page, :, s % page] = rows[0][t].astype(dst)
            pool[1][s // page, :, s % page] = rows[1][t].astype(dst)
    np.testing.assert_array_equal(kp.cpu().numpy(), pool[0])
    np.testing.assert_array_equal(vp.cpu().numpy(), pool[1])
    got_b, got_s = bounds.cpu().numpy(), scales.cpu().numpy()
    for p in range(pages - 1):
        want_b, want_s = key_bounds(pool[0][p, :, :last[p]])
        np.testing.assert_array_equal(got_s[p], want_s)
        np.testing.assert_array_equal(got_b[p], want_b)
    assert (got_b[-1] == 99).all() and (got_s[-1] == -7).all()


def test_append_without_bounds_and_of_nothing():
    k = torch.randn((3, 2, 128), device="cuda")
    pools = [torch.zeros((4, 2, 16, 128), device="cuda", dtype=torch.float16) for _ in range(2)]
    ops.append_kv(k, k, torch.tensor([0, 1, 63], device="cuda"), *pools)
    assert torch.equal(pools[0][3, :, 15], k[2].half()) and torch.equal(pools[1][0, :, 1], k[1].half())
    ops.append_kv(k[:0], k[:0], torch.empty(0, dtype=torch.int64, device="cuda"), *pools)
    with pytest.raises(ZcError):
        ops.append_kv(k, k, torch.tensor([0, 1], device="cuda"), *pools)
    with pytest.raises(ZcError):
        ops.append_kv(k.double(), k.double(), torch.tensor([0, 1, 2], device="cuda"), *pools)


# ---------------------------------------------------------------------------------------------------------
# page-sparse attention
# ---------------------------------------------------------------------------------------------------------


def plain_select(q, codes, scales, n, budget, sink, recent):
    """q [group, hd] fp32; codes [n, 2, hd]; scales [n] (None entries: no such page) -> ascending page list."""
    if n <= budget:
        return list(range(n))
    top = np.abs(q).max(-1)
    s_q = (top.astype(np.float64) / 32512).astype(np.float32)
    d = np.where(s_q > 0, s_q, 1)[:, None].astype(np.float64)
    qi = np.rint((q / d).astype(np.float32)).astype(np.int64)
    isum = np.maximum(qi[:, None] * codes[None, :, 0].astype(np.int64),
                      qi[:, None] * codes[None, :, 1].astype(np.int64)).sum(-1)
    score = (isum.astype(np.float32) * s_q[:, None]).max(0) * scales
    order = [(-np.inf if p < sink or p >= n - recent else (np.inf if np.isnan(scales[p]) else -score[p]), p)
             for p in range(n)]
    return sorted(p for _, p in sorted(order)[:budget])


def plain_attention(q, k, v, scale):
    """One head group over gathered tokens in 64 bits; also the size of the score terms, for the tolerance."""
    z = q.astype(np.float64) @ k.T.astype(np.float64) * scale
    mag = (np.abs(q).astype(np.float64) @ np.abs(k.T).astype(np.float64)).max() * abs(scale) if len(k) else 0.0
    z = np.exp(z - z.max(-1, keepdims=True))
    return z @ v.astype(np.float64) / z.sum(-1, keepdims=True), mag


def sparse_case(rng, ctx, hq, hkv, hd, page, half, head_major=True, per=None, bad_pages=False):
    batch = len(ctx)
    per = per or max(1, max(-(-x // page) for x in ctx))
    pages = batch * per + 3
    table = rng.permutation(pages)[:batch * per].reshape(batch, per).astype(np.int32)
    if bad_pages:
        table[rng.random(table.shape) < 0.2] = rng.choice([-1, pages, 2 ** 31 - 1])
    dt = np.float16 if half else np.float32
    k = (rng.standard_normal((pages, hkv, page, hd)) + 1.5 * rng.standard_normal((pages, hkv, 1, hd))).astype(dt)
    v = rng.standard_normal((pages, hkv, page, hd)).astype(dt)
    codes, scales = key_bounds(k)
    # slots behind a sequence's last token hold anything
    for b, x in enumerate(ctx):
        p = table[b, x // page] if x % page else -1
        if 0 <= p < pages:
            codes[p], scales[p] = key_bounds(k[p, :, :x % page])
            k[p, :, x % page:], v[p, :, x % page:] = np.nan, np.inf
    q = rng.standard_normal((batch, hq, hd)).astype(np.float32)

    def up(x):
        return dev(x) if head_major else dev(x.transpose(0, 2, 1, 3)).transpose(1, 2)

    return q, k, v, codes, scales, table, (up(k), up(v), dev(codes), dev(scales), dev(table))


def check_sparse(q, k, v, codes, scales, table, ctx, budget, sink, recent, out, sel, rows=None):
    """Selection exactly.  Output tolerance, relative to the largest value attended: a score is off by at most hd
    roundings of 2^-23 of the terms it adds (products of hi + lo pairs hold 2^-22), which moves a weight by as much
    relatively, on both sides of the quotient; sums over T tokens add T / 8 accumulator roundings and a constant."""
    batch, hq, hd = q.shape
    pages, hkv, page, _ = k.shape
    group = hq // hkv
    scale = 1 / np.sqrt(hd)
    out, sel = out.cpu().numpy(), sel.cpu().numpy()
    for b in range(batch):
        r = b if rows is None else rows[b]
        n = -(-int(ctx[b]) // page) if 0 <= r < len(table) else 0
        for h in range(hkv):
            hs = slice(h * group, (h + 1) * group)
            t = table[r, :n] if n else table[0, :0]
            ok = (t >= 0) & (t < pages)
            at = np.where(ok, t, 0)
            sc = np.where(ok, scales[at, h], np.nan).astype(np.float32)
            want = plain_select(q[b, hs], codes[at, h], sc, n, budget, sink, recent)
            assert sel[b, h].tolist() == want + [-1] * (budget - len(want)), (b, h)
            keep = [(p, j) for p in want if ok[p] for j in range(page) if p * page + j < ctx[b]]
            if not keep:
                assert (out[b, hs] == 0).all()
                continue
            kk = np.stack([k[t[p], h, j] for p, j in keep])
            vv = np.stack([v[t[p], h, j] for p, j in keep])
            ref, mag = plain_attention(q[b, hs], kk, vv, scale)
            tol = np.abs(vv.astype(np.float64)).max() * (2 * hd * 2.0 ** -23 * mag + (len(keep) / 8 + 64) * 2.0 ** -23)
            assert np.abs(out[b, hs] - ref).max() <= tol, (b, h, np.abs(out[b, hs] - ref).max(), tol)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("hq,hkv,hd,page,ctx,budget,sink,recent", [
    (8, 2, 128, 16, [1, 15, 16, 17, 0, 300], 4, 1, 1), (4, 4, 64, 16, [129, 1000, 64], 8, 0, 1),
    (32, 8, 128, 16, [2049], 16, 1, 2), (7, 1, 64, 8, [777, 63], 12, 2, 3), (6, 2, 256, 32, [1500, 31], 9, 1, 1),
    (16, 1, 128, 16, [700, 1200], 20, 1, 4), (24, 2, 64, 24, [1000], 11, 0, 0), (12, 12, 64, 16, [640], 40, 1, 1),
    (40, 2, 128, 64, [5000, 4999], 30, 1, 1), (8, 8, 128, 16, [333] * 40, 6, 1, 2), (2, 1, 128, 16, [9000], 1, 0, 1)])
def test_sparse_attention(hq, hkv, hd, page, ctx, budget, sink, recent, half):
    rng = np.random.default_rng(hq * 100 + hd + page)
    q, k, v, codes, scales, table, d = sparse_case(rng, ctx, hq, hkv, hd, page, half, head_major=hd != 64)
    out, sel = ops.sparse_paged_attention(dev(q), *d, ints(ctx), budget, sink=sink, recent=recent)
    check_sparse(q, k, v, codes, scales, table, ctx, budget, sink, recent, out, sel)


@pytest.mark.parametrize("half", [True, False])
def test_sparse_attention_rows_strides_and_bad_pages(half):
    """Queries that share table rows, rows without a sequence, a strided q, table entries outside the pool, and a
    max_ctx below a length."""
    rng = np.random.default_rng(9)
    lens = [500, 37, 900]
    q, k, v, codes, scales, table, d = sparse_case(rng, lens, 8, 2, 128, 16, half, bad_pages=True)
    rows = [2, 0, 0, -1, 1, 3, 2, 2 ** 31 - 1]
    ctx = [899, 500, 499, 12, 37, 5, 16, 3]
    q = rng.standard_normal((8, 8, 128)).astype(np.float32)
    wide = torch.zeros((8, 12 * 128), device="cuda")
    wide[:, 128:9 * 128] = dev(q.reshape(8, -1))
    view = wide[:, 128:9 * 128].view(8, 8, 128)
    # token 499 of row 0 and 898 of row 2 are the last ones with keys: shorter rows see only stored tokens
    out, sel = ops.sparse_paged_attention(view, *d, ints(ctx), 10, rows=ints(rows), recent=2)
    check_sparse(q, k, v, codes, scales, table, ctx, 10, 1, 2, out, sel, rows)
    cut, sel_cut = ops.sparse_paged_attention(view, *d, ints(ctx), 10, rows=ints(rows), recent=2, max_ctx=320)
    check_sparse(q, k, v, codes, scales, table, [min(x, 320) for x in ctx], 10, 1, 2, cut, sel_cut, rows)


def test_sparse_attention_whole_budget_is_paged_attention():
    """With a budget that holds every page the result is that of paged_attention_batched (both hold fp32 to 1e-5)."""
    rng = np.random.default_rng(10)
    ctx = [1, 200, 640, 0]
    q, k, v, codes, scales, table, d = sparse_case(rng, ctx, 12, 4, 128, 16, True)
    out, _ = ops.sparse_paged_attention(dev(q), *d, ints(ctx), 40)
    pools = [torch.nan_to_num(x, nan=0.0, posinf=0.0) for x in d[:2]]
    sp, sh, ss, _ = pools[0].stride()
    ref = ops.paged_attention_batched(dev(q), *pools, d[4], ints(ctx), 4, 16, pools[0].shape[0], sp, ss, sh,
                                      1 / np.sqrt(128), 640)
    assert (out - ref).abs().max() <= 1e-5 * ref.abs().max()


def test_sparse_attention_extreme_queries():
    """Queries far outside fp16's range, all zero, and with one element that dwarfs the rest."""
    rng = np.random.default_rng(11)
    ctx = [400, 400, 400, 400]
    q, k, v, codes, scales, table, d = sparse_case(rng, ctx, 4, 2, 64, 16, True)
    q[0] *= np.float32(1e6)
    q[1] *= np.float32(1e-20)
    q[2] = 0
    q[3, :, 5] = 3e5
    out, sel = ops.sparse_paged_attention(dev(q), *d, ints(ctx), 7, sink=0)
    check_sparse(q, k, v, codes, scales, table, ctx, 7, 0, 1, out, sel)
    q[1, 0, 0] = np.nan
    out, _ = ops.sparse_paged_attention(dev(q), *d, ints(ctx), 7)
    assert torch.isnan(out[1, 0]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2:]).all()


def test_sparse_attention_equal_pages_go_to_the_lower_one():
    page, hd = 16, 64
    k = torch.ones((40, 1, page, hd), dtype=torch.float16, device="cuda")
    k[20:] = 2
    codes, scales = (dev(x) for x in key_bounds(k.cpu().numpy()))
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    q = torch.ones((1, 1, hd), device="cuda")
    for budget in (3, 20, 25, 39):
        _, sel = ops.sparse_paged_attention(q, k, k, codes, scales, table, ints([640]), budget, sink=0, recent=0)
        high = list(range(20, min(40, 20 + budget)))
        assert sel[0, 0].tolist() == sorted(high + list(range(budget - len(high))))


def test_sparse_attention_pages_with_infinite_keys_come_first():
    """As append_kv leaves them: codes 0 and an infinite scale, for queries of either sign and of zeros."""
    page, hd = 16, 64
    k = torch.randn((40, 1, page, hd), device="cuda")
    k[17, 0, 3, 9], k[30, 0, 0, 0], k[33, 0, 5, 4] = float("inf"), -float("inf"), float("nan")
    pools = [torch.zeros((40, 1, page, hd), device="cuda") for _ in range(2)]
    bounds, scales = torch.zeros((40, 1, 2, hd), dtype=torch.int8, device="cuda"), torch.zeros((40, 1), device="cuda")
    rows = k.transpose(1, 2).reshape(-1, 1, hd)
    ops.append_kv(rows, rows, torch.arange(640, device="cuda"), *pools, bounds, scales)
    assert torch.isfinite(scales).flatten().logical_not().nonzero().flatten().tolist() == [17, 30]
    q = torch.randn((3, 1, hd), device="cuda")
    q[1] *= -1e-20
    q[2] = 0
    table = torch.arange(40, dtype=torch.int32, device="cuda").expand(3, 40).contiguous()
    _, sel = ops.sparse_paged_attention(q, *pools, bounds, scales, table, ints([640] * 3), 2, sink=0, recent=0)
    assert sel.flatten(1).tolist() == [[17, 30]] * 3


def test_sparse_attention_long_sequence_many_pages():
    """More pages than one CTA scores, in a pool whose far pages lie beyond 32-bit element offsets."""
    rng = np.random.default_rng(12)
    page, hd, n = 8, 64, 20000
    pages = (1 << 31) // (page * hd) + 64  # elements of the pool: just past 2^31
    k = torch.zeros((pages, 1, page, hd), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.randperm(pages - 1, device="cuda")[:n].int()[None]
    table[0, -1] = pages - 1
    q = rng.standard_normal((1, 3, hd)).astype(np.float32)
    ks = rng.standard_normal((n, 1, page, hd)).astype(np.float16)
    vs = rng.standard_normal((n, 1, page, hd)).astype(np.float16)
    at = table[0].long()
    k[at], v[at] = dev(ks), dev(vs)
    codes, scales = key_bounds(ks)
    bounds = torch.zeros((pages, 1, 2, hd), dtype=torch.int8, device="cuda")
    sc = torch.zeros((pages, 1), device="cuda")
    bounds[at], sc[at] = dev(codes), dev(scales)
    ctx = n * page - 3
    out, sel = ops.sparse_paged_attention(dev(q), k, v, bounds, sc, table, ints([ctx]), 50)
    check_sparse(q, ks, vs, codes, scales, np.arange(n, dtype=np.int32)[None], [ctx], 50, 1, 1, out, sel)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_sparse_attention_long_sums_have_no_bias(dtype):
    """Equal weights over 65,536 values in [1, 2), so that a weight, the sum of weights and hi parts are exact and an
    output is a mean.  A block's sum in the tensor core may lose less than an ulp (2^-23) per addend, 16 products (8 of
    fp32) and the accumulator; whatever is rounded to nearest errs to either side, by at most 2^-24 in each of the 1,024
    additions of a warp, which six standard deviations of the mean over 19,200 outputs bound by 1e-7."""
    batch, pages, page, hkv, hd = 150, 2048, 32, 2, 64
    g = torch.Generator(device="cuda").manual_seed(31)
    v = (1 + torch.rand(pages, hkv, page, hd, device="cuda", generator=g)).to(dtype)
    codes, scales = torch.zeros(pages, hkv, 2, hd, dtype=torch.int8, device="cuda"), torch.zeros(pages, hkv, device="cuda")
    table = torch.stack([torch.randperm(pages, device="cuda", generator=g) for _ in range(batch)]).int()
    q = torch.zeros(batch, hkv, hd, device="cuda")
    out, _ = ops.sparse_paged_attention(q, v, v, codes, scales, table, ints([pages * page] * batch), pages)
    want = v.double().mean((0, 2))
    addends = 17 if dtype == torch.float16 else 9
    assert abs(float((out.double() / want - 1).mean())) <= addends * 2.0 ** -23 + 1e-7


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("batch", [1, 20, 80])
@pytest.mark.parametrize("hq,hkv,hd,every", [(1, 1, 64, 1 << 20), (8, 2, 128, 128), (2, 2, 256, 1 << 20), (12, 1, 64, 16)])
def test_sparse_attention_rows_carried_by_small_weights(hq, hkv, hd, every, batch, half):
    """Tokens of value 0 (every `every`-th one) take nearly all of the softmax and give nothing to the output, which is
    the sum of weights 12 to 30 nats below them: attention sinks.  Every other value lies in [0.5, 1.5], so outputs have no
    cancellation and are compared relative to themselves.  A score is off by at most hd roundings of 2^-23 of the terms
    it adds (|q| |k| scale <= gap + 2), which moves a weight by as much relatively, here in the numerator and in the
    sink's weight; sums over T tokens add T / 8 roundings of 2^-23 and a constant, which holds a weight's two halves.
    Weights of fp16 pools are held to 2^-50 of the largest one among 16 neighbours, where those have a sink among them."""
    rng = np.random.default_rng(hq * hd + batch)
    page, tokens = 16, 2040
    n = -(-tokens // page)
    dt = np.float16 if half else np.float32
    k = np.zeros((n, hkv, page, hd), dt)
    k[..., 1] = (-2 * rng.random((n, hkv, page))).astype(dt)
    v = (0.5 + rng.random((n, hkv, page, hd))).astype(dt)
    flat_k, flat_v = k.transpose(0, 2, 1, 3).reshape(n * page, hkv, hd).copy(), \
        v.transpose(0, 2, 1, 3).reshape(n * page, hkv, hd).copy()
    sinks = np.arange(3, tokens, every)
    flat_k[sinks, :, 0], flat_k[sinks, :, 1], flat_v[sinks] = 1, 0, 0
    k = flat_k.reshape(n, page, hkv, hd).transpose(0, 2, 1, 3)
    v = flat_v.reshape(n, page, hkv, hd).transpose(0, 2, 1, 3)
    gaps = np.linspace(12, 30, batch * hq).reshape(batch, hq) if batch > 1 else np.linspace(16, 22, hq)[None]
    q = np.zeros((batch, hq, hd), np.float32)
    q[..., 0], q[..., 1] = gaps, 1
    codes, scales = key_bounds(k)
    table = np.tile(np.arange(n, dtype=np.int32), (batch, 1))
    out, _ = ops.sparse_paged_attention(dev(q), dev(k), dev(v), dev(codes), dev(scales), dev(table), ints([tokens] * batch),
                                        n, scale=1.0)
    out = out.cpu().numpy()
    group = hq // hkv
    for b in range(batch):
        for h in range(hq):
            ref, _ = plain_attention(q[b, h:h + 1], flat_k[:tokens, h // group], flat_v[:tokens, h // group], 1.0)
            tol = 2 * hd * 2.0 ** -23 * (gaps[b, h] + 2) + (tokens / 8 + 64) * 2.0 ** -23
            if half:
                tol += min(1, 16 * len(sinks) / tokens) * 2.0 ** -50 * np.exp(gaps[b, h] + 2)
            err = np.abs(out[b, h] / ref[0] - 1).max()
            assert err <= tol, (b, h, gaps[b, h], err, tol)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("large", [1e3, 1e6, 1e20])
def test_sparse_attention_query_element_that_dwarfs_the_rest(half, large):
    """A query whose largest element meets keys of 0: scores come from the others, held to 2^-22 of themselves or 2^-32 of
    the largest (fp32 pools: 2^-22).  Tolerance as in check_sparse, with the terms that are added up, and the latter."""
    rng = np.random.default_rng(15)
    hd, page, n = 64, 16, 20
    dt = np.float16 if half else np.float32
    k, v = (rng.standard_normal((n, 1, page, hd)).astype(dt) for _ in range(2))
    k[..., 9] = 0
    q = rng.standard_normal((1, 4, hd)).astype(np.float32)
    codes, scales = key_bounds(k)
    q[..., 9] = large
    out, _ = ops.sparse_paged_attention(dev(q), dev(k), dev(v), dev(codes), dev(scales), ints([list(range(n))]),
                                        ints([n * page]), n)
    kk, vv = k[:, 0].reshape(-1, hd), v[:, 0].reshape(-1, hd)
    ref, mag = plain_attention(q[0], kk, vv, 1 / np.sqrt(hd))
    lost = np.abs(kk.astype(np.float64)).sum(-1).max() / np.sqrt(hd) * np.float64(large) * 2.0 ** -32 if half else 0.0
    tol = np.abs(vv.astype(np.float64)).max() * (2 * hd * 2.0 ** -23 * mag + 2 * lost + (n * page / 8 + 64) * 2.0 ** -23)
    if 2 * lost < 0.5:  # beyond, the weights are anybody's
        assert np.abs(out[0].cpu().numpy() - ref).max() <= tol
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("half", [True, False])
def test_sparse_attention_cuts_lengths_to_max_ctx(half):
    """A length above max_ctx counts as max_ctx, which need not end a page; the tokens behind it are there."""
    rng = np.random.default_rng(14)
    ctx = [200, 100, 99, 640, 7]
    q, k, v, codes, scales, table, d = sparse_case(rng, ctx, 8, 2, 64, 16, half)
    for max_ctx in (0, 1, 15, 16, 100, 109, 333):
        cut = [min(x, max_ctx) for x in ctx]
        for budget in (4, 40):
            out, sel = ops.sparse_paged_attention(dev(q), *d, ints(ctx), budget, max_ctx=max_ctx)
            check_sparse(q, k, v, codes, scales, table, cut, budget, 1, 1, out, sel)


def test_sparse_attention_in_a_captured_graph():
    rng = np.random.default_rng(13)
    ctx = [600, 350]
    q, k, v, codes, scales, table, d = sparse_case(rng, ctx, 8, 2, 128, 16, True)
    qd, cd = dev(q), ints([100, 350])
    out, sel = torch.zeros((2, 8, 128), device="cuda"), torch.zeros((2, 2, 9), dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.sparse_paged_attention(qd, *d, cd, 9, out=out, sel=sel)
    cd.copy_(ints(ctx))
    g.replay()
    check_sparse(q, k, v, codes, scales, table, ctx, 9, 1, 1, out, sel)


# ---------------------------------------------------------------------------------------------------------
# adapters
# ---------------------------------------------------------------------------------------------------------


def lora_case(rng, rows, k, n, rank, adapters, w, run):
    t = getattr(torch, w)
    x = rng.standard_normal((rows, k)).astype(np.float32)
    y = rng.standard_normal((rows, n)).astype(np.float32)
    a = (torch.from_numpy(rng.standard_normal((adapters, rank, k)).astype(np.float32)) / k ** 0.5).to(t)
    b = (torch.from_numpy(rng.standard_normal((adapters, n, rank)).astype(np.float32)) / rank ** 0.5).to(t)
    adapter = rng.integers(-1, adapters + 1, -(-rows // run)).repeat(run)[:rows].astype(np.int32)
    ranks = rng.integers(0, rank + 1, adapters).astype(np.int32)
    ranks[0] = rank
    scales = (rng.random(adapters) * 2 - 0.5).astype(np.float32)
    return x, y, a, b, adapter, ranks, scales


def plain_lora(x, y, a, b, adapter, ranks, scales):
    """(result, size of the products added up), in 64 bits."""
    out, mag = y.astype(np.float64), np.abs(y).astype(np.float64)
    for e in range(len(ranks)):
        at = adapter == e
        r = ranks[e]
        A, B = a[e, :r].double().numpy(), b[e, :, :r].double().numpy()
        xe = x[at].astype(np.float64)
        out[at] += float(scales[e]) * (xe @ A.T) @ B.T
        mag[at] += abs(float(scales[e])) * (np.abs(xe) @ np.abs(A.T)) @ np.abs(B.T)
    return out, mag


@pytest.mark.parametrize("w", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,k,n,rank,adapters,run", [
    (1, 32, 1, 8, 1, 1), (1, 4096, 4096, 16, 2, 1), (3, 96, 77, 24, 2, 1), (64, 768, 2304, 64, 9, 1),
    (17, 2048, 1001, 128, 4, 3), (200, 256, 300, 40, 30, 1), (257, 512, 255, 16, 5, 70), (300, 1024, 640, 64, 40, 1),
    (1000, 768, 768, 8, 3, 333), (513, 4096, 515, 128, 3, 100), (2000, 160, 1030, 32, 7, 11)])
def test_lora(rows, k, n, rank, adapters, run, w):
    """Tolerance, relative to the products added up in each element: (k / 8 + 40) half ulps of fp32 for the two sums (at
    most 8 products between two roundings of a partial sum, truncated in the tensor core, hence whole ulps: 2^-23), and
    2^-21 for the pairs that hold x and t."""
    rng = np.random.default_rng(rows * 3 + rank)
    c = x, y, a, b, adapter, ranks, scales = lora_case(rng, rows, k, n, rank, adapters, w, run)
    want, mag = plain_lora(*c)
    tol = ((k / 8 + 40) * 2.0 ** -23 + 2.0 ** -21) * mag
    d = dev(x), a.cuda(), b.cuda(), dev(adapter)
    kw = dict(ranks=dev(ranks), scales=dev(scales))
    out = ops.lora_add(dev(y), *d, out=torch.full((rows, n), 7.0, device="cuda"), **kw)
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()
    # in place on a slice of a wider, misaligned activation, from a slice of one
    wide = torch.full((rows, n + 5), 3.0, device="cuda")
    wide[:, 1:1 + n] = dev(y)
    xw = torch.zeros((rows, k + 8), device="cuda")
    xw[:, 4:4 + k] = d[0]
    ops.lora_add(wide[:, 1:1 + n], xw[:, 4:4 + k], *d[1:], **kw)
    assert torch.equal(wide[:, 1:1 + n], out)
    assert (wide[:, 0] == 3).all() and (wide[:, 1 + n:] == 3).all()


@pytest.mark.parametrize("rows", [5, 300])
def test_lora_rows_do_not_meet(rows):
    """NaN and infinities of one adapter, of an unused rank, and of one row's input stay where they are."""
    rng = np.random.default_rng(21)
    x, y, a, b, adapter, ranks, scales = lora_case(rng, rows, 64, 50, 16, 4, "float16", 1)
    adapter[:] = np.arange(rows) % 4
    adapter[4] = -1
    ranks[:] = [16, 11, 3, 16]
    for e in (1, 2):  # unused ranks of two adapters
        a[e, ranks[e]:] = float("nan")
        b[e, :, ranks[e]:] = float("inf")
    a[3], x[0, 7] = float("nan"), np.inf
    args = dev(x), a.cuda(), b.cuda(), dev(adapter)
    out = ops.lora_add(dev(y), *args, ranks=dev(ranks), scales=dev(scales)).cpu().numpy()
    bad = (adapter == 3) | (np.arange(rows) == 0)
    assert np.isfinite(out[~bad]).all() and not np.isfinite(out[bad]).any()
    keep = ~bad & (adapter >= 0)
    a[3], x[0] = 0, 0
    want, mag = plain_lora(x, y, a.nan_to_num(0), b.nan_to_num(0, 0, 0), adapter, ranks, scales)
    assert (np.abs(out - want)[keep] <= 1e-5 * mag[keep]).all()
    assert (out[4] == y[4]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_lora_long_sums_have_no_bias(dtype):
    """300 rows (tiles) of x in [1, 2), k 131,072, A in [1, 2), B the identity: an output is one sum over k.  A sum of 32
    columns in the tensor core may lose less than an ulp (2^-23) per addend: two products of 16 and the accumulator (four
    of 8 in fp32), the hi parts' lower terms beside that as little as they are; whatever is rounded to nearest errs to
    either side, by at most 2^-22 in x's terms and 2^-24 in each of 270 additions, whose mean over 2,400 outputs stays
    below 2e-7 (six standard deviations)."""
    rows, k = 300, 131072
    g = torch.Generator(device="cuda").manual_seed(32)
    x = 1 + torch.rand(rows, k, device="cuda", generator=g)
    a = (1 + torch.rand(1, 8, k, device="cuda", generator=g)).to(dtype)
    b = torch.eye(8, device="cuda").to(dtype)[None]
    got = ops.lora_add(torch.zeros(rows, 8, device="cuda"), x, a, b, ints([0] * rows))
    want = x.double() @ a[0].double().t()
    addends = 36 if dtype == torch.float32 else 34
    assert abs(float((got.double() / want - 1).mean())) <= addends * 2.0 ** -23 + 2e-7


@pytest.mark.parametrize("w", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,adapters", [(300, 5), (1500, 600)])
def test_lora_order_of_a_large_batch_does_not_matter(rows, adapters, w):
    """Rows of tiles are sorted by adapter: any order of the batch gives every row the same bits, in place too."""
    rng = np.random.default_rng(23)
    x, y, a, b, adapter, ranks, scales = lora_case(rng, rows, 160, 70, 24, adapters, w, 1)
    d, kw = (a.cuda(), b.cuda()), dict(ranks=dev(ranks), scales=dev(scales))
    out = ops.lora_add(dev(y), dev(x), *d, dev(adapter), **kw).cpu().numpy()
    want, mag = plain_lora(x, y, a, b, adapter, ranks, scales)
    assert (np.abs(out - want) <= 1e-5 * mag).all() and (out[adapter < 0] == y[adapter < 0]).all()
    for order in (np.argsort(adapter, kind="stable"), rng.permutation(rows)):
        place = dev(y[order])
        ops.lora_add(place, dev(x[order]), *d, dev(adapter[order]), out=place, **kw)
        assert (place.cpu().numpy() == out[order]).all()


@pytest.mark.parametrize("w", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows", [7, 300])
@pytest.mark.parametrize("large,at", [(1e3, 5), (1e6, 5), (1e6, 700), (1e9, 1000)])
def test_lora_element_that_dwarfs_the_rest(rows, large, at, w):
    """Rows with an element far above the others, which meets weights of 0, at the row's start or far into it: the others
    are held to 2^-22 of themselves or, with fp16 adapters over many rows, 2^-31 of the row's largest.  Tolerance as in
    test_lora, and the latter through both products."""
    rng = np.random.default_rng(rows + at)
    k, n, rank = 1024, 130, 16
    x, y = rng.standard_normal((rows, k)).astype(np.float32), rng.standard_normal((rows, n)).astype(np.float32)
    a = torch.from_numpy(rng.standard_normal((2, rank, k)).astype(np.float32) / k ** 0.5)
    a[..., at] = 0
    a, b = a.to(getattr(torch, w)), torch.from_numpy(rng.standard_normal((2, n, rank)).astype(np.float32)).to(
        getattr(torch, w))
    adapter = rng.integers(-1, 2, rows)
    x[:, at] = large
    ref, mag = plain_lora(x, y, a, b, adapter, [rank] * 2, [1.0] * 2)
    lost = np.zeros((rows, n))
    if w == "float16" and rows > 256:
        for e in range(2):
            A, B = a[e].double().abs().numpy(), b[e].double().abs().numpy()
            lost[adapter == e] = large * 2.0 ** -31 * (B @ A.sum(-1))
    out = ops.lora_add(dev(y), dev(x), a.cuda(), b.cuda(), ints(adapter)).cpu().numpy()
    assert (np.abs(out - ref) <= ((k / 8 + 40) * 2.0 ** -23 + 2.0 ** -21) * mag + lost).all()


def test_lora_same_rows_alone_and_in_a_batch():
    """A row's bits do not depend on what shares the batch (same form of the kernel)."""
    rng = np.random.default_rng(22)
    x, y, a, b, adapter, ranks, scales = lora_case(rng, 100, 512, 700, 32, 6, "bfloat16", 1)
    d = a.cuda(), b.cuda()
    kw = dict(ranks=dev(ranks), scales=dev(scales))
    out = ops.lora_add(dev(y), dev(x), *d, dev(adapter), **kw)
    for r in (0, 41, 99):
        one = ops.lora_add(dev(y[r:r + 1]), dev(x[r:r + 1]), *d, dev(adapter[r:r + 1]), **kw)
        assert torch.equal(one[0], out[r])


def test_lora_refuse():
    y, x = torch.zeros((2, 40), device="cuda"), torch.zeros((2, 64), device="cuda")
    a, b = torch.zeros((1, 8, 64), device="cuda"), torch.zeros((1, 40, 8), device="cuda")
    ops.lora_add(y, x, a, b, ints([0, 0]))
    for bad in ((y, x[:1], a, b), (y, x, a, b.half()), (y, x, a.double(), b.double()), (y, x, a, b[:, :39]),
                (y.half(), x, a, b), (y.t(), x, a, b), (y, x, a.cpu(), b)):
        with pytest.raises(ZcError):
            ops.lora_add(*bad, ints([0, 0]))


# ---------------------------------------------------------------------------------------------------------
# logits rules
# ---------------------------------------------------------------------------------------------------------


def plain_logits(x, past, past_len, prompt_len, past_rows, rep, freq, pres, bias, mask, mask_rows):
    """(values, magnitude of what was added up) in 64 bits; bias: a list of (ids, values) per row."""
    v, big = x.astype(np.float64), np.abs(x.astype(np.float64))
    rows, vocab = x.shape
    for r in range(rows):
        if past is not None and 0 <= past_rows[r] < len(past):
            h = past[past_rows[r]][:past_len[past_rows[r]]]
            gen = h[prompt_len[past_rows[r]]:]
            ok = h[(h >= 0) & (h < vocab)]
            for t in np.unique(ok):
                v[r, t] = v[r, t] / rep[r] if v[r, t] > 0 else v[r, t] * rep[r]
                c = int((gen == t).sum())
                big[r, t] = max(abs(x[r, t]), abs(v[r, t])) + abs(freq[r]) * c + abs(pres[r])
                if c:
                    v[r, t] -= float(freq[r]) * c + float(pres[r])
        if bias is not None:
            for t, b in zip(*bias[r]):
                if 0 <= t < vocab:
                    v[r, t] += float(b)
                    big[r, t] += abs(float(b))
        if mask is not None and 0 <= mask_rows[r] < len(mask):
            bits = np.unpackbits(mask[mask_rows[r]].view(np.uint8), bitorder="little")[:vocab]
            v[r, bits == 0] = -np.inf
    return v, big


def rules(rng, rows, vocab, cap, n_bias, masks, dup=True):
    past = rng.integers(-2, vocab + 2, (rows + 1, cap)).astype(np.int32)
    past[:, cap // 2:] = past[:, :cap - cap // 2]  # repeats, across the prompt's end
    past_len = rng.integers(0, cap + 1, rows + 1).astype(np.int32)
    past_len[0] = cap
    prompt_len = (past_len * rng.random(rows + 1)).astype(np.int32)
    past_rows = rng.permutation(rows + 1)[:rows].astype(np.int32)
    if rows > 2:
        past_rows[1] = -1
    rep, freq, pres = (rng.random(rows).astype(np.float32) * k + o for k, o in ((0.8, 0.9), (1.0, -0.3), (1.0, -0.2)))
    if rows > 3:
        rep[2], freq[2], pres[2] = 1, 0, 0
    bias = None
    if n_bias:
        bias = []
        for r in range(rows):
            n = 0 if r == rows - 1 and rows > 1 else n_bias
            ids = rng.integers(-1, vocab + 1, n).astype(np.int32)
            if dup and n > 2:
                ids[-1] = ids[0]
                ids[n // 2] = ids[0]
            bias.append((ids, rng.standard_normal(n).astype(np.float32) * 3))
    mask = mask_rows = None
    if masks:
        mask = rng.integers(-2 ** 31, 2 ** 31, (masks, (vocab + 31) // 32 + 1)).astype(np.int32)
        mask[0] = 0  # a state that allows nothing
        mask_rows = rng.integers(-1, masks + 1, rows).astype(np.int32)
        mask_rows[0] = 0 if rows > 1 else masks - 1
    return past, past_len, prompt_len, past_rows, rep, freq, pres, bias, mask, mask_rows


@pytest.mark.parametrize("x_type", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,cap,n_bias,masks", [
    (1, 1, 1, 1, 1), (1, 32000, 700, 0, 2), (2, 31, 5, 3, 2), (5, 1000, 64, 0, 0), (4, 1003, 300, 40, 3),
    (9, 8193, 17, 5, 4), (3, 100003, 4000, 300, 2), (6, 131072, 333, 1, 0)])
def test_logits_rules(rows, vocab, cap, n_bias, masks, x_type):
    """Tolerance: at most 8 fp32 roundings (quotient or product, frequency times count, three sums, the bias sum's two
    more), each half an ulp (2^-24) of no more than the magnitudes added up."""
    rng = np.random.default_rng(rows * 7 + vocab)
    t = getattr(torch, x_type)
    x = (torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)) * 4).to(t)
    x[0, 0] = float("nan")
    x[rows - 1, vocab // 2] = -float("inf")
    a = rules(rng, rows, vocab, cap, n_bias, masks)
    past, past_len, prompt_len, past_rows, rep, freq, pres, bias, mask, mask_rows = a
    with np.errstate(invalid="ignore"):
        want, big = plain_logits(x.double().numpy(), *a)
    kw = dict(past=dev(past), past_len=dev(past_len), prompt_len=dev(prompt_len), past_rows=dev(past_rows),
              repetition=dev(rep), frequency=dev(freq), presence=dev(pres))
    if bias:
        kw.update(bias_start=ints(np.cumsum([0] + [len(b[0]) for b in bias])),
                  bias_ids=dev(np.concatenate([b[0] for b in bias])), bias=dev(np.concatenate([b[1] for b in bias])))
    if masks:
        kw.update(mask=dev(mask), mask_rows=dev(mask_rows))
    tol = 8 * 2.0 ** -24 * np.where(np.isfinite(big), big, 0)

    def near(got):
        got = got.cpu().numpy().astype(np.float64)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        assert (np.abs(got - want)[fine] <= tol[fine]).all()

    first = ops.process_logits(x.cuda(), **kw)
    near(first)
    # a strided input into a strided, misaligned output
    wide = torch.full((rows, 2 * vocab + 3), 5.0, dtype=t, device="cuda")
    wide[:, 1:1 + vocab] = x.cuda()
    out = torch.full((rows, vocab + 3), -1.0, device="cuda")
    ops.process_logits(wide[:, 1:1 + vocab], out=out[:, 2:2 + vocab], **kw)
    assert torch.equal(out[:, 2:2 + vocab].nan_to_num(), first.nan_to_num())
    assert (out[:, :2] == -1).all() and (out[:, 2 + vocab:] == -1).all()
    if t is torch.float32:  # in place
        y = x.cuda()
        assert ops.process_logits(y, **kw) is y
        assert torch.equal(y.nan_to_num(), first.nan_to_num())


def test_logits_without_rules_are_a_copy():
    x = torch.randn((3, 777), device="cuda", dtype=torch.bfloat16)
    assert torch.equal(ops.process_logits(x), x.float())
    y = x.float()
    assert torch.equal(ops.process_logits(y, past=torch.empty((3, 0), dtype=torch.int32, device="cuda"),
                                          past_len=ints([0, 0, 0]), repetition=torch.full((3,), 2.0, device="cuda")),
                       x.float())
    assert ops.process_logits(x[:0]).shape == (0, 777)


def test_logits_refuse():
    x = torch.randn((3, 64), device="cuda")
    with pytest.raises(ZcError):
        ops.process_logits(x, past=ints([[1]]), past_len=ints([1]))  # one history for three rows
    with pytest.raises(ZcError):
        ops.process_logits(x, bias=torch.ones(1, device="cuda"))
    with pytest.raises(ZcError):
        ops.process_logits(x, mask=ints([[1], [1], [1]]))  # 64 tokens need two words
    with pytest.raises(ZcError):
        ops.process_logits(x.double())
    with pytest.raises(ZcError):
        ops.process_logits(x.t())


# ---------------------------------------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------------------------------------


class Step:
    """A small model's serving step over the operators: plan, projection with adapters, append, sparse attention, head,
    rules, greedy token.  Every buffer is kept, so that a captured step replays on changed contents."""

    def __init__(self, rng, batch, tokens, hq=4, hkv=2, hd=64, k=128, vocab=600, page=16, max_pages=12, budget=4):
        self.hq, self.hkv, self.hd, self.page, self.budget, self.vocab = hq, hkv, hd, page, budget, vocab
        n = (hq + 2 * hkv) * hd
        self.host = Pool(rng, batch + 2, max_pages, batch * max_pages, page)
        self.pool = upload(self.host)
        f = lambda *s: dev(rng.standard_normal(s).astype(np.float32))  # noqa: E731
        self.w, self.head = f(n, k) / k ** 0.5, f(vocab, hq * hd) / (hq * hd) ** 0.5
        self.a, self.b = (f(3, 8, k) / k ** 0.5).half(), (f(3, n, 8) / 8 ** 0.5).half()
        self.kv = [torch.zeros((batch * max_pages, hkv, page, hd), dtype=torch.float16, device="cuda") for _ in "kv"]
        self.bounds = torch.zeros((batch * max_pages, hkv, 2, hd), dtype=torch.int8, device="cuda")
        self.scales = torch.zeros((batch * max_pages, hkv), device="cuda")
        self.new, self.rows = ints([0] * batch), ints(rng.permutation(batch + 2)[:batch])
        self.plan = ops.PagePlan.empty(batch, tokens)
        self.x, self.adapter = torch.zeros((tokens, k), device="cuda"), ints([-1] * tokens)
        self.past = torch.zeros((batch + 2, 200), dtype=torch.int32, device="cuda")
        self.past_len = ints([0] * (batch + 2))
        self.rep = torch.full((tokens,), 1.3, device="cuda")
        self.freq, self.pres = torch.full((tokens,), 0.2, device="cuda"), torch.full((tokens,), 0.1, device="cuda")
        self.mask = torch.full((1, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
        self.mask[0, 3] = 0
        self.mask_rows = ints([0] * tokens)

    def __call__(self):
        ops.reserve_pages(*self.pool, self.new, self.page, rows=self.rows, out=self.plan)
        qkv = ops.lora_add(self.x @ self.w.t(), self.x, self.a, self.b, self.adapter)
        q, k, v = qkv.split([self.hq * self.hd, self.hkv * self.hd, self.hkv * self.hd], 1)
        ops.append_kv(k.unflatten(1, (self.hkv, self.hd)), v.unflatten(1, (self.hkv, self.hd)), self.plan.slots,
                      *self.kv, self.bounds, self.scales)
        out, sel = ops.sparse_paged_attention(q.unflatten(1, (self.hq, self.hd)), *self.kv, self.bounds, self.scales,
                                              self.pool[0], self.plan.ctx_len, self.budget,
                                              rows=self.plan.token_rows)
        raw = out.flatten(1) @ self.head.t()
        logits = ops.process_logits(raw, out=torch.empty_like(raw), past=self.past, past_len=self.past_len,
                                    past_rows=self.plan.token_rows, repetition=self.rep, frequency=self.freq,
                                    presence=self.pres, mask=self.mask, mask_rows=self.mask_rows)
        token = ops.LlmSampler.sample(logits.clone(), temperature=0.0, repetition_penalty=1.0)
        return qkv, out, sel, raw, logits, token

    def check(self, got, new, x, adapter):
        """The step's results against the host, stage by stage on the stage's own inputs."""
        qkv, out, sel, raw, logits, token = (t.cpu() for t in got)
        rows = self.rows.tolist()
        want = self.host.reserve(rows, new, len(self.plan.slots))
        same_plan(self.plan, want)
        same_pool(self.host, self.pool)
        y = (dev(x) @ self.w.t()).cpu().numpy()
        ref, mag = plain_lora(x, y, self.a.cpu(), self.b.cpu(), adapter, [8] * 3, [1.0] * 3)
        assert (np.abs(qkv.numpy() - ref) <= (64 * 2.0 ** -23 + 2.0 ** -21) * mag).all()
        kv = [t.cpu().numpy() for t in self.kv]
        cut = self.hq * self.hd, (self.hq + self.hkv) * self.hd
        for t, s in enumerate(want[1]):
            if s >= 0:
                for i, part in enumerate((qkv[t, cut[0]:cut[1]], qkv[t, cut[1]:])):
                    np.testing.assert_array_equal(kv[i][s // self.page, :, s % self.page],
                                                  part.half().numpy().reshape(self.hkv, self.hd))
        codes, scales = self.bounds.cpu().numpy(), self.scales.cpu().numpy()
        for r in rows:
            for c in range(-(-int(self.host.lens[r]) // self.page)):
                p, held = self.host.table[r, c], min(self.page, int(self.host.lens[r]) - c * self.page)
                for have, ref in zip((codes[p], scales[p]), key_bounds(kv[0][p, :, :held])):
                    np.testing.assert_array_equal(have, ref)
        q = qkv[:, :cut[0]].numpy().reshape(-1, self.hq, self.hd)
        check_sparse(q, *kv, codes, scales, self.host.table, want[4], self.budget, 1, 1, out, sel, rows=want[3])
        past = self.past.cpu().numpy(), self.past_len.cpu().numpy()
        zero = np.zeros_like(past[1])
        ref, mag = plain_logits(raw.numpy(), *past, zero, want[3], *(t.cpu().numpy() for t in (
            self.rep, self.freq, self.pres)), None, self.mask.cpu().numpy(), [0] * len(q))
        fine = np.isfinite(ref)
        np.testing.assert_array_equal(np.isfinite(logits.numpy()), fine)
        assert (np.abs(logits.numpy() - ref)[fine] <= 8 * 2.0 ** -24 * mag[fine]).all()
        assert (token.numpy() == logits.numpy().argmax(1)).all()
        return want


@pytest.mark.parametrize("captured", [False, True])
def test_steps_of_a_mixed_batch(captured):
    """Prompts of different lengths, then decode steps of one to three tokens with rejected drafts and finished requests;
    the same steps eagerly and as replays of one captured graph."""
    rng = np.random.default_rng(31)
    batch, tokens = 6, 96
    step = Step(rng, batch, tokens)
    graph = got = None
    if captured:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()  # no request adds a token
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
    plans = [[40, 3, 0, 17, 1, 30]] + [[1, 1, 2, 1, 3, 1], [1] * 6, [16, 1, 0, 1, 1, 20], [1, 3, 70, 2, 1, 0]]
    for i, new in enumerate(plans):
        x = rng.standard_normal((tokens, 128)).astype(np.float32)
        adapter = rng.integers(-1, 3, tokens).astype(np.int32)
        step.x.copy_(dev(x))
        step.adapter.copy_(dev(adapter))
        step.new.copy_(ints(new))
        if captured:
            graph.replay()
        else:
            got = step()
        want = step.check(got, new, x, adapter)
        # the sampled token of each request's last row joins its history
        token = got[-1].tolist()
        for b, r in enumerate(step.rows.tolist()):
            if new[b] and want[5][b]:
                n = int(step.past_len[r])
                step.past[r, n] = token[want[0][b + 1] - 1]
                step.past_len[r] = n + 1
        # two drafts of request 4 are rejected after the second step; request 0 ends after the fourth
        keep = step.host.lens[step.rows.tolist()].copy()
        if i == 1:
            keep[4] -= 2
        if i == 3:
            keep[0] = 0
        ops.trim_pages(*step.pool, ints(keep), step.page, rows=step.rows)
        step.host.trim(step.rows.tolist(), keep)
        same_pool(step.host, step.pool)


def test_documented_step_runs():
    """The step that the integration guide shows, as it stands there: a prompt step and a decode step with padding, checked
    stage by stage on the stage's own inputs."""
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    code = re.search(r"```python\n(.*?)```", text[text.index("## 9. "):], re.S).group(1)
    rng = np.random.default_rng(61)
    f = lambda *s: dev(rng.standard_normal(s).astype(np.float32))  # noqa: E731
    hq, hkv, hd, dim, vocab, T, max_pos = 4, 2, 64, 128, 320, 48, 64
    weight = lambda n, k: ops.QuantizedWeight.upload(8, ops.quantize(8, f(n, k) / k ** 0.5), n, k)  # noqa: E731
    host = Pool(rng, 5, 4, 20, 16)
    angle = np.arange(max_pos)[:, None] * 10000.0 ** (-np.arange(hd // 2) * 2 / hd)
    env = dict(zip(("page_table", "seq_len", "free_pages", "free_count"), upload(host)), rows=ints([4, 1, 2]), T=T, hq=hq,
               hkv=hkv, hd=hd, max_pos=max_pos, cos=dev(np.cos(angle).astype(np.float32)),
               sin=dev(np.sin(angle).astype(np.float32)), w_qkv=weight((hq + 2 * hkv) * hd, dim),
               w_head=weight(vocab, hq * hd), lora_a=f(3, 8, dim) / dim ** 0.5, lora_b=f(3, (hq + 2 * hkv) * hd, 8),
               lora_scale=f(3), k_pool=torch.zeros((20, hkv, 16, hd), dtype=torch.float16, device="cuda"),
               v_pool=torch.zeros((20, hkv, 16, hd), dtype=torch.float16, device="cuda"),
               bounds=torch.zeros((20, hkv, 2, hd), dtype=torch.int8, device="cuda"),
               scales=torch.zeros((20, hkv), device="cuda"), history=dev(rng.integers(0, vocab, (5, 30)), torch.int32),
               history_len=ints([30, 3, 0, 7, 12]), rep=torch.full((T,), 1.2, device="cuda"),
               freq=torch.full((T,), 0.1, device="cuda"), pres=torch.full((T,), 0.1, device="cuda"),
               grammar=torch.full((1, 10), -2, dtype=torch.int32, device="cuda"), state=ints([0] * T))
    for new in ([30, 5, 9], [1, 2, 1]):
        x, adapter = rng.standard_normal((T, dim)).astype(np.float32), rng.integers(-1, 3, T)
        keep = host.lens[[4, 1, 2]] + new
        env.update(x=dev(x), n_new=ints(new), adapter_of_token=ints(adapter), accepted_len=ints(keep))
        exec(code, env)
        want = host.reserve([4, 1, 2], new, T)
        same_plan(env["plan"], want)
        same_pool(host, tuple(env[n] for n in ("page_table", "seq_len", "free_pages", "free_count")))
        dq = env["w_qkv"].qs.double() * env["w_qkv"].d.view(torch.float16).double().repeat_interleave(32, 1)
        y = (env["x"].double() @ dq.t()).cpu().numpy()
        ref, mag = plain_lora(x, y, env["lora_a"].cpu(), env["lora_b"].cpu(), adapter, [8] * 3,
                              env["lora_scale"].tolist())
        # the GEMM rounds each weight to fp16 (2^-11 of it): that much of the sum of the products' sizes
        slack = np.abs(x).astype(np.float64) @ np.abs(dq.cpu().numpy().T) * 2.0 ** -11
        assert (np.abs(env["qkv"].cpu().numpy() - ref) <= (64 * 2.0 ** -23 + 2.0 ** -21) * mag + slack).all()
        z = env["qkv"].double().cpu().numpy().reshape(T, -1, hd)
        a = angle[want[2]][:, None]
        rot = np.stack([z[..., ::2] * np.cos(a) - z[..., 1::2] * np.sin(a),
                        z[..., ::2] * np.sin(a) + z[..., 1::2] * np.cos(a)], -1).reshape(z.shape)
        for name, part in (("q", rot[:, :hq]), ("k", rot[:, hq:hq + hkv]), ("v", z[:, hq + hkv:])):
            assert np.abs(env[name].cpu().numpy() - part).max() <= 4 * 2.0 ** -24 * 1.5 * np.abs(z).max(), name
        kv = [env[n].cpu().numpy() for n in ("k_pool", "v_pool")]
        for t, s in enumerate(want[1]):
            if s >= 0:
                for i, n in enumerate("kv"):
                    np.testing.assert_array_equal(kv[i][s // 16, :, s % 16], env[n][t].half().cpu().numpy())
        check_sparse(env["q"].cpu().numpy(), *kv, env["bounds"].cpu().numpy(), env["scales"].cpu().numpy(), host.table,
                     want[4], 128, 1, 4, env["out"], env["pages"], rows=want[3])
        lg = env["logits"].cpu()
        assert torch.isinf(lg[:, ::32]).all() and torch.isfinite(lg[:, 1:32]).all()
        assert torch.equal(env["token"].cpu().long(), lg.argmax(1))
        host.trim([4, 1, 2], keep)
        same_pool(host, tuple(env[n] for n in ("page_table", "seq_len", "free_pages", "free_count")))


def test_operators_on_two_streams_at_once():
    """Two steps on streams of their own, interleaved call by call, give what each gives alone."""
    def make(seed):
        rng = np.random.default_rng(seed)
        s = Step(rng, 5, 64)
        s.x.copy_(dev(rng.standard_normal((64, 128)).astype(np.float32)))
        s.adapter.copy_(ints(rng.integers(-1, 3, 64)))
        s.new.copy_(ints([20, 1, 7, 30, 3]))
        return s

    alone = [[t.clone() for t in make(seed)()] for seed in (41, 42)]
    both, streams, got = [make(41), make(42)], [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    torch.cuda.synchronize()
    for turn in range(3):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                if turn:  # take the last turn back, so that every turn is the first again
                    ops.trim_pages(*both[i].pool, torch.zeros_like(both[i].new), both[i].page, rows=both[i].rows)
                got[i] = both[i]()
    torch.cuda.synchronize()
    for i in (0, 1):
        for a, b in zip(alone[i], got[i]):
            assert torch.equal(a, b)


def test_calls_from_two_host_threads():
    """Calls whose kernels ask for different amounts of shared memory, from two threads at once: each is taken and gives
    what it gives alone."""
    import ctypes as C
    import threading

    from zeroplatform_b200 import _lib
    L, page, hd = _lib.lib(), 16, 64
    torch.manual_seed(7)

    def sparse(max_ctx):
        n = max_ctx // page
        k = torch.randn((n, 1, page, hd), device="cuda").half()
        codes, scales = (dev(x) for x in key_bounds(k.cpu().numpy()))
        keep = [torch.randn((1, 1, hd), device="cuda"), k, codes, scales,
                torch.arange(n, dtype=torch.int32, device="cuda"), ints([max_ctx]), torch.zeros((1, 1, hd), device="cuda"),
                torch.zeros((1, 1, 8), dtype=torch.int32, device="cuda")]
        q, k, codes, scales, table, ctx, out, sel = (t.data_ptr() for t in keep)

        def call(stream, keep=keep):
            return L.zcu_sparse_paged_attention(q, hd, k, k, 1, codes, scales, table, 1, None, ctx, out, sel, 1, 1, 1, hd,
                                                page, n, n, page * hd, hd, page * hd, 0.125, max_ctx, 8, 1, 1, stream)
        return call, keep[6]

    def logits(vocab):
        x = torch.randn((1, vocab), device="cuda")
        out, rep = torch.zeros_like(x), torch.full((1,), 1.5, device="cuda")
        past, plen = torch.randint(0, vocab, (1, 40000), device="cuda").int(), ints([40000])  # 32-bit counts
        r = _lib.LogitsRules(past=past.data_ptr(), past_len=plen.data_ptr(), past_cap=40000, past_count=1,
                             repetition=rep.data_ptr())

        def call(stream, keep=(x, out, rep, past, plen)):
            return L.zcu_process_logits(x.data_ptr(), 0, vocab, out.data_ptr(), vocab, 1, vocab, C.byref(r), stream)
        return call, out

    for pair in ((sparse(80000), sparse(240000)), (logits(200000), logits(400000))):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        alone = []
        for (call, out), s in zip(pair, streams):
            assert call(s.cuda_stream) == 0
            torch.cuda.synchronize()
            alone.append(out.clone())
        go, bad = threading.Barrier(2), [[], []]

        def work(i):
            go.wait()
            for turn in range(4000):
                rc = pair[i][0](streams[i].cuda_stream)
                if rc:
                    bad[i].append((turn, rc))
                if turn % 500 == 499:
                    streams[i].synchronize()

        threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert bad == [[], []]
        for (_, out), ref in zip(pair, alone):
            assert torch.equal(out, ref)


_TRIM_THREADS = r"""
#include <pthread.h>
#include <stdint.h>
typedef int32_t (*trim_t)(int32_t*, int32_t*, int32_t*, int32_t*, int32_t, int32_t, int32_t, int32_t, const int32_t*,
                          const int32_t*, int32_t, void*);
typedef int32_t (*sync_t)(void*);
typedef struct {
  trim_t trim;
  sync_t sync;
  int32_t* at[5];
  int32_t batch, turns, bad;
  void* stream;
} work;
static void* run(void* p) {
  work* w = (work*)p;
  for (int i = 0; i < w->turns; ++i) {
    w->bad += w->trim(w->at[0], w->at[1], w->at[2], w->at[3], w->batch, 1, 1, 16, 0, w->at[4], w->batch, w->stream) != 0;
    if (i % 256 == 255) w->bad += w->sync(w->stream) != 0;
  }
  return 0;
}
void both(work* w) {
  pthread_t t[2];
  for (int i = 0; i < 2; ++i) pthread_create(&t[i], 0, run, &w[i]);
  for (int i = 0; i < 2; ++i) pthread_join(t[i], 0);
}
"""


def test_calls_from_two_native_threads(tmp_path):
    """The same without Python between the calls: two threads that free sequences of batches of two sizes."""
    import ctypes as C
    import subprocess

    from zeroplatform_b200 import _lib
    (tmp_path / "t.c").write_text(_TRIM_THREADS)
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-pthread", str(tmp_path / "t.c"), "-o", str(tmp_path / "t.so")],
                   check=True)

    class Work(C.Structure):
        _fields_ = [("trim", C.c_void_p), ("sync", C.c_void_p), ("at", C.c_void_p * 5), ("batch", C.c_int32),
                    ("turns", C.c_int32), ("bad", C.c_int32), ("stream", C.c_void_p)]

    sync = C.CFUNCTYPE(C.c_int32, C.c_void_p)(lambda s: torch.cuda.ExternalStream(s).synchronize() or 0)
    streams, work, keep = [torch.cuda.Stream(), torch.cuda.Stream()], (Work * 2)(), []
    for i, batch in enumerate((3000, 10000)):
        pool = [torch.full((batch, 1), -1, dtype=torch.int32, device="cuda"), ints([0] * batch), ints([0]), ints([1]),
                ints([0] * batch)]
        keep.append(pool)
        work[i] = Work(C.cast(_lib.lib().zcu_pages_trim, C.c_void_p), C.cast(sync, C.c_void_p),
                       (C.c_void_p * 5)(*[t.data_ptr() for t in pool]), batch, 8192, 0, streams[i].cuda_stream)
    torch.cuda.synchronize()
    C.CDLL(str(tmp_path / "t.so")).both(work)
    torch.cuda.synchronize()
    assert [w.bad for w in work] == [0, 0]


def test_operators_through_either_binding(monkeypatch):
    """What _dispatch takes and what goes through ctypes (its absence, a stream argument, tensor subclasses) is the same."""
    from zeroplatform_b200 import _lib

    def make():
        rng = np.random.default_rng(51)
        s = Step(rng, 5, 64)
        s.x.copy_(dev(rng.standard_normal((64, 128)).astype(np.float32)))
        s.adapter.copy_(ints(rng.integers(-1, 3, 64)))
        s.new.copy_(ints([20, 1, 7, 30, 3]))
        return s

    assert _lib.dispatch is not None
    ref = [t.clone() for t in make()()]
    x = torch.nn.Parameter(torch.randn((2, 50), device="cuda"), requires_grad=False)
    plain = x.detach().clone()
    assert not _lib.dispatch.process_logits(x, x, *[None] * 12)
    assert torch.equal(ops.process_logits(x.half()), plain.half().float())
    assert torch.equal(ops.process_logits(x), plain)
    assert torch.equal(ops.process_logits(plain.half(), stream=torch.cuda.current_stream()), plain.half().float())
    monkeypatch.setattr(_lib, "dispatch", None)
    for a, b in zip(ref, make()()):
        assert torch.equal(a, b)


def test_numbers_beyond_32_bits_raise():
    """A size whose low 32 bits are a good one is refused by the functions, whichever binding they take."""
    pool = (torch.full((1, 4), -1, dtype=torch.int32, device="cuda"), ints([0]), ints([0, 1, 2, 3]), ints([4]))
    before = [t.clone() for t in pool]
    for page in ((1 << 32) + 16, 16.0, "16"):
        with pytest.raises(ZcError):
            ops.reserve_pages(*pool, ints([3]), page, tokens=3)
        with pytest.raises(ZcError):
            ops.trim_pages(*pool, ints([0]), page)
    k = torch.zeros((4, 1, 16, 64), device="cuda")
    bounds, scales = torch.zeros((4, 1, 2, 64), dtype=torch.int8, device="cuda"), torch.zeros((4, 1), device="cuda")
    args = (torch.zeros((1, 1, 64), device="cuda"), k, k, bounds, scales, pool[0], ints([3]), 2)
    for bad in (dict(sink=(1 << 32) + 1), dict(recent=(1 << 32) + 1), dict(max_ctx=(1 << 32) + 16), dict(sink=1.0)):
        with pytest.raises(ZcError):
            ops.sparse_paged_attention(*args, **bad)
    for a, b in zip(pool, before):
        assert torch.equal(a, b)


def test_dispatch_declines_what_it_must_not_take():
    """Wrong types, shapes, devices, strides and argument counts are declined before anything is enqueued."""
    from zeroplatform_b200 import _lib
    d = _lib.dispatch
    y, x = torch.zeros((2, 40), device="cuda"), torch.ones((2, 64), device="cuda")
    a, b, e = torch.ones((1, 8, 64), device="cuda"), torch.ones((1, 40, 8), device="cuda"), ints([0, 0])
    good = [y, x, a, b, e, None, None, y]
    assert d.lora_add(*good)
    torch.cuda.synchronize()
    before = y.clone()
    wrong = {0: [y.cpu(), y.half(), y[:1], y.t(), y[:, ::2], None, 3], 1: [x.cpu(), x[:, :32], x.double(), y],
             2: [a.cpu(), a.transpose(1, 2), a[0], a.double(), None], 3: [b[:, :39], b.half(), None],
             4: [e.long(), e.cpu(), ints([0]), None], 5: [e, ints([8, 8])], 6: [ints([1])], 7: [y[:1], None, y.cpu()]}
    for i, values in wrong.items():
        for v in values:
            assert not d.lora_add(*good[:i], v, *good[i + 1:]), (i, v)
    assert not d.lora_add(*good[:-1]) and not d.lora_add()
    torch.cuda.synchronize()
    assert torch.equal(y, before)


def test_operators_when_another_device_is_current(monkeypatch):
    """The call goes to the tensors' device, on its current stream, whichever device is current."""
    seen = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: seen.append(1) or -1)
    x = torch.randn((2, 100), device="cuda")
    assert torch.equal(ops.process_logits(x.half()), x.half().float())
    assert seen
    if torch.cuda.device_count() > 1:
        monkeypatch.undo()
        y = torch.randn((2, 100), device="cuda:1", dtype=torch.float16)
        assert torch.cuda.current_device() == 0 and torch.equal(ops.process_logits(y), y.float())
