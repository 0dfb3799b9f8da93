"""The serving operators against plain 64-bit implementations, at the sizes and masks where they can go wrong.

Tolerances.  attend: operands are carried as bf16 limbs to 2^-24 (products of limbs below 2^-26 left out: 2^-24 of the
product for three of them) and products are summed in f32 whose last bit may be cut instead of rounded, so a score is off by
at most
    ds = |scale| sum|q||k| (head_size + 16) 2^-23
and by the rounding of its exponent's argument and of the exponential itself, (|s - max| + 4) 2^-23.  A weight is then off
by a relative dw = ds + ds(max) + (|s - max| + 4) 2^-23, and an output by sum w|v| (2 dw + dp + (keys + 16) 2^-23), with
dp = 2^-23 for limbed weights or 2^-8 for one rounded to bf16 (half a step; the sum of the weights is taken before that),
and half a step of the output's own type.  The logarithm of the sum moves with its scores:
max ds + (max|s - max| + keys + 8) 2^-23 + |lse| 2^-23.
Everything else is equal to the bit: lists, slots, tokens, and a bf16 rounding."""
import numpy as np
import pytest

from ava_b200 import build, engine

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    build.build()
    engine.lib()


@pytest.fixture(scope="module")
def T():
    import torch
    return torch


@pytest.fixture(scope="module")
def S():
    from ava_b200 import serving
    return serving


# ------------------------------------------------------------------------------------------------------------ plan
def plain_plan(cached, fresh, table, owned, stack, page, trim):
    """(table, owned, the stack's contents after the given pages, its height, q_start, slot, pos, row)"""
    table, owned, stack = [list(t) for t in table], list(owned), list(stack)
    need = [-(-(c + f) // page) for c, f in zip(cached, fresh)]
    for r, n in enumerate(need):
        if trim and owned[r] > n:
            stack += table[r][n:owned[r]]
            owned[r] = n
    held = list(stack)
    for r, n in enumerate(need):
        while owned[r] < n:
            table[r][owned[r]] = stack.pop()
            owned[r] += 1
    start, slot, pos, row = [0], [], [], []
    for r, (c, f) in enumerate(zip(cached, fresh)):
        for p in range(c, c + f):
            slot.append(table[r][p // page] * page + p % page)
            pos.append(p)
            row.append(r)
        start.append(start[-1] + f)
    return table, owned, held, len(stack), start, slot, pos, row


def plan_case(rng, rows, page, most_cached, most_fresh, spare=9):
    cached = rng.integers(0, most_cached + 1, rows)
    fresh = rng.integers(0, most_fresh + 1, rows)
    cached[::5] = 0
    fresh[1::4] = 0
    fresh[0] = most_fresh
    if rows > 2:
        cached[2] = fresh[2] = 0
    need = -(-(cached + fresh) // page)
    owned = np.maximum(-(-cached // page) + rng.integers(0, 3, rows), 0)
    width = int(max(need.max(), owned.max())) + 2
    n_pages = int(np.maximum(need, owned).sum()) + spare
    ids = rng.permutation(n_pages)
    table = np.full((rows, width), -1)
    at = 0
    for r in range(rows):
        table[r, :owned[r]] = ids[at:at + owned[r]]
        at += owned[r]
    free = np.full(n_pages, -5)
    free[:n_pages - at] = ids[at:]
    return cached, fresh, table, owned, free, n_pages - at


class Lists:
    """The tensors of a plan call."""

    def __init__(self, T, cached, fresh, table, owned, free, count, tokens):
        i32 = lambda v: T.tensor(np.asarray(v), dtype=T.int32, device="cuda:0")  # noqa: E731
        self.cached, self.fresh, self.table, self.owned, self.free, self.count = i32(cached), i32(fresh), i32(table), i32(owned), i32(free), i32([count])
        self.q_start = i32(np.full(len(cached) + 1, -9))
        self.slot = T.full((tokens,), -9, dtype=T.int64, device="cuda:0")
        self.pos, self.row, self.status = i32(np.full(tokens, -9)), i32(np.full(tokens, -9)), i32([99])

    def call(self, S, page, trim, **kw):
        S.plan(self.cached, self.fresh, self.table, self.owned, self.free, self.count, page, self.q_start, self.slot, pos=self.pos, row=self.row, status=self.status,
               trim=trim, **kw)


def check_plan(x, want, stack_low, tokens):
    table, owned, held, height, start, slot, pos, row = want
    n = len(slot)
    assert x.status.item() == 0
    assert x.owned.tolist() == owned and x.count.item() == height and x.q_start.tolist() == start
    assert x.table.tolist() == table
    assert x.free.tolist()[:len(held)] == held and x.free.tolist()[len(held):] == stack_low[len(held):]
    assert x.slot.tolist() == slot + [-1] * (tokens - n) and x.pos.tolist() == pos + [-1] * (tokens - n) and x.row.tolist() == row + [-1] * (tokens - n)


@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("rows,page,most_cached,most_fresh", [(1, 1, 0, 1), (1, 7, 50, 6000), (2, 16, 40, 1), (33, 16, 500, 4), (256, 64, 3000, 1), (1023, 8, 60, 3),
                                                             (1024, 16, 90, 9), (1025, 3, 40, 20), (2500, 100, 900, 40)])
def test_plan(T, S, rows, page, most_cached, most_fresh, trim):
    rng = np.random.default_rng(rows * 10 + page)
    cached, fresh, table, owned, free, count = plan_case(rng, rows, page, most_cached, most_fresh)
    for extra in (0, 13):
        tokens = int(fresh.sum()) + extra
        x = Lists(T, cached, fresh, table, owned, free, count, tokens)
        x.call(S, page, trim)
        check_plan(x, plain_plan(cached, fresh, table, owned, free[:count].tolist(), page, trim), free.tolist(), tokens)


def test_plan_with_counts_beside_its_inputs_and_no_positions(T, S):
    rng = np.random.default_rng(3)
    cached, fresh, table, owned, free, count = plan_case(rng, 70, 8, 100, 5)
    x = Lists(T, cached, fresh, table, owned, free, count, int(fresh.sum()) + 1)
    owned_out, count_out = T.full_like(x.owned, -3), T.full_like(x.count, -3)
    S.plan(x.cached, x.fresh, x.table, x.owned, x.free, x.count, 8, x.q_start, x.slot, trim=True, owned_out=owned_out, free_count_out=count_out)
    want = plain_plan(cached, fresh, table, owned, free[:count].tolist(), 8, True)
    assert x.owned.tolist() == owned.tolist() and x.count.item() == count
    assert owned_out.tolist() == want[1] and count_out.item() == want[3] and x.slot.tolist() == want[5] + [-1]


def test_plan_takes_what_another_request_gives_in_the_same_step(T, S):
    x = Lists(T, [0, 10, 0], [9, 0, 0], [[-1, -1, -1], [4, 5, 6], [1, 2, 3]], [0, 3, 3], [-5] * 7, 0, 12)
    x.call(S, 4, True)
    check_plan(x, plain_plan([0, 10, 0], [9, 0, 0], [[-1] * 3, [4, 5, 6], [1, 2, 3]], [0, 3, 3], [], 4, True), [-5] * 7, 12)


@pytest.mark.parametrize("tokens", [40, 5000])
@pytest.mark.parametrize("what", ["pages", "table", "negative", "owned", "overflow", "tokens", "stack", "given"])
def test_plan_refuses_as_a_whole(T, S, what, tokens):
    cached, fresh, owned = [10, 3, 0], [4, 5, 1], [3, 1, 0]
    table, free, count = [[0, 1, 2, -1], [3, -1, -1, -1], [-1] * 4], [4, 5, 6, 7, -1, -1, -1, -1], 4
    bit = {"pages": S.NO_PAGES, "table": S.NO_TABLE, "tokens": S.NO_TOKENS}.get(what, S.BAD_LENGTH)
    trim = False
    if what == "pages":
        count = 1
    elif what == "table":
        fresh[1] = 40 if tokens == 5000 else 14
    elif what == "negative":
        fresh[2] = -1
    elif what == "owned":
        owned[0] = 5
    elif what == "overflow":
        cached[0], fresh[0], bit = 2147483647, 4, S.BAD_LENGTH
    elif what == "tokens":
        tokens = 9
    elif what == "stack":
        count = 9
    elif what == "given":
        cached, fresh, count, trim = [0, 0, 0], [0, 0, 0], 6, True     # four given pages on a stack with room for two
    x = Lists(T, cached, fresh, table, owned, free, count, tokens)
    x.call(S, 4, trim)
    assert x.status.item() & bit and x.status.item() & ~(bit | S.NO_PAGES) == 0
    assert x.table.tolist() == table and x.owned.tolist() == owned and x.free.tolist() == free and x.count.item() == count
    assert x.q_start.tolist() == [0] * 4 and set(x.slot.tolist()) == {-1} and set(x.pos.tolist()) == {-1} and set(x.row.tolist()) == {-1}


@pytest.mark.parametrize("tokens", [20, 5000])
def test_plan_reports_a_page_outside_the_store(T, S, tokens):
    x = Lists(T, [0, 4], [6, 2], [[-1, -1], [77, -1]], [0, 1], [3, 9, -1, -1, -1], 2, tokens)
    x.call(S, 4, False)      # 9 and 3 come off the stack; 9 is no page of a store of five; request 1 owns page 77 and takes a third: refused
    assert x.status.item() == S.NO_PAGES
    x = Lists(T, [0, 4], [6, 0], [[-1, -1], [77, -1]], [0, 1], [3, 9, -1, -1, -1], 2, tokens)
    x.call(S, 4, False)
    assert x.status.item() == S.BAD_PAGE
    assert x.slot.tolist()[:7] == [-1] * 4 + [12, 13] + [-1]


def test_plan_replayed_from_a_graph_follows_the_lengths(T, S):
    rng = np.random.default_rng(11)
    cached, fresh, table, owned, free, count = plan_case(rng, 40, 8, 60, 9, spare=200)
    tokens = 600
    x = Lists(T, cached, fresh, table, owned, free, count, tokens)
    stream = T.cuda.Stream()
    with T.cuda.stream(stream):
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g, stream=stream):
            x.call(S, 8, True)
    T.cuda.synchronize()
    assert x.status.item() == 99                       # captured, not run
    state = (table.tolist(), owned.tolist(), free[:count].tolist(), count)
    for step in range(3):
        low = x.free.tolist()
        g.replay()
        T.cuda.synchronize()
        want = plain_plan(cached, fresh, state[0], state[1], state[2], 8, True)
        check_plan(x, want, low, tokens)
        state = (want[0], want[1], want[2][:want[3]], want[3])
        cached = np.where(rng.random(40) < 0.3, 0, cached + fresh)
        fresh = rng.integers(0, 9, 40)
        x.cached.copy_(T.tensor(cached, dtype=T.int32))
        x.fresh.copy_(T.tensor(fresh, dtype=T.int32))


# ---------------------------------------------------------------------------------------------------------- append
def pools(T, rng, layout, pages, heads, page, hs, dtype, fill=None):
    """k and v [pages, heads, places, channels] in one of three layouts."""
    shape = {"heads": (pages, heads, page, hs), "places": (pages, page, heads, hs), "both": (pages, 2, heads, page, hs)}[layout]
    out = []
    for i in range(1 if layout == "both" else 2):
        x = rng.standard_normal(shape, dtype=np.float32) if fill is None else np.full(shape, fill, np.float32)
        out.append(T.tensor(x, device="cuda:0").to(dtype))
    if layout == "both":
        return out[0][:, 0], out[0][:, 1]
    return tuple(x if layout == "heads" else x.transpose(1, 2) for x in out)


@pytest.mark.parametrize("layout", ["heads", "places", "both"])
@pytest.mark.parametrize("dt,tokens,heads,hs,page,packed", [("f32-bf16", 1, 1, 1, 1, False), ("f32-bf16", 37, 3, 64, 16, True), ("f32-f32", 9, 2, 20, 7, True),
                                                            ("bf16-bf16", 300, 5, 128, 24, True), ("bf16-bf16", 11, 2, 33, 8, False), ("f32-bf16", 65, 12, 36, 100, False)])
def test_append(T, S, dt, tokens, heads, hs, page, packed, layout):
    rng = np.random.default_rng(tokens)
    din, dst = ({"f32": T.float32, "bf16": T.bfloat16}[x] for x in dt.split("-"))
    pages = -(-tokens // page) + 2
    kp, vp = pools(T, rng, layout, pages, heads, page, hs, dst)
    if packed:
        qkv = T.tensor(rng.standard_normal((tokens, 3 * heads, hs), dtype=np.float32), device="cuda:0").to(din)
        k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    else:
        k, v = (T.tensor(rng.standard_normal((tokens, heads, hs), dtype=np.float32), device="cuda:0").to(din) for _ in range(2))
    k[0, 0, 0] = float("inf")
    v[-1, -1, -1] = float("nan")
    slot = T.tensor(rng.permutation(pages * page)[:tokens], device="cuda:0")
    if tokens > 4:
        slot[3] = -1
        slot[tokens - 2] = -(2 ** 40)
    want = []
    for x, pool in ((k, kp), (v, vp)):
        y = pool.clone()
        for t, s in enumerate(slot.tolist()):
            if s >= 0:
                y[s // page, :, s % page] = x[t].to(dst)
        want.append(y)
    status = T.zeros(1, dtype=T.int32, device="cuda:0")
    S.append(k, v, slot, kp, vp, status=status)
    for got, y in zip((kp, vp), want):
        assert T.equal(T.nan_to_num(got.float(), 12345.0), T.nan_to_num(y.float(), 12345.0))
    assert status.item() == 0


def test_append_passes_over_slots_outside_the_store(T, S):
    kp, vp = pools(T, np.random.default_rng(0), "heads", 3, 2, 4, 32, T.float32)
    k0, v0 = kp.clone(), vp.clone()
    x = T.ones(4, 2, 32, device="cuda:0")
    status = T.zeros(1, dtype=T.int32, device="cuda:0")
    S.append(x, x, T.tensor([12, 2 ** 33, 2 ** 62, -1], device="cuda:0"), kp, vp, status=status)
    assert status.item() == S.BAD_PAGE and T.equal(kp, k0) and T.equal(vp, v0)
    S.append(x[:0], x[:0], T.zeros(0, dtype=T.int64, device="cuda:0"), kp, vp)
    assert T.equal(kp, k0)


# ---------------------------------------------------------------------------------------------------------- attend
def attend_inputs(T, rng, lengths, heads, kv_heads, hs, page, dt, layout="heads", first=None, spread=1.0, gap=0):
    """lengths: (stored, new) per request.  Everything of the store that no request owns, and the rest of last pages, is NaN."""
    dq, dkv = ({"f32": T.float32, "bf16": T.bfloat16}[x] for x in dt.split("-"))
    need = [-(-(c + f) // page) for c, f in lengths]
    pages = sum(need) + 3
    ids = rng.permutation(pages)
    table = np.full((len(lengths), max(max(need), 1) + 1), -1)
    kp, vp = pools(T, rng, layout, pages, kv_heads, page, hs, dkv, fill=np.nan)
    ks, vs, at = [], [], 0
    for r, (c, f) in enumerate(lengths):
        table[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]
        n = c + f
        k, v = (T.tensor(rng.standard_normal((kv_heads, n, hs), dtype=np.float32), device="cuda:0").to(dkv) for _ in range(2))
        for i in range(need[r]):
            m = min(page, n - i * page)
            kp[int(table[r, i]), :, :m] = k[:, i * page:i * page + m]
            vp[int(table[r, i]), :, :m] = v[:, i * page:i * page + m]
        ks.append(k.double())
        vs.append(v.double())
    tokens = sum(f for _, f in lengths)
    wide = T.tensor(rng.standard_normal((tokens + gap, heads + 1, hs), dtype=np.float32) * spread, device="cuda:0").to(dq)
    q = wide[:, :heads]
    start = np.concatenate([[0], np.cumsum([f for _, f in lengths])])
    i32 = lambda v: T.tensor(np.asarray(v), dtype=T.int32, device="cuda:0")  # noqa: E731
    return dict(q=q, kp=kp, vp=vp, table=i32(table), cached=i32([c for c, _ in lengths]), start=i32(start), first=None if first is None else i32(first), ks=ks, vs=vs,
                lengths=lengths, firsts=first or [0] * len(lengths), dt=dt, fresh=max(f for _, f in lengths))


def call_attend(T, S, x, scale, window=0, max_fresh=None, status=None, room=None):
    out = T.full_like(x["q"], 7.0)
    lse = T.full(x["q"].shape[:2], 7.0, device="cuda:0")
    if room is None:
        room = T.full((S.attend_workspace("cuda:0", x["q"].shape[2]),), 255, dtype=T.uint8, device="cuda:0")
    S.attend(x["q"], x["kp"], x["vp"], x["table"], x["cached"], x["start"], out, max_fresh=x["fresh"] if max_fresh is None else max_fresh, workspace=room, scale=scale,
             window=window, first=x["first"], lse=lse, status=status)
    return out, lse


def check_attend(T, x, out, lse, scale, window=0, only=None):
    f32q = x["dt"].startswith("f32")
    hs, at = x["q"].shape[2], 0
    for r, (c, f) in enumerate(x["lengths"]):
        if f and (only is None or r in only):
            k, v = x["ks"][r], x["vs"][r]
            group = x["q"].shape[1] // k.shape[0]
            q = x["q"][at:at + f].double().transpose(0, 1)
            k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
            s = q @ k.transpose(1, 2) * scale
            pos, key = T.arange(c, c + f, device="cuda:0")[:, None], T.arange(c + f, device="cuda:0")[None]
            seen = (key <= pos) & (key >= x["firsts"][r]) & ((pos - key < window) if window else (key >= 0))
            none = ~seen.any(-1)
            s = s.masked_fill(~seen, -float("inf"))
            top = s.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
            e = T.exp(s - top)
            total = e.sum(-1, keepdim=True)
            w = e / total.clamp(min=1e-300)
            want_lse = T.where(total > 0, top + total.log(), -float("inf"))[..., 0]
            want = w @ v
            ds = abs(scale) * (q.abs() @ k.abs().transpose(1, 2)) * (hs + 16) * 2.0 ** -23
            ds_top = ds.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            dw = ds + ds_top + ((s - top).abs().masked_fill(~seen, 0.0) + 4) * 2.0 ** -23
            dp = 2.0 ** -23 if f32q else 2.0 ** -8
            tol = (w * (2 * dw + dp + (c + f + 16) * 2.0 ** -23)) @ v.abs() + 1e-30
            got = out[at:at + f].double().transpose(0, 1)
            if not f32q:
                tol = tol + (want.abs() + tol) * 2.0 ** -8
            off = (got - want).abs()
            assert T.isfinite(got).all(), (r, "not finite")
            assert (off <= tol).all(), (r, (off / tol).max().item(), off.max().item())
            got_lse = lse[at:at + f].double().transpose(0, 1)
            assert (got[:, none] == 0).all() and T.isneginf(got_lse[:, none]).all()
            span = (s - top).abs().masked_fill(~seen, 0.0).amax(-1)
            tol = ds_top[..., 0] + (span + c + f + 8) * 2.0 ** -23 + want_lse.abs() * 2.0 ** -23
            off = (got_lse - want_lse).abs()[:, ~none]
            assert (off <= tol[:, ~none]).all(), (r, (off / tol[:, ~none]).max().item())
        at += f
    assert (out[at:] == 7).all() and (lse[at:] == 7).all()      # places behind the last sequence stay as they were


TYPES = ["f32-bf16", "bf16-bf16", "f32-f32"]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,page", [(1, 1, 1), (6, 2, 16), (8, 1, 24), (5, 5, 64), (12, 3, 128), (40, 2, 256)])
def test_attend_single_tokens(T, S, dt, hs, heads, kv_heads, page):
    rng = np.random.default_rng(hs + heads + page)
    x = attend_inputs(T, rng, [(0, 1), (15, 1), (16, 1), (63, 1), (0, 0), (200, 1), (129, 1), (7, 0)], heads, kv_heads, hs, page, dt, gap=2)
    out, lse = call_attend(T, S, x, hs ** -0.5)
    check_attend(T, x, out, lse, hs ** -0.5)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads,page,window", [(2, 2, 16, 0), (6, 2, 8, 0), (4, 1, 100, 37), (3, 3, 64, 1), (4, 2, 32, 130), (2, 1, 128, 0), (2, 1, 256, 200)])
def test_attend_chunks(T, S, dt, hs, heads, kv_heads, page, window):
    rng = np.random.default_rng(hs * 7 + heads + page)
    x = attend_inputs(T, rng, [(0, 70), (33, 5), (300, 129), (0, 0), (128, 128), (1, 260), (511, 1)], heads, kv_heads, hs, page, dt, gap=1)
    out, lse = call_attend(T, S, x, hs ** -0.5, window)
    check_attend(T, x, out, lse, hs ** -0.5, window)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("fresh", [2, 9, 33, 150])
def test_attend_behind_left_padding_with_rows_that_see_nothing(T, S, dt, fresh):
    rng = np.random.default_rng(fresh)
    lengths = [(40, fresh), (0, fresh), (100, fresh), (9, fresh), (250, fresh)]
    first = [40, 5, 10 ** 9, 10, -3]      # all stored keys hidden; the first five; everything; one new token; nothing hidden
    x = attend_inputs(T, rng, lengths, 8, 2, 64, 16, dt, first=first)
    for window in (0, 20):
        out, lse = call_attend(T, S, x, 0.125, window)
        check_attend(T, x, out, lse, 0.125, window)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("layout", ["places", "both"])
@pytest.mark.parametrize("hs,fresh", [(64, 3), (128, 200), (32, 90)])
def test_attend_other_layouts_and_scales(T, S, dt, layout, hs, fresh):
    rng = np.random.default_rng(hs + fresh)
    x = attend_inputs(T, rng, [(20, fresh), (0, 1), (77, fresh // 2)], 4, 2, hs, 16, dt, layout=layout)
    for scale in (-0.3, 0.0, 1.0):
        out, lse = call_attend(T, S, x, scale)
        check_attend(T, x, out, lse, scale)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("max_fresh", [0, 1, 64, 100000])
def test_attend_reads_all_whatever_the_host_believed(T, S, dt, max_fresh):
    """max_fresh only chooses the kernel."""
    rng = np.random.default_rng(5)
    x = attend_inputs(T, rng, [(100, 1), (3, 170), (700, 20), (0, 300)], 4, 2, 64, 32, dt)
    out, lse = call_attend(T, S, x, 0.125, max_fresh=max_fresh)
    check_attend(T, x, out, lse, 0.125)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("lengths", [[(30000, 1)], [(9000, 1)] * 3, [(8000, 150), (5, 1)], [(0, 1)] * 1500, [(0, 3000)], [(20, 1)] * 300 + [(20000, 1)]])
def test_attend_long_and_many(T, S, dt, lengths, hs):
    rng = np.random.default_rng(len(lengths))
    x = attend_inputs(T, rng, lengths, 4, 2, hs, 64, dt)
    out, lse = call_attend(T, S, x, hs ** -0.5)
    check_attend(T, x, out, lse, hs ** -0.5)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("fresh", [1, 200])
def test_attend_peaked_and_growing_scores(T, S, dt, fresh):
    """Scores that grow along the keys (the running maximum moves in every tile) and single keys that take all the weight."""
    rng = np.random.default_rng(9)
    x = attend_inputs(T, rng, [(500, fresh), (1000, fresh)], 2, 1, 64, 16, dt)
    for r, (c, f) in enumerate(x["lengths"]):
        n = c + f
        grow = T.linspace(0, 40, n, device="cuda:0")[None, :, None].to(x["kp"].dtype)
        k = x["ks"][r].to(x["kp"].dtype) * 0.05 + grow * 0.25
        x["ks"][r] = k.double()
        for i, page in enumerate(x["table"][r].tolist()):
            if page >= 0:
                m = min(16, n - i * 16)
                x["kp"][page, :, :m] = k[:, i * 16:i * 16 + m]
    x["q"].copy_(x["q"].abs() * 0.5)
    for scale in (0.125, 1.0):
        out, lse = call_attend(T, S, x, scale)
        check_attend(T, x, out, lse, scale)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("fresh", [1, 140])
def test_attend_flags_bad_pages_and_lengths_and_leaves_the_others(T, S, dt, fresh):
    rng = np.random.default_rng(2)
    x = attend_inputs(T, rng, [(50, fresh), (60, fresh), (70, fresh), (10, fresh)], 4, 2, 64, 16, dt)
    status = T.zeros(1, dtype=T.int32, device="cuda:0")
    out, lse = call_attend(T, S, x, 0.125, status=status)
    assert status.item() == 0
    x["table"][1, 2] = 10 ** 6
    x["table"][3, 0] = -4
    out, lse = call_attend(T, S, x, 0.125, status=status)
    assert status.item() == S.BAD_PAGE
    check_attend(T, x, out, lse, 0.125, only=[0, 2])
    status.zero_()
    x["cached"][0] = -5
    x["cached"][2] = 2 ** 31 - 20
    out, lse = call_attend(T, S, x, 0.125, status=status)
    assert status.item() & S.BAD_LENGTH
    x["cached"][:] = T.tensor([50, 60, 70, 10], dtype=T.int32)
    x["table"][1, 2] = x["table"][0, 0]
    x["table"][3, 0] = x["table"][0, 0]
    for bad in ([0, 2 * fresh, fresh, 3 * fresh, 4 * fresh], [-3, fresh, 2 * fresh, 3 * fresh, 4 * fresh], [0, fresh, 2 * fresh, 3 * fresh, 4 * fresh + 99]):
        status.zero_()
        x["start"].copy_(T.tensor(bad, dtype=T.int32))
        out, lse = call_attend(T, S, x, 0.125, status=status)
        assert status.item() & S.BAD_LENGTH, bad


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("fresh", [1, 150])
def test_attend_infinite_and_nan_keys_that_are_hidden_do_not_leak(T, S, dt, fresh):
    rng = np.random.default_rng(4)
    x = attend_inputs(T, rng, [(64, fresh), (40, fresh)], 2, 2, 64, 16, dt, first=[16, 20])
    for r, hidden in ((0, 16), (1, 20)):
        for j in range(hidden):
            page = int(x["table"][r, j // 16])
            x["kp"][page, :, j % 16] = float("nan") if j % 2 else float("inf")
            x["vp"][page, :, j % 16] = float("inf") if j % 3 else float("nan")
    out, lse = call_attend(T, S, x, 0.125)
    check_attend(T, x, out, lse, 0.125)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("fresh,page,window", [(2, 16, 0), (5, 24, 0), (9, 16, 6), (40, 8, 0), (200, 16, 0), (300, 64, 100), (130, 100, 0)])
def test_attend_values_that_are_not_finite_reach_the_rows_that_see_them_only(T, S, dt, hs, fresh, page, window):
    """Infinite and NaN values of single new tokens, of one stored one, and of one in front of the padding: a row that
    sees none of them is the finite row; one that sees them is not finite in that channel, and finite elsewhere."""
    rng = np.random.default_rng(fresh + hs)
    first = [0, 30, 0]
    x = attend_inputs(T, rng, [(70, fresh), (64, fresh), (3, 1)], 4, 2, hs, page, dt, first=first)
    clean = call_attend(T, S, x, 0.125, window)
    check_attend(T, x, *clean, 0.125, window)
    marks = [(0, 70 + fresh - 1, 3, float("nan")), (0, 70 + fresh // 2, 5, float("inf")), (0, 20, 7, -float("inf")), (1, 64 + fresh // 3, hs - 1, float("inf")),
             (1, 29, 9, float("nan"))]
    for r, j, ch, v in marks:
        x["vp"][int(x["table"][r, j // page]), 1, j % page, ch] = v
    out, lse = call_attend(T, S, x, 0.125, window)
    assert T.equal(lse, clean[1])
    at = 0
    for r, (c, f) in enumerate(x["lengths"]):
        pos = T.arange(c, c + f, device="cuda:0")
        bad = T.zeros(f, hs, dtype=T.bool, device="cuda:0")
        for rr, j, ch, v in marks:
            if rr == r and j >= first[r]:
                bad[:, ch] |= (pos >= j) & ((pos - j < window) if window else (pos >= 0))
        o, o0 = out[at:at + f].float(), clean[0][at:at + f].float()
        assert T.equal(o[:, :2], o0[:, :2]), r                       # the other key head
        assert T.isfinite(o[:, 2:][~bad[:, None].expand(-1, 2, -1)]).all(), r
        assert not T.isfinite(o[:, 2:][bad[:, None].expand(-1, 2, -1)]).any(), r
        assert T.equal(o[:, 2:][~bad[:, None].expand(-1, 2, -1)], o0[:, 2:][~bad[:, None].expand(-1, 2, -1)]), r
        at += f


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("fresh,page,hs", [(1, 16, 32), (5, 24, 64), (9, 8, 128), (200, 16, 64)])
def test_attend_the_types_largest_values_in_hidden_places_do_not_leak(T, S, dt, fresh, page, hs):
    """Padding in front of the sequence, and the last new token, which the rows before it do not see."""
    rng = np.random.default_rng(fresh)
    x = attend_inputs(T, rng, [(64, fresh), (40, fresh)], 4, 2, hs, page, dt, first=[16, 21])
    clean = call_attend(T, S, x, 0.125)
    check_attend(T, x, *clean, 0.125)
    big = T.finfo(x["kp"].dtype).max
    for r, hidden in ((0, 16), (1, 21)):
        last = [64, 40][r] + fresh - 1
        for j in list(range(hidden)) + [last] * (fresh > 1):
            at = int(x["table"][r, j // page])
            x["kp"][at, :, j % page] = x["vp"][at, :, j % page] = -big if j % 2 else big
    out, lse = call_attend(T, S, x, 0.125)
    keep = [i for i in range(2 * fresh) if fresh == 1 or i % fresh != fresh - 1]
    assert T.equal(out[keep], clean[0][keep]) and T.equal(lse[keep], clean[1][keep])


@pytest.mark.parametrize("dt,max_fresh", [("f32-bf16", 2), ("f32-bf16", 200), ("bf16-bf16", 200), ("f32-f32", 2)])
def test_attend_more_requests_than_the_line_keeps_sums_for(T, S, dt, max_fresh):
    """Several requests to a sum (more than 2048 of them), many without new tokens, one long one among them; either kernel."""
    rng = np.random.default_rng(8)
    lengths = [(int(rng.integers(0, 40)), int(rng.integers(0, 3)) * int(rng.random() < 0.6)) for _ in range(4500)]
    lengths[3001] = (5000, 130)
    lengths[-1] = (0, 1)
    x = attend_inputs(T, rng, lengths, 2, 1, 64, 16, dt)
    out, lse = call_attend(T, S, x, 0.125, max_fresh=max_fresh)
    check_attend(T, x, out, lse, 0.125, only=set(range(0, 4500, 61)) | {3000, 3001, 3002, 4498, 4499})
    assert T.isfinite(out.float()).all() and not (lse == 7).any()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("hs,fresh", [(32, 1), (64, 2), (64, 150), (128, 70)])
@pytest.mark.parametrize("scale", [0.125, -0.3, 0.0])
def test_attend_queries_and_results_at_odd_addresses(T, S, dt, hs, fresh, scale):
    """Rows that begin at any element and lie any distance apart: the aligned call's results, and nothing between them touched."""
    rng = np.random.default_rng(fresh + hs)
    x = attend_inputs(T, rng, [(70, fresh), (0, fresh), (33, 1)], 4, 2, hs, 16, dt)
    want = call_attend(T, S, x, scale)
    check_attend(T, x, *want, scale)
    q = x["q"]
    shape, strides = q.shape, (4 * (hs + 5) + 3, hs + 5, 1)
    odd = lambda t: T.as_strided(t, shape, strides, 1)  # noqa: E731
    n = shape[0] * strides[0] + 8
    q_room, out_room = T.zeros(n, dtype=q.dtype, device="cuda:0"), T.full((n,), 7.0, dtype=q.dtype, device="cuda:0")
    odd(q_room).copy_(q)
    lse = T.empty_like(want[1])
    room = T.zeros(S.attend_workspace("cuda:0", hs), dtype=T.uint8, device="cuda:0")
    S.attend(odd(q_room), x["kp"], x["vp"], x["table"], x["cached"], x["start"], odd(out_room), max_fresh=fresh, workspace=room, scale=scale, lse=lse)
    assert T.equal(odd(out_room), want[0]) and T.equal(lse, want[1])
    odd(out_room).fill_(7.0)
    assert (out_room == 7).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("fresh", [1, 6, 150])
def test_attend_pages_that_requests_share(T, S, dt, fresh):
    """Two requests behind the same stored pages, and a request whose table names one page over and over."""
    rng = np.random.default_rng(fresh)
    x = attend_inputs(T, rng, [(64, fresh), (64, fresh), (80, fresh)], 8, 2, 64, 16, dt)
    table = x["table"]
    table[1, :4] = table[0, :4]
    table[2, :5] = table[2, 0].clone()
    for which in ("ks", "vs"):
        x[which][1][:, :64] = x[which][0][:, :64]
        for i in range(1, 5):
            x[which][2][:, 16 * i:16 * i + 16] = x[which][2][:, :16]
    out, lse = call_attend(T, S, x, 0.125)
    check_attend(T, x, out, lse, 0.125)


def test_attend_takes_offsets_beyond_32_bits(T, S):
    """Pages that lie more than 2^31 elements into the pools (k and v share one)."""
    rng = np.random.default_rng(6)
    page, hs = 16, 64
    x = attend_inputs(T, rng, [(100, 1), (50, 140)], 2, 2, hs, page, "bf16-bf16")
    n = x["kp"].shape[0]
    stride = 2 ** 31 // 8                        # elements between pages
    big = T.empty((n + 10) * stride, dtype=T.bfloat16, device="cuda:0")
    kp = T.as_strided(big, (n, 2, page, hs), (stride, page * hs, hs, 1))
    vp = T.as_strided(big, (n, 2, page, hs), (stride, page * hs, hs, 1), 2 * page * hs)
    kp.copy_(x["kp"])
    vp.copy_(x["vp"])
    x["kp"], x["vp"] = kp, vp
    out, lse = call_attend(T, S, x, 0.125)
    check_attend(T, x, out, lse, 0.125)
    new = T.ones(2, 2, hs, dtype=T.bfloat16, device="cuda:0")
    S.append(new, 2 * new, T.tensor([(n - 1) * page + 3, -1], device="cuda:0"), kp, vp)
    assert (kp[n - 1, :, 3] == 1).all() and (vp[n - 1, :, 3] == 2).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("fresh", [1, 200])
def test_attend_on_two_streams_and_in_graphs(T, S, dt, fresh):
    rng = np.random.default_rng(8)
    xs = [attend_inputs(T, rng, [(3000, fresh), (100 * (i + 1), fresh), (5, 1)], 4, 2, 64, 64, dt) for i in range(2)]
    rooms = [T.full((S.attend_workspace("cuda:0", 64),), 255, dtype=T.uint8, device="cuda:0") for _ in xs]
    want = [call_attend(T, S, x, 0.125) for x in xs]
    for x, (out, lse) in zip(xs, want):
        check_attend(T, x, out, lse, 0.125)
    streams = [T.cuda.Stream() for _ in xs]
    T.cuda.synchronize()
    got = [None, None]
    for rep in range(3):
        for i, (x, st) in enumerate(zip(xs, streams)):
            with T.cuda.stream(st):
                got[i] = call_attend(T, S, x, 0.125, room=rooms[i])
    T.cuda.synchronize()
    for a, b in zip(want, got):
        assert T.equal(a[0], b[0]) and T.equal(a[1], b[1])       # the same bits on every run
    graphs = []
    for i, x in enumerate(xs):
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g):
            held = call_attend(T, S, x, 0.125, room=rooms[0])     # one workspace for both graphs: replayed one after the other
        graphs.append((g, held))
    for rep in range(2):
        for g, _ in graphs:
            g.replay()
    T.cuda.synchronize()
    for a, (_, b) in zip(want, graphs):
        assert T.equal(a[0], b[0]) and T.equal(a[1], b[1])


# ---------------------------------------------------------------------------------------------------------- verify
def test_calls_from_several_threads_at_once(T, S):
    import threading
    cases = [("f32-bf16", 64, [(300, 1)] * 5), ("bf16-bf16", 128, [(90, 70), (5, 200)]), ("f32-bf16", 64, [(50, 150)]), ("f32-f32", 32, [(200, 3)] * 4)]
    inputs = [attend_inputs(T, np.random.default_rng(i), lengths, 4, 2, hs, 16, dt) for i, (dt, hs, lengths) in enumerate(cases)]
    want = [call_attend(T, S, x, 0.125) for x in inputs]
    T.cuda.synchronize()
    got, errors = [None] * len(cases), []

    def work(i):
        try:
            stream = T.cuda.Stream()
            with T.cuda.stream(stream):
                for _ in range(20):
                    got[i] = call_attend(T, S, inputs[i], 0.125)
                try:
                    S.attend(inputs[i]["q"], inputs[i]["kp"], inputs[i]["vp"], inputs[i]["table"], inputs[i]["cached"], inputs[i]["start"], got[i][0], max_fresh=1,
                             workspace=T.zeros(16, dtype=T.uint8, device="cuda:0"), scale=0.125, window=i)
                    errors.append((i, "not refused"))
                except engine.EngineError as e:                        # each thread has its own error
                    if "workspace" not in str(e):
                        errors.append((i, str(e)))
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for g, w in zip(got, want):
        assert T.equal(g[0], w[0]) and T.equal(g[1], w[1])


def test_a_process_whose_first_call_is_captured():
    import subprocess
    import sys
    code = '''
import torch
from ava_b200 import serving as S
d = "cuda:0"
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=d)
q = torch.randn(70, 4, 64, device=d).bfloat16()
k, v = torch.randn(9, 2, 16, 64, device=d).bfloat16(), torch.randn(9, 2, 16, 64, device=d).bfloat16()
table, cached, start = torch.arange(9, dtype=torch.int32, device=d)[None].contiguous(), i32(60), i32(0, 70)
out, room = torch.zeros_like(q), torch.zeros(S.attend_workspace(d, 64), dtype=torch.uint8, device=d)
call = lambda to: S.attend(q, k, v, table, cached, start, to, max_fresh=70, workspace=room, scale=0.125)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    call(out)
g.replay()
torch.cuda.synchronize()
again = torch.zeros_like(q)
call(again)
assert out.abs().sum() > 0 and torch.equal(out, again)
'''
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]


def plain_verify(p, q, tok, start, u, max_out):
    """In exact order of the definition, f64."""
    out, counts = np.full((len(start) - 1, max_out), -1, np.int64), []
    clean = lambda x: np.where(x > 0, x, 0).astype(np.float64)  # noqa: E731
    for r in range(len(start) - 1):
        a, b = start[r], start[r + 1]
        n = b - a - 1
        if n < 0:
            counts.append(0)
            continue
        kept, final = 0, None
        while kept <= n:
            row = p[a + kept]
            if u is None:
                best = int(np.where(np.isnan(row), -np.inf, row).argmax())
                if kept < n and tok[a + 1 + kept] == best:
                    out[r, kept] = best
                    kept += 1
                    continue
                final = best
                break
            w = clean(row)
            if kept == n:
                final = w
                break
            d = int(tok[a + 1 + kept])
            if 0 <= d < len(w) and u[a + kept] * (1.0 if q is None else clean(q[a + kept])[d]) < w[d]:
                out[r, kept] = d
                kept += 1
                continue
            if q is None:
                final = w.copy()
                if 0 <= d < len(w):
                    final[d] = 0
            else:
                final = np.maximum(w - clean(q[a + kept]), 0)
            if not (0 < final.sum() < np.inf):
                final = w
            break
        if u is not None:
            total = final.sum()
            if 0 < total < np.inf:
                c = np.cumsum(final)
                over = np.nonzero(c > u[b - 1] * c[-1])[0]
                final = int(over[0]) if len(over) else int(np.nonzero(final)[0][-1])
            else:
                final = -1
        out[r, kept] = final
        counts.append(kept + 1)
    return out, counts


def verify_case(rng, rows, vocab, drafts, mode):
    n = [drafts] + [int(rng.integers(0, drafts + 1)) for _ in range(rows - 1)]
    start = np.concatenate([[0], np.cumsum([x + 1 for x in n])])
    if rows > 3:      # a request that fed nothing
        start[3:] -= start[3] - start[2]
    tokens = int(start[-1])
    z = rng.standard_normal((tokens, vocab)) * 2
    soft = lambda x: (np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)).astype(np.float32)  # noqa: E731
    p, q = soft(z), soft(z * 0.8 + 0.4 * rng.standard_normal(z.shape))
    tok = np.zeros(tokens, np.int64)
    for t in range(tokens - 1):
        if mode == "draft":
            tok[t + 1] = rng.choice(vocab, p=q[t].astype(np.float64) / q[t].astype(np.float64).sum())
        else:
            tok[t + 1] = p[t].argmax() if rng.random() < 0.8 else rng.integers(vocab)
    return p, q if mode == "draft" else None, tok, start, None if mode == "greedy" else rng.random(tokens)


def call_verify(T, S, p, q, tok, start, u, max_out, pad=0, offset=0):
    f = lambda x: None if x is None else T.nn.functional.pad(T.tensor(x, device="cuda:0"), (offset, pad))[:, offset:x.shape[1] + offset]  # noqa: E731
    i32 = lambda x: T.tensor(np.asarray(x), dtype=T.int32, device="cuda:0")  # noqa: E731
    rows = len(start) - 1
    out, n_out, status = i32(np.full((rows, max_out), -9)), i32(np.full(rows, -9)), i32([0])
    S.verify_drafts(f(p), i32(tok), i32(start), out, n_out, q=f(q), uniform=None if u is None else T.tensor(u, dtype=T.float64, device="cuda:0"), status=status)
    return out.cpu().numpy(), n_out.tolist(), status.item()


@pytest.mark.parametrize("mode", ["draft", "point", "greedy"])
@pytest.mark.parametrize("rows,vocab,drafts,pad,offset", [(1, 2, 3, 0, 0), (5, 17, 0, 0, 0), (40, 100, 5, 3, 0), (7, 4097, 4, 0, 0), (6, 8193, 40, 2, 1), (3, 16384, 4, 0, 0),
                                                         (200, 50, 7, 2, 2), (2, 70001, 3, 0, 0)])
def test_verify(T, S, mode, rows, vocab, drafts, pad, offset):
    rng = np.random.default_rng(rows + vocab)
    case = verify_case(rng, rows, vocab, drafts, mode)
    out, n, status = call_verify(T, S, *case, drafts + 2, pad, offset)
    want, counts = plain_verify(*case, drafts + 2)
    assert n == counts and np.array_equal(out, want) and status == 0


def test_verify_borders(T, S):
    """Uniform numbers at 0 and just below 1, equal probabilities, drafts of probability 0, a difference without mass."""
    p = np.array([[0.5, 0.5, 0.0, 0.0], [0.0, 0.0, 1.0, 0.0], [0.25, 0.25, 0.25, 0.25]], np.float32)
    last = 1 - 2.0 ** -53
    for tok in ([0, 0, 2], [0, 1, 2], [0, 2, 1], [0, 3, 3]):
        for u in ([0.0, 0.0, 0.0], [last] * 3, [0.5, 0.999, 0.25], [0.0, last, last], [1 - 2.0 ** -24, 0.5, 0.75]):
            for q in (p.copy(), p[[2, 2, 2]], None, np.zeros_like(p)):
                case = (p, q, np.array(tok), [0, 3], np.array(u))
                out, n, status = call_verify(T, S, *case, 3)
                want, counts = plain_verify(*case, 3)
                assert n == counts and np.array_equal(out, want) and status == 0, (tok, u, q)


def test_verify_flags_what_it_cannot_use(T, S):
    p = np.full((4, 8), 0.125, np.float32)
    u = np.array([0.1, 0.2, 0.3, 0.4])
    out, n, status = call_verify(T, S, p, p, np.array([0, 8, 2, 3]), [0, 4], u, 4)
    assert status == S.BAD_TOKEN and n == [1] and out[0].tolist() == [3, -1, -1, -1]         # p - p has no mass: p itself, 0.4 of it
    out, n, status = call_verify(T, S, p, None, np.array([0, 2 ** 31 - 1, 2, 3]), [0, 4], None, 4)
    assert status == S.BAD_TOKEN and n == [1] and out[0].tolist() == [0, -1, -1, -1]
    out, n, status = call_verify(T, S, p, p, np.array([0, 1, 2, 3]), [0, 4], u, 3)             # three drafts, room for two
    assert status == S.BAD_LENGTH and n == [0] and set(out[0].tolist()) == {-1}
    for start in ([0, 5], [-1, 3], [3, 1]):
        out, n, status = call_verify(T, S, p, p, np.array([0, 1, 2, 3]), start, u, 9)
        assert status == S.BAD_LENGTH and n == [0] and set(out[0].tolist()) == {-1}, start
    for x in (0.0, np.nan, -1.0, np.inf):
        bad = np.full((2, 8), x, np.float32)
        out, n, status = call_verify(T, S, bad, None, np.array([0, 1]), [0, 2], np.array([0.5, 0.5]), 2)
        want = [1, -1] if x == np.inf else [-1, -1]                                           # an infinite probability keeps its draft
        assert status == S.NO_MASS and out[0].tolist() == want and n == [len(want) - want.count(-1) + 1]
    out, n, status = call_verify(T, S, np.full((2, 8), np.nan, np.float32), None, np.array([0, 0]), [0, 2], None, 2)
    assert out[0].tolist() == [0, 0] and status == 0


@pytest.mark.parametrize("vocab", [64, 40000])
def test_verify_numbers_outside_their_range_still_draw_a_token_with_mass(T, S, vocab):
    p = np.zeros((1, vocab), np.float32)
    p[0, [vocab // 2, vocab - 3]] = 0.5
    for u, want in ((-0.5, vocab // 2), (-np.inf, vocab // 2), (1.0, vocab - 3), (7.0, vocab - 3), (np.inf, vocab - 3), (np.nan, vocab - 3)):
        for rows in (1, 700):
            out, n, status = call_verify(T, S, np.repeat(p, rows, 0), None, np.zeros(rows), np.arange(rows + 1), np.full(rows, u), 2)
            assert (out == [want, -1]).all() and n == [1] * rows and status == 0, (u, rows)


def test_verify_keeps_the_targets_distribution(T, S):
    """Many independent draws of one draft each: the first token's frequencies are p's, whatever q is."""
    rng = np.random.default_rng(1)
    rows, vocab = 20000, 6
    p1 = np.array([0.4, 0.3, 0.15, 0.1, 0.05, 0.0], np.float32)
    q1 = np.array([0.05, 0.15, 0.2, 0.1, 0.2, 0.3], np.float32)
    p, q = np.tile(p1, (2 * rows, 1)), np.tile(q1, (2 * rows, 1))
    tok = rng.choice(vocab, size=2 * rows, p=q1.astype(np.float64) / q1.astype(np.float64).sum())
    out, n, status = call_verify(T, S, p, q, tok, np.arange(rows + 1) * 2, rng.random(2 * rows), 2)
    share = np.bincount(out[:, 0], minlength=vocab) / rows
    assert np.all(np.abs(share - p1) <= 5 * np.sqrt(p1 * (1 - p1) / rows) + 1e-12) and status == 0   # five standard deviations, seeds fixed


# ---------------------------------------------------------------------------------------------------- used together
@pytest.mark.parametrize("graph", [False, True])
def test_a_drafted_generation_is_the_plain_one(T, S, graph):
    """plan, append, attend and verify as a server runs them: prompts of different lengths, then steps of three drafted
    tokens (some right, some wrong) held greedily against the target; a one-layer model whose logits come from what attend
    read.  The tokens are those of the same model run one token at a time with all keys in one piece, in f64."""
    rng = np.random.default_rng(12)
    V, H, KV, HS, page, rows, want_len, drafts = 50, 4, 2, 64, 8, 5, 24, 3
    emb = rng.standard_normal((V, 3, H, HS)).astype(np.float32)
    emb[:, 1:] = np.repeat(emb[:, 1:, :KV], H // KV, 2)[:, :, :H]
    head = rng.standard_normal((H * HS, V)).astype(np.float32)
    prompts = [rng.integers(0, V, n).tolist() for n in (1, 3, 19, 40, 9)]
    kx, vx = (T.tensor(emb[:, i, ::H // KV]).to(T.bfloat16).double().numpy() for i in (1, 2))

    def plain(seq):
        k, v = kx[seq], vx[seq]
        q = emb[seq[-1], 0].astype(np.float64)
        o = []
        for h in range(H):
            s = k[:, h // (H // KV)] @ q[h] * HS ** -0.5
            w = np.exp(s - s.max())
            o.append(w @ v[:, h // (H // KV)] / w.sum())
        lg = np.concatenate(o) @ head.astype(np.float64)
        top = np.sort(lg)
        return int(lg.argmax()), top[-1] - top[-2]

    seqs, gap = [list(p) for p in prompts], 1e9
    for s in seqs:
        for _ in range(want_len):
            t, g = plain(s)
            s.append(t)
            gap = min(gap, g)
    assert gap > 1e-3        # no tie that rounding could turn

    dev = "cuda:0"
    n_pages, width, cap = 60, 12, 100
    kp, vp = (T.full((n_pages, KV, page, HS), float("nan"), dtype=T.bfloat16, device=dev) for _ in range(2))
    x = Lists(T, [0] * rows, [len(p) for p in prompts], np.full((rows, width), -1), [0] * rows, np.arange(n_pages), n_pages, cap)
    tok = T.zeros(cap, dtype=T.int32, device=dev)
    e = T.tensor(emb, device=dev)
    w = T.tensor(head, device=dev)
    read, lse = T.zeros(cap, H, HS, device=dev), T.zeros(cap, H, device=dev)
    out, n_out = T.zeros(rows, drafts + 1, dtype=T.int32, device=dev), T.zeros(rows, dtype=T.int32, device=dev)
    room = T.zeros(S.attend_workspace(dev, HS), dtype=T.uint8, device=dev)
    status = T.zeros(1, dtype=T.int32, device=dev)
    gathered, logits = T.zeros(cap, 3, H, HS, device=dev), T.zeros(cap, V, device=dev)

    def step(max_fresh):
        x.call(S, page, False)
        gathered.copy_(e[tok.long()])
        S.append(gathered[:, 1, ::H // KV], gathered[:, 2, ::H // KV], x.slot, kp, vp, status=status)
        S.attend(gathered[:, 0], kp, vp, x.table, x.cached, x.q_start, read, max_fresh=max_fresh, workspace=room, scale=HS ** -0.5, lse=lse, status=status)
        logits.copy_(read.view(cap, H * HS) @ w)
        S.verify_drafts(logits, tok, x.q_start, out, n_out, status=status)

    # the prompts: the token behind the last one (every prompt's last row as a run of one token)
    flat = sum(prompts, [])
    tok[:len(flat)] = T.tensor(flat, dtype=T.int32)
    x.call(S, page, False)
    gathered.copy_(e[tok.long()])
    S.append(gathered[:, 1, ::H // KV], gathered[:, 2, ::H // KV], x.slot, kp, vp, status=status)
    S.attend(gathered[:, 0], kp, vp, x.table, x.cached, x.q_start, read, max_fresh=40, workspace=room, scale=HS ** -0.5, lse=lse, status=status)
    first = (read.view(cap, -1) @ w)[x.q_start[1:].long() - 1].argmax(-1).tolist()
    got = [p + [t] for p, t in zip(prompts, first)]
    x.cached += x.fresh
    x.fresh.fill_(drafts + 1)
    g = None
    if graph:
        T.cuda.synchronize()
        side = T.cuda.Stream()
        with T.cuda.stream(side):
            kept = [t.clone() for t in (x.table, x.owned, x.free, x.count)]
            step(drafts + 1)              # once outside, so that libraries are set up
            for t, k in zip((x.table, x.owned, x.free, x.count), kept):
                t.copy_(k)
            status.zero_()
        T.cuda.synchronize()
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g, stream=side):
            step(drafts + 1)
    while min(len(s) - len(p) for s, p in zip(got, prompts)) < want_len:
        feed, most = [], 0
        fresh = []
        for r, s in enumerate(got):
            n = drafts if graph else int(rng.integers(0, drafts + 1))
            truth = (seqs[r] + [0] * 9)[len(s):len(s) + n]
            feed += [s[-1]] + [t if rng.random() < 0.7 else (t + 1) % V for t in truth]
            fresh.append(n + 1)
            most = max(most, n + 1)
        tok[:len(feed)] = T.tensor(feed, dtype=T.int32)
        x.fresh.copy_(T.tensor(fresh, dtype=T.int32))
        if g is not None:
            g.replay()
        else:
            step(most)
        assert x.status.item() == 0 and status.item() == 0
        x.cached += n_out
        for r, (n, row) in enumerate(zip(n_out.tolist(), out.tolist())):
            got[r] += row[:n]
    for r in range(rows):
        assert got[r][:len(seqs[r])] == seqs[r][:len(got[r])], r
    # everyone done: the pages come back
    x.cached.zero_()
    x.fresh.zero_()
    x.call(S, page, True)
    assert x.count.item() == n_pages and sorted(x.free.tolist()) == list(range(n_pages)) and x.owned.tolist() == [0] * rows
