"""Page tables, paged rotary embedding and paged attention against plain 64-bit implementations of the same formulas.

Tolerances, from the roundings alone: a bf16 result is off by at most half a step, 2^-8 of itself; what is held in 32 bits before
that adds a few 2^-24 of the largest summand.  Attention: probabilities that are held in 8 bits (2^-8 of each, so at most 2^-8 of the sum
of their magnitudes times the values') come on top where a request has many rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = 2.0 ** -8


# ------------------------------------------------------------------------------------------------ tables
def plain_step(q_len, length, table, free, n_free, page, rows):
    """the step in Python: (cu_rows, length, n_free, slot, pos, owner, table, status)"""
    r, width, n_pages = len(q_len), len(table[0]), len(free)
    table = [list(x) for x in table]
    need = [-(-(a + b) // page) - -(-b // page) for a, b in zip(q_len, length)]
    flags = (1 if sum(need) > n_free else 0) | (2 if sum(q_len) > rows else 0) | (
        4 if any(a and -(-(a + b) // page) > width for a, b in zip(q_len, length)) else 0)
    if flags:
        return [0] * (r + 1), list(length), n_free, [-1] * rows, [0] * rows, [-1] * rows, table, [flags, sum(need)]
    cu, slot, pos, owner = [0], [], [], []
    top = n_free
    for i in range(r):
        have = -(-length[i] // page)
        for j in range(need[i]):
            top -= 1
            table[i][have + j] = free[top]
        for j in range(q_len[i]):
            p = length[i] + j
            pg = table[i][p // page]
            slot.append(pg * page + p % page if 0 <= pg < n_pages else -1)
            pos.append(p)
            owner.append(i)
        cu.append(cu[-1] + q_len[i])
    pad = rows - len(slot)
    return cu, [a + b for a, b in zip(q_len, length)], top, slot + [-1] * pad, pos + [0] * pad, owner + [-1] * pad, table, [0, sum(need)]


def random_state(seed, requests, page, longest, spare):
    g = torch.Generator().manual_seed(seed)
    length = torch.randint(0, longest + 1, (requests,), generator=g).tolist()
    have = [-(-n // page) for n in length]
    n_pages = sum(have) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    width = longest // page + 40
    table, at = [], 0
    for h in have:
        table.append(order[at:at + h] + [-1] * (width - h))
        at += h
    free = order[at:] + [-7] * at                     # what lies above the top of the stack is nobody's
    return length, table, free, n_pages - at


def on_gpu(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def check_step(q_len, length, table, free, n_free, page, rows, in_place):
    from ixrun_b200.paged import PageStep, page_step

    want = plain_step(q_len, length, table, free, n_free, page, rows)
    gq, gl, gt, gf, gn = on_gpu(q_len), on_gpu(length), on_gpu(table), on_gpu(free), on_gpu([n_free])
    out = PageStep.empty(len(q_len), rows, DEV, length=gl, n_free=gn) if in_place else None
    st = page_step(gq, gl, gt, gf, gn, page, rows, out=out)
    got = (st.cu_rows, st.length, st.n_free, st.slot, st.pos, st.owner, gt, st.status)
    for name, a, b in zip(("cu_rows", "length", "n_free", "slot", "pos", "owner", "table", "status"), got, want):
        assert a.cpu().tolist() == ([b] if name == "n_free" else b), name
    if not in_place:
        assert gl.tolist() == length and gn.tolist() == [n_free]
    assert gf.tolist() == free


@pytest.mark.parametrize("requests,page,longest,new,rows,in_place", [
    (1, 16, 40, 1, 1, False), (1, 16, 0, 0, 0, True), (3, 16, 100, 1, 8, True), (40, 64, 300, 1, 64, True), (7, 32, 500, 70, 600, False),
    (513, 16, 200, 3, 2048, True), (33, 256, 3000, 900, 40000, True), (4096, 128, 700, 2, 9000, False)])
def test_page_step(requests, page, longest, new, rows, in_place):
    length, table, free, n_free = random_state(requests * page, requests, page, longest, requests * (new // page + 2) + 3)
    g = torch.Generator().manual_seed(new)
    q_len = torch.randint(0, new + 1, (requests,), generator=g).tolist()
    if sum(q_len) > rows:
        q_len = [min(q, rows // requests) for q in q_len]
    check_step(q_len, length, table, free, n_free, page, rows, in_place)


@pytest.mark.parametrize("what", ["pages", "rows", "table", "all"])
def test_page_step_that_does_not_fit_takes_nothing(what):
    length, table, free, n_free = random_state(5, 6, 16, 60, 4)
    q_len, rows = [1, 0, 2, 0, 1, 1], 16
    if what in ("pages", "all"):
        q_len[2] = 16 * 5 + 1
        rows = 128
    if what in ("rows", "all"):
        rows = sum(q_len) - 1
    if what in ("table", "all"):
        q_len[4] = 16 * len(table[0])
        free, n_free, rows = free + list(range(100, 200)), n_free, rows if what == "all" else 4000
    for in_place in (False, True):
        check_step(q_len, length, table, free, n_free, 16, rows, in_place)


def test_page_step_with_numbers_that_make_no_sense():
    """negative lengths and counts are zero, a page outside the pool gives no slot, the stack's top is held inside the stack"""
    from ixrun_b200.paged import page_step

    table = on_gpu([[3, 9, -1, -1], [-5, 2, -1, -1], [-1, -1, -1, -1]])
    st = page_step(on_gpu([2, 1, -4]), on_gpu([17, 3, -2]), table, on_gpu([0, 1, 4, 5]), on_gpu([99]), 16, 5)
    assert st.cu_rows.tolist() == [0, 2, 3, 3] and st.length.tolist() == [19, 4, 0] and st.n_free.tolist() == [4]
    assert st.slot.tolist() == [-1, -1, -1, -1, -1] and st.owner.tolist() == [0, 0, 1, -1, -1] and st.status.tolist() == [0, 0]


def test_release_gives_pages_back_and_a_pool_serves_for_good():
    """requests that come and go for many steps: every page is held once or free, never both"""
    from ixrun_b200.paged import PageTables

    g = torch.Generator().manual_seed(3)
    t = PageTables(9, 60, 16, 12, DEV)
    out = t.new_step(128)
    held = [0] * 9
    for step in range(40):
        q = torch.randint(0, 14, (9,), generator=g).tolist()
        q = [min(a, 12 * 16 - n) for a, n in zip(q, held)]
        st = t.step(on_gpu(q), 128, out=out)
        if st.status[0].item() == 0:
            held = [a + n for a, n in zip(q, held)]
        assert t.length.tolist() == held
        done = torch.rand(9, generator=g) < 0.2
        status = t.release(done.to(DEV))
        assert status[0].item() == 0
        held = [0 if d else n for d, n in zip(done.tolist(), held)]
        pages = [p for n, row in zip(held, t.table.tolist()) for p in row[:-(-n // 16)]]
        free = t.free.tolist()[:t.n_free.item()]
        assert sorted(pages + free) == list(range(60)) and t.length.tolist() == held
    # a stack that is full already takes nothing
    t.length.fill_(32)
    before = (t.free.tolist(), t.n_free.tolist())
    t.n_free.fill_(59)
    assert t.release(torch.ones(9, dtype=torch.bool, device=DEV)).tolist() == [4, 18]
    assert t.free.tolist() == before[0] and t.n_free.tolist() == [59] and t.length.tolist() == [32] * 9


# ------------------------------------------------------------------------------------------------ rotary embedding and write
def rope64(x, cos, sin, pos, rot, w, eps):
    """x [rows, heads, D] in 64 bits: norm, rotate-half over the first rot dimensions"""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)


@pytest.mark.parametrize("rows,hq,hkv,d,rot,norm,page,in_place,shift", [
    (1, 1, 1, 64, 64, False, 16, True, 0), (5, 16, 8, 128, 128, False, 64, False, 0), (40, 24, 4, 256, 64, True, 32, False, 0),
    (257, 3, 1, 128, 32, True, 256, True, 0), (9, 7, 7, 64, 64, True, 16, False, 0), (6, 4, 2, 128, 36, True, 16, True, 0),
    (6, 4, 2, 64, 64, False, 16, False, 2), (3, 6, 2, 256, 256, True, 128, True, 0)])
def test_rope_kv_paged(rows, hq, hkv, d, rot, norm, page, in_place, shift):
    """shift: q, k and v start `shift` elements into a row, so nothing is aligned"""
    from ixrun_b200.glue import rope_tables
    from ixrun_b200.paged import rope_kv_paged

    g = torch.Generator(device=DEV).manual_seed(rows * d + rot)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    n_pages = rows // page + 3
    cos, sin = rope_tables(400, rot, 10000.0, DEV)
    x = rnd(rows, (hq + 2 * hkv) * d + 8)[:, shift:shift + (hq + 2 * hkv) * d]
    q, k, v = x[:, :hq * d], x[:, hq * d:(hq + hkv) * d], x[:, (hq + hkv) * d:]
    x0 = x.clone()
    kp, vp = rnd(n_pages, page, hkv, d), rnd(n_pages, 2, page, hkv, d)[:, 1]         # pages of the values lie apart
    kp0, vp0 = kp.clone(), vp.clone()
    slot = torch.randperm(n_pages * page, generator=g, device=DEV)[:rows].int()
    pos = torch.randint(0, 400, (rows,), generator=g, device=DEV).int()
    skipped = torch.zeros(rows, dtype=torch.bool, device=DEV)
    if rows > 4:
        slot[1], slot[3] = -1, n_pages * page
        skipped[1] = skipped[3] = True
    qn, kn = (rnd(d) * 0.1 + 1, rnd(d) * 0.1 + 1) if norm else (None, None)
    out = None if in_place else torch.full((rows, hq * d), 7.0, dtype=torch.bfloat16, device=DEV)
    got = rope_kv_paged(q, k, v, pos, slot, kp, vp, cos, sin, hq, hkv, d, rot_dim=rot, q_norm=qn, k_norm=kn, eps=1e-6, out=out)
    assert got.data_ptr() == (q if in_place else out).data_ptr()
    q0, k0, v0 = x0[:, :hq * d].reshape(rows, hq, d), x0[:, hq * d:(hq + hkv) * d].reshape(rows, hkv, d), x0[:, (hq + hkv) * d:]
    live = ~skipped
    for want, have in ((rope64(q0, cos, sin, pos.long(), rot, qn, 1e-6), got.view(rows, hq, d)),
                       (rope64(k0, cos, sin, pos.long(), rot, kn, 1e-6), None)):
        if have is None:
            have = torch.zeros_like(want)
            have[live] = kp.flatten(0, 1)[slot[live].long()].double()
        # one rounding of the result, and 32-bit arithmetic on terms as large as the pair's (16 operations)
        size = want.abs() + 16 * 2.0 ** -15 * want.abs().amax(-1, keepdim=True)
        assert ((have.double() - want).abs()[live] <= (BF16 * size)[live]).all()
    assert torch.equal(vp.flatten(0, 1)[slot[live].long()], v0.reshape(rows, hkv, d)[live])
    untouched = torch.ones(n_pages * page, dtype=torch.bool, device=DEV)
    untouched[slot[live].long()] = False
    assert torch.equal(kp.flatten(0, 1)[untouched], kp0.flatten(0, 1)[untouched])
    assert torch.equal(vp.flatten(0, 1)[untouched], vp0.flatten(0, 1)[untouched])
    if in_place:
        assert torch.equal(q[skipped], x0[:, :hq * d][skipped])
    else:
        assert (out[skipped] == 7).all() and torch.equal(x, x0)


def test_rope_kv_paged_equals_the_static_cache_without_norms():
    """the same arithmetic as glue.rope_kv where no norm is asked: bit for bit"""
    from ixrun_b200.glue import rope_kv, rope_tables
    from ixrun_b200.paged import rope_kv_paged

    rows, hq, hkv, d = 37, 16, 8, 128
    cos, sin = rope_tables(64, d, 10000.0, DEV)
    q, k, v = (torch.randn(rows, h * d, device=DEV).bfloat16() for h in (hq, hkv, hkv))
    kc, vc = (torch.zeros(64, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kp, vp = (torch.zeros(4, 16, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    at = torch.arange(11, 11 + rows, dtype=torch.int32, device=DEV)
    got = rope_kv_paged(q, k, v, at, at, kp, vp, cos, sin, hq, hkv, d, out=torch.empty_like(q))
    rope_kv(q, k, v, at[:1], kc, vc, cos, sin, hq, hkv, d)
    assert torch.equal(got, q) and torch.equal(kp.flatten(0, 1), kc) and torch.equal(vp.flatten(0, 1), vc)


# ------------------------------------------------------------------------------------------------ attention
def batch(seed, lens, hq, hkv, d, page, pad=0, poison=True, apart=False):
    """lens: (new tokens, tokens in all) of every request; pool rows that belong to nobody are NaN"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    held = [-(-n // page) for _, n in lens]
    n_pages, width = sum(held) + 3, max(held) + 2
    order = torch.randperm(n_pages, generator=g, device=DEV).tolist()
    shape = (n_pages, 2, page, hkv, d) if apart else (2, n_pages, page, hkv, d)
    pool = rnd(*shape)
    kp, vp = (pool[:, 0], pool[:, 1]) if apart else (pool[0], pool[1])
    table, at = [], 0
    dead = torch.ones(n_pages, page, dtype=torch.bool, device=DEV)
    for (_, n), h in zip(lens, held):
        own = order[at:at + h]
        at += h
        # behind the request's pages: numbers outside the pool, of which nothing may be read
        table.append(own + [[-1, n_pages, 2**31 - 1, -2**31][i % 4] for i in range(width - h)])
        for i, p in enumerate(own):
            dead[p, :max(0, min(page, n - i * page))] = False
    if poison:
        kp[dead], vp[dead] = float("nan"), float("nan")
    rows = sum(q for q, _ in lens)
    q = rnd(rows + pad, hq * d + 16)[:, 8:8 + hq * d] * 2
    if pad and poison:
        q[rows:] = float("nan")
    cu = [sum(a for a, _ in lens[:i]) for i in range(len(lens) + 1)]
    return {"q": q, "k_pages": kp, "v_pages": vp, "table": on_gpu(table), "length": on_gpu([n for _, n in lens]), "cu_rows": on_gpu(cu)}


def attn64(s, hq, hkv, d, scale=None):
    """(result, sum of p |v|) in 64 bits; rows that see nothing are zero"""
    q, kp, vp, table = s["q"], s["k_pages"], s["v_pages"], s["table"].tolist()
    rows, g = q.shape[0], hq // hkv
    out = torch.zeros(rows, hkv, g, d, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(out)
    cu, length, page = s["cu_rows"].tolist(), s["length"].tolist(), kp.shape[1]
    for r, n in enumerate(length):
        a, b = cu[r], cu[r + 1]
        if a == b or n <= 0:
            continue
        k, v = (torch.cat([t[p] if 0 <= p < t.shape[0] else torch.zeros_like(t[0]) for p in table[r][:-(-n // page)]])[:n].double() for t in (kp, vp))
        for i in range(a, b):
            see = n - (b - a) + (i - a) + 1
            if see <= 0:
                continue
            x = q[i].double().view(hkv, g, d)
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", x, k[:see]) * (d ** -0.5 if scale is None else scale), -1)
            out[i] = torch.einsum("hgn,nhd->hgd", p, v[:see])
            mag[i] = torch.einsum("hgn,nhd->hgd", p, v[:see].abs())
    return out.view(rows, hq * d), mag.view(rows, hq * d)


def check_attn(s, hq, hkv, d, max_q=None, scale=None, attn=None):
    from ixrun_b200.paged import AttnPaged

    attn = attn or AttnPaged(hq, hkv, d, DEV)
    n = s["cu_rows"][-1].item()
    out = torch.full((s["q"].shape[0], hq * d), 5.0, dtype=torch.bfloat16, device=DEV)
    got = attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"], max_q=max_q, out=out, scale=scale)
    assert got.data_ptr() == out.data_ptr() and (out[n:] == 5).all()
    want, mag = attn64(s, hq, hkv, d, scale)
    # one rounding of the result; probabilities in 8 bits, each off by at most 2^-8 of itself, and the same sum below; 32-bit scores of
    # a few tens: exponents off by some 2^-18
    tol = BF16 * want.abs() + (BF16 + 2.0 ** -14) * mag
    assert torch.isfinite(got[:n]).all()
    assert ((got[:n].double() - want[:n]).abs() <= tol[:n]).all(), ((got[:n].double() - want[:n]).abs() / tol[:n]).max()
    # and on average by far less: the roundings' signs are random
    assert (got[:n].double() - want[:n]).norm() <= 0.75 * BF16 * want[:n].norm() + 1e-12
    again = torch.empty_like(out)
    attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"], max_q=max_q, out=again, scale=scale)
    assert torch.equal(again[:n], got[:n])             # the same bits every time
    words = attn.scratch[:4096].view(torch.int32)
    assert not words.any()
    return got


SINGLES = [[(1, 1)], [(1, 2)], [(1, 15)], [(1, 16), (1, 17)], [(1, 128), (1, 129), (1, 1)], [(1, 1100)], [(1, n) for n in (5, 700, 64, 63, 65, 2000, 1)],
           [(1, 100 + 7 * i) for i in range(50)], [(0, 40), (1, 33), (0, 0), (1, 1), (0, 500)], [(1, 5000)], [(1, 200)] * 301]


@pytest.mark.parametrize("lens", SINGLES, ids=lambda v: f"{len(v)}x{v[0][1]}")
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (6, 1, 64, 64), (12, 2, 256, 32), (3, 3, 128, 256)])
def test_attention_of_single_tokens(lens, hq, hkv, d, page):
    check_attn(batch(len(lens), lens, hq, hkv, d, page, pad=len(lens) % 3), hq, hkv, d, max_q=1)


DRAFTS = [[(2, 2)], [(5, 700)], [(3, 100), (1, 1), (0, 9), (7, 7), (2, 1500)], [(5, 300 + 11 * i) for i in range(16)], [(8, 8)] * 40]


@pytest.mark.parametrize("lens", DRAFTS, ids=lambda v: f"{len(v)}x{v[0][0]}-{v[0][1]}")
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (24, 4, 256, 32), (8, 8, 64, 128), (20, 1, 128, 64)])
def test_attention_of_drafts(lens, hq, hkv, d, page):
    check_attn(batch(len(lens), lens, hq, hkv, d, page, pad=2, apart=True), hq, hkv, d, max_q=8)


CHUNKS = [[(17, 17)], [(64, 64)], [(128, 128)], [(129, 400)], [(300, 300)], [(256, 1000), (1, 700)], [(40, 41), (333, 333), (1, 5), (0, 3), (90, 1200)]]


@pytest.mark.parametrize("lens", CHUNKS, ids=lambda v: f"{len(v)}x{v[0][0]}-{v[0][1]}")
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (6, 2, 256, 64), (5, 1, 64, 32), (4, 4, 128, 256), (7, 1, 128, 128)])
def test_attention_of_chunks(lens, hq, hkv, d, page):
    check_attn(batch(len(lens), lens, hq, hkv, d, page, pad=5), hq, hkv, d)


@pytest.mark.parametrize("max_q", [1, 3, 1000])
def test_attention_does_not_need_max_q_to_be_true(max_q):
    s = batch(4, [(1, 90), (33, 150), (6, 6), (200, 260)], 8, 2, 128, 16)
    check_attn(s, 8, 2, 128, max_q=max_q)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [3, 70])
def test_rows_that_see_nothing_are_zero(d, new):
    """more new tokens than the request has: the first rows sit at negative positions"""
    s = batch(1, [(new, new), (new, new + 9)], 4, 2, d, 16)
    s["length"] = on_gpu([new - 2, 0])
    s["k_pages"], s["v_pages"] = torch.nan_to_num(s["k_pages"]), torch.nan_to_num(s["v_pages"])
    got = check_attn(s, 4, 2, d)
    assert (got[:2] == 0).all() and (got[new:] == 0).all() and (got[2:new] != 0).any()


@pytest.mark.parametrize("new", [1, 4, 90])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_pages_outside_the_pool_are_zeros(new, d):
    s = batch(2, [(new, 200), (new, 130)], 4, 2, d, 32)
    s["table"][0, 2], s["table"][1, 0], s["table"][0, 4] = -1, s["k_pages"].shape[0], 2**31 - 1
    s["k_pages"], s["v_pages"] = torch.nan_to_num(s["k_pages"]), torch.nan_to_num(s["v_pages"])
    check_attn(s, 4, 2, d)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("new,total", [(1, 200), (5, 5), (5, 300), (140, 140), (60, 500)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_is_not_finite_reaches_the_rows_that_see_it_and_no_other(value, new, total, d):
    """a value that is not finite at a late position, and a key that is NaN at the last one"""
    hq, hkv = 4, 2
    s = batch(3, [(new, total), (1, 77)], hq, hkv, d, 16, poison=False)
    at = max(0, total - 2)
    page, row = s["table"][0, at // 16].item(), at % 16
    s["v_pages"][page, row, 1, 3] = value
    last = total - 1
    if new > 1:
        s["k_pages"][s["table"][0, last // 16].item(), last % 16, 0, 0] = float("nan")
    from ixrun_b200.paged import AttnPaged

    got = AttnPaged(hq, hkv, d, DEV)(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"]).double()
    want, mag = attn64(s, hq, hkv, d)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    assert ((got - want).abs()[fine] <= (BF16 * want.abs() + (BF16 + 2.0 ** -14) * mag.nan_to_num(0, 0, 0))[fine]).all()


def test_scores_of_any_size_and_a_scale_of_ones_own():
    for mul, scale in ((40.0, None), (0.01, None), (1.0, 0.3)):
        for lens in ([(1, 900), (4, 90)], [(130, 300)]):
            s = batch(6, lens, 4, 2, 128, 16)
            s["q"] = s["q"] * mul
            n = s["cu_rows"][-1].item()
            from ixrun_b200.paged import AttnPaged

            got = AttnPaged(4, 2, 128, DEV)(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"], scale=scale)
            want, mag = attn64(s, 4, 2, 128, scale)
            # scores of up to some 1500 in 32 bits: exponents off by 1500 * 2^-21
            assert ((got[:n].double() - want[:n]).abs() <= (BF16 * want.abs() + (BF16 + 2.0 ** -9) * mag)[:n]).all()


def test_a_long_cache_passes_32_bits():
    """element offsets behind 2^32, in a pool of nine gigabytes whose used pages lie at its end"""
    hq, hkv, d, page = 4, 2, 128, 256
    s = batch(7, [(1, 700), (90, 300)], hq, hkv, d, page, poison=False)
    n = s["k_pages"].shape[0]
    far = (2**32 // (page * hkv * d)) + 5
    for name in ("k_pages", "v_pages"):
        big = torch.empty(far + n, page, hkv, d, dtype=torch.bfloat16, device=DEV)
        big[far:] = s[name]
        s[name] = big
    s["table"] = torch.where((s["table"] >= 0) & (s["table"] < n), s["table"] + far, -1)
    check_attn(s, hq, hkv, d)


def test_one_object_serves_steps_of_all_kinds_in_turn_and_in_a_graph():
    from ixrun_b200.paged import AttnPaged

    hq, hkv, d = 16, 8, 128
    attn = AttnPaged(hq, hkv, d, DEV)
    cases = [batch(i, lens, hq, hkv, d, 16) for i, lens in enumerate(([(1, 900)], [(200, 700), (1, 50)], [(1, 100)] * 40, [(5, 60), (64, 64)]))]
    want = [check_attn(s, hq, hkv, d, attn=attn) for s in cases]
    outs = [torch.empty_like(w) for w in want]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for s, o in zip(cases, outs):
            attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"], out=o)
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for s, o, w in zip(cases, outs, want):
            n = s["cu_rows"][-1].item()
            assert torch.equal(o[:n], w[:n])
    # the lengths of a captured step may change between replays
    s = cases[0]
    s["length"].fill_(333)
    graph.replay()
    ref, mag = attn64(s, hq, hkv, d)
    assert ((outs[0].double() - ref).abs() <= BF16 * ref.abs() + 2.0 ** -10 * mag).all()


def test_dependent_launches_give_the_same_bits():
    from ixrun_b200.p6 import set_pdl
    from ixrun_b200.paged import AttnPaged

    hq, hkv, d = 8, 4, 128
    attn = AttnPaged(hq, hkv, d, DEV)
    cases = [batch(i, lens, hq, hkv, d, 32) for i, lens in enumerate(([(1, 3000)] * 3, [(200, 900), (1, 50)], [(1, 10)] * 40))]
    want = [check_attn(s, hq, hkv, d, attn=attn) for s in cases]
    prev = set_pdl(True)
    try:
        for _ in range(10):
            got = [attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"]) for s in cases]
            for w, o in zip(want, got):
                assert torch.equal(o, w)
    finally:
        set_pdl(prev)


def test_another_stream_and_two_objects_at_once():
    from ixrun_b200.paged import AttnPaged

    hq, hkv, d = 16, 8, 128
    cases = [batch(i, [(1, 2000 + 100 * i)] * 5, hq, hkv, d, 64) for i in range(2)]
    objects = [AttnPaged(hq, hkv, d, DEV) for _ in range(2)]
    want = [check_attn(s, hq, hkv, d, max_q=1, attn=a) for s, a in zip(cases, objects)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                s = cases[i]
                got[i].append(objects[i](s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"], max_q=1))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)


def test_table_write_and_attention_together():
    """prompts in chunks and single tokens over a shared pool against attention over each request's own keys"""
    from ixrun_b200.glue import rope_tables
    from ixrun_b200.paged import AttnPaged, PageTables, rope_kv_paged

    hq, hkv, d, page, width = 4, 2, 64, 16, 20
    g = torch.Generator(device=DEV).manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    cos, sin = rope_tables(page * width, d, 10000.0, DEV)
    t = PageTables(3, 40, page, width, DEV)
    kp, vp = (torch.full((40, page, hkv, d), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    attn = AttnPaged(hq, hkv, d, DEV)
    keys, values = [[], [], []], [[], [], []]
    for q_len in ([50, 0, 7], [33, 1, 1], [1, 100, 1], [1, 1, 1], [0, 1, 30], [1, 0, 1]):
        rows = sum(q_len) + 3
        st = t.step(on_gpu(q_len), rows)
        x = rnd(rows, (hq + 2 * hkv) * d)
        x0 = x.clone()
        q, k, v = x[:, :hq * d], x[:, hq * d:(hq + hkv) * d], x[:, (hq + hkv) * d:]
        rope_kv_paged(q, k, v, st.pos, st.slot, kp, vp, cos, sin, hq, hkv, d)
        out = attn(q, kp, vp, t.table, st.length, st.cu_rows)
        cu, pos = st.cu_rows.tolist(), st.pos.long()
        qr = rope64(x0[:, :hq * d].reshape(rows, hq, d), cos, sin, pos, d, None, 0)
        kr = rope64(x0[:, hq * d:(hq + hkv) * d].reshape(rows, hkv, d), cos, sin, pos, d, None, 0)
        for r in range(3):
            a, b = cu[r], cu[r + 1]
            if a == b:
                continue
            keys[r].append(kr[a:b].bfloat16().double())
            values[r].append(x0[a:b, (hq + hkv) * d:].reshape(b - a, hkv, d).double())
            kk, vv = torch.cat(keys[r]), torch.cat(values[r])
            n = kk.shape[0]
            assert n == st.length[r].item()
            for i in range(a, b):
                see = n - (b - i) + 1
                p = torch.softmax(torch.einsum("hgd,nhd->hgn", qr[i].bfloat16().double().view(hkv, 2, d), kk[:see]) * d ** -0.5, -1)
                want, mag = (torch.einsum("hgn,nhd->hgd", p, w).reshape(-1) for w in (vv[:see], vv[:see].abs()))
                # a rotated element may fall to the other side of a rounding border: one step of it in a score of a few units
                assert ((out[i].double() - want).abs() <= BF16 * want.abs() + 4 * BF16 * mag).all()


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (8, 8, 64, 64), (12, 2, 256, 32)])
def test_pairs_about_the_length_up_to_which_they_are_not_cut(hq, hkv, d, page):
    """256 KB of a KV head's keys and values: 512 positions of 128 dimensions, 1024 of 64, 256 of 256; shorter and longer requests in
    every order, few and many of them"""
    edge = 65536 // d
    near = [edge - 1, edge, edge + 1, edge + 128, 2 * edge, 2 * edge + 1, 3, 128, 129, 1]
    for seed, lens in enumerate(([(1, edge + 1)], [(1, n) for n in near], [(1, n) for n in reversed(near)], [(1, near[7 * i % 10]) for i in range(70)],
                                 [(1, 9 * edge), (1, 2), (1, edge), (0, 40), (1, 9 * edge + 5), (1, 17)])):
        check_attn(batch(seed, lens, hq, hkv, d, page), hq, hkv, d, max_q=1)


@pytest.mark.parametrize("lens,hq,hkv,d,max_q", [
    ([(1, 1 + i % 37) for i in range(4096)], 4, 2, 64, 1),                     # as many requests as there may be
    ([(1 if i % 9 else 12, 12 + i % 37) for i in range(2000)], 4, 2, 64, None),
    ([(0, 5)] * 4000 + [(70, 90)] + [(0, 0)] * 95, 4, 2, 128, None),
    ([(1, 300), (1, 7), (3, 140)], 256, 1, 64, None),                          # more query heads of a KV head than rows of a tile
    ([(1, 300)], 130, 1, 64, 1),
    ([(2, 300), (1, 9)], 33, 1, 256, None),
    ([(129, 129)] * 30, 2, 1, 128, None),                                      # units with one row in their second tile
    ([(1000, 1100), (1000, 1000)], 3, 3, 256, None),
], ids=lambda v: f"{len(v)}x{v[-1][0]}" if isinstance(v, list) else None)
def test_many_requests_and_large_groups(lens, hq, hkv, d, max_q):
    check_attn(batch(1, lens, hq, hkv, d, 16), hq, hkv, d, max_q=max_q)


@pytest.mark.parametrize("requests,rows", [(1, 0), (1, 1), (4096, 0), (4096, 5000)])
def test_tables_of_one_page_and_steps_without_rows(requests, rows):
    from ixrun_b200.paged import PageTables

    t = PageTables(requests, 5000, 16, 1, DEV)
    st = t.step(on_gpu([0] * requests), rows)
    assert st.status.tolist() == [0, 0] and (st.slot == -1).all() and (st.cu_rows == 0).all()
    if rows:
        st = t.step(on_gpu([1] * requests), rows)
        assert st.status.tolist() == [0, requests] and st.owner[:requests].tolist() == list(range(requests)) and (st.owner[requests:] == -1).all()
        assert t.n_free.item() == 5000 - requests and len(set(st.slot[:requests].tolist())) == requests


def test_captured_steps_of_changing_requests():
    """tables, write and attention of a step as one graph of dependent launches, with chunks and single tokens side by side and other
    numbers of new tokens at every replay: the bits of the same calls made one by one"""
    from ixrun_b200.p6 import set_pdl
    from ixrun_b200.paged import AttnPaged, PageStep, page_step, rope_kv_paged

    hq, hkv, d, page, requests, rows, n_pages, width = 16, 8, 64, 16, 9, 400, 400, 60
    g = torch.Generator(device=DEV).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    ang = torch.arange(width * page, device=DEV)[:, None] * 10000.0 ** (-torch.arange(d // 2, device=DEV) / (d // 2))
    cos, sin = ang.cos(), ang.sin()
    qkv = rnd(rows, (hq + 2 * hkv) * d)
    steps = [[1, 300, 0, 5, 1, 17, 1, 1, 40], [1] * requests, [200, 1, 1, 1, 150, 1, 0, 1, 20], [0, 0, 1, 0, 0, 0, 0, 0, 0], [3, 1, 1, 2, 1, 1, 90, 1, 1]]

    def new():
        st = PageStep.empty(requests, rows, DEV)
        state = {"length": torch.zeros(requests, dtype=torch.int32, device=DEV), "table": torch.full((requests, width), -1, dtype=torch.int32, device=DEV),
                 "free": torch.arange(n_pages, dtype=torch.int32, device=DEV), "n_free": on_gpu([n_pages]), "q_len": on_gpu([0] * requests),
                 "k": torch.zeros(n_pages, page, hkv, d, dtype=torch.bfloat16, device=DEV), "out": torch.zeros(rows, hq * d, dtype=torch.bfloat16, device=DEV)}
        state["v"] = torch.zeros_like(state["k"])
        state["step"] = st._replace(length=state["length"], n_free=state["n_free"])
        state["attn"] = AttnPaged(hq, hkv, d, DEV)
        state["q"] = torch.zeros(rows, hq * d, dtype=torch.bfloat16, device=DEV)
        return state

    def once(s, wait):
        q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        page_step(s["q_len"], s["length"], s["table"], s["free"], s["n_free"], page, rows, out=s["step"])
        wait()
        rope_kv_paged(q, k, v, s["step"].pos, s["step"].slot, s["k"], s["v"], cos, sin, hq, hkv, d, out=s["q"])
        wait()
        s["attn"](s["q"], s["k"], s["v"], s["table"], s["length"], s["step"].cu_rows, out=s["out"])
        wait()

    plain, fast = new(), new()
    prev = set_pdl(True)
    try:
        once(fast, lambda: None)                       # (nothing new: no row)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            once(fast, lambda: None)
        for i in range(20):
            n_new = on_gpu(steps[i % len(steps)] if i < 12 else [1] * requests)
            fast["q_len"].copy_(n_new)
            graph.replay()
    finally:
        torch.cuda.synchronize()
        set_pdl(prev)
    got = {n: fast[n].clone() for n in ("length", "n_free", "k", "v", "out")}
    for i in range(20):
        plain["q_len"].copy_(on_gpu(steps[i % len(steps)] if i < 12 else [1] * requests))
        once(plain, torch.cuda.synchronize)
        assert plain["step"].status[0].item() == 0
    for n, t in got.items():
        assert torch.equal(t, plain[n]), n
    assert got["out"].float().abs().sum() > 0


def test_refusals():
    from ixrun_b200 import _lib
    from ixrun_b200.paged import AttnPaged, PageStep, PageTables, page_release, page_step, rope_kv_paged

    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    ok = dict(q_len=i(2), length=i(2), table=i(2, 3), free=i(4), n_free=i(1), page=16, rows=5)
    page_step(**ok)
    for bad in (dict(page=24), dict(q_len=i(2).long()), dict(q_len=i(3)), dict(table=i(2, 6)[:, ::2]), dict(free=torch.zeros(4, dtype=torch.int32)),
                dict(n_free=i(2)), dict(rows=-1), dict(out=PageStep.empty(2, 4, DEV)), dict(q_len=i(0), length=i(0), table=i(0, 3)), dict(length=i(2).cpu())):
        with pytest.raises(ValueError):
            page_step(**{**ok, **bad})
    with pytest.raises(ValueError):
        page_release(i(2), i(2), i(2, 3), i(4), i(1), 16)
    for args in ((0, 4, 16, 3), (5000, 4, 16, 3), (2, 0, 16, 3), (2, 4, 8, 3), (2, 2**28, 16, 3)):
        with pytest.raises(ValueError):
            PageTables(*args, DEV)
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    f = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    ok = dict(q=b(3, 256), k=b(3, 128), v=b(3, 128), pos=i(3), slot=i(3), k_pages=b(4, 16, 2, 64), v_pages=b(4, 16, 2, 64), cos=f(9, 32), sin=f(9, 32),
              hq=4, hkv=2, head_dim=64)
    rope_kv_paged(**ok)
    for bad in (dict(q=b(3, 128)), dict(k=b(3, 64)), dict(v=b(2, 128)), dict(pos=i(2)), dict(slot=i(3).long()), dict(k_pages=b(4, 16, 2, 32)),
                dict(v_pages=b(5, 16, 2, 64)), dict(cos=f(9, 16)), dict(sin=f(8, 32)), dict(rot_dim=32), dict(q_norm=b(32)), dict(out=b(3, 128)),
                dict(q=f(3, 256)), dict(k_pages=b(4, 32, 2, 64)[:, ::2]), dict(pos=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            rope_kv_paged(**{**ok, **bad})
    for args in ((3, 2, 64), (4, 2, 96), (0, 1, 64)):
        with pytest.raises(ValueError):
            AttnPaged(*args, DEV)
    with pytest.raises(ValueError):
        AttnPaged(4, 2, 64, "cpu")
    attn = AttnPaged(4, 2, 64, DEV)
    ok = dict(q=b(3, 256), k_pages=b(4, 16, 2, 64), v_pages=b(4, 16, 2, 64), table=i(2, 2), length=i(2), cu_rows=i(3))
    attn(**ok)
    for bad in (dict(q=b(3, 192)), dict(q=f(3, 256)), dict(k_pages=b(3, 16, 2, 64)), dict(table=i(3, 2)), dict(length=i(2).long()), dict(cu_rows=i(2)),
                dict(max_q=0), dict(out=b(2, 256)), dict(v_pages=b(4, 16, 2, 64).cpu()), dict(q=b(3, 256).t())):
        with pytest.raises(ValueError):
            attn(**{**ok, **bad})
    for bad in (dict(q=b(3, 260)[:, :256]), dict(q=b(3, 264)[:, 4:260])):
        with pytest.raises(_lib.IxbError):                          # rows of q that do not start on 16 bytes
            attn(**{**ok, **bad})


def test_rope_kv_paged_refuses_an_output_of_other_columns():
    from ixrun_b200.paged import rope_kv_paged

    hq, hkv, d = 4, 2, 64
    q, k, v = (torch.ones(3, n * d, dtype=torch.bfloat16, device=DEV) for n in (hq + 1, hkv, hkv))
    pool = torch.zeros(2, 16, hkv, d, dtype=torch.bfloat16, device=DEV)
    cos = torch.ones(9, d // 2, device=DEV)
    args = (k, v, on_gpu([0, 1, 2]), on_gpu([0, 1, 2]), pool, pool.clone(), cos, cos, hq, hkv, d)
    for columns in (hq - 1, hq + 1):
        with pytest.raises(ValueError):
            rope_kv_paged(q, *args, out=torch.zeros(3, columns * d, dtype=torch.bfloat16, device=DEV))
    assert (pool == 0).all()
    assert rope_kv_paged(q, *args) is q                # in place, in the first columns
    # 1 * 1 - 1 * 1 and 1 * 1 + 1 * 1
    assert (q[:, hq * d:] == 1).all() and (pool[0, :3, :, :d // 2] == 0).all() and (pool[0, :3, :, d // 2:] == 2).all()


@pytest.mark.parametrize("new,total,width,page", [(20, 60, 3, 16), (2, 60, 3, 16), (200, 700, 5, 32), (1, 129, 1, 128), (40, 600, 2, 256), (150, 149, 4, 16)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_length_beyond_the_table(new, total, width, page, d):
    """more positions than the table has entries for: the rows behind them see those that are there"""
    s = batch(1, [(new, total), (3, 30)], 4, 2, d, page, poison=False)
    s["table"] = s["table"][:, :width].contiguous()
    check_attn(s, 4, 2, d)


def test_a_pair_that_is_gone_through_again_for_longer_than_a_wait():
    """An infinite value in sight of sixteen rows behind 2.1 million positions (the same page over and over): the slow way through
    them takes more than a wait's 1.5 seconds, while the next pair's blocks are asked for."""
    from ixrun_b200.paged import AttnPaged

    d, page, requests, new, n_pages = 128, 256, 149, 16, 8400
    g = torch.Generator(device=DEV).manual_seed(1)
    kp, vp = (torch.randn(2, page, 1, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    vp[0, 0, 0, 3] = float("inf")
    q = torch.randn(requests * new, d, generator=g, device=DEV).bfloat16()
    cu = torch.arange(requests + 1, dtype=torch.int32, device=DEV) * new
    table = torch.zeros(requests, n_pages + 1, dtype=torch.int32, device=DEV)
    table[:, n_pages] = 1                              # the new tokens' own page
    length = torch.full((requests,), n_pages * page + new, dtype=torch.int32, device=DEV)
    got = AttnPaged(1, 1, d, DEV)(q, kp, vp, table, length, cu, max_q=new).double()
    e = torch.exp(q.double() @ torch.cat([kp[0, :, 0], kp[1, :new, 0]]).double().t() * d ** -0.5)
    seen = torch.cat([torch.full((requests * new, page), float(n_pages), device=DEV, dtype=torch.float64),
                      (torch.arange(new, device=DEV) <= (torch.arange(requests * new, device=DEV) % new)[:, None]).double()], 1)
    p = e * seen / (e * seen).sum(1, keepdim=True)
    v = torch.cat([vp[0, :, 0], vp[1, :new, 0]]).double()
    assert (got[:, 3] == float("inf")).all()
    fine = [i for i in range(d) if i != 3]
    want, mag = p @ v[:, fine], p @ v[:, fine].abs()
    # a rounding of the result, probabilities of 17 bits, and 32-bit sums one after the other: a warp adds up 16801 slices' values, a lane of it
    # twice as many probabilities
    assert ((got[:, fine] - want).abs() <= BF16 * want.abs() + (2.0 ** -12 + 3 * 16801 * 2.0 ** -24) * mag).all()


def test_refusals_have_one_type_on_both_host_paths(monkeypatch):
    """what the extension takes at once and what the Python path checks: the same ValueError, not an error of the C entry"""
    from ixrun_b200 import _lib, paged
    from ixrun_b200.paged import AttnPaged, PageStep, page_step, rope_kv_paged

    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    cos = torch.zeros(9, 32, device=DEV)
    attn = AttnPaged(4, 2, 64, DEV)
    step = dict(q_len=i(2), length=i(2), table=i(2, 3), free=i(4), n_free=i(1), page=16, rows=5, out=PageStep.empty(2, 5, DEV))
    many = dict(q_len=i(5000), length=i(5000), table=i(5000, 3), out=PageStep.empty(5000, 5, DEV))
    rope = dict(q=b(3, 256), k=b(3, 128), v=b(3, 128), pos=i(3), slot=i(3), k_pages=b(4, 16, 2, 64), v_pages=b(4, 16, 2, 64), cos=cos, sin=cos, hq=4,
                hkv=2, head_dim=64)
    call = dict(q=b(3, 256), k_pages=b(4, 16, 2, 64), v_pages=b(4, 16, 2, 64), table=i(2, 2), length=i(2), cu_rows=i(3))
    odd = dict(k_pages=b(4, 48, 2, 64), v_pages=b(4, 48, 2, 64))
    cases = [(page_step, step, dict(page=24)), (page_step, step, dict(page=512)), (page_step, step, many), (rope_kv_paged, rope, odd), (attn, call, odd),
             (attn, call, dict(table=i(5000, 2), length=i(5000), cu_rows=i(5001))), (attn, call, dict(scale=float("inf"))),
             (attn, call, dict(scale=float("nan"))), (attn, call, dict(scale=0.0)), (attn, call, dict(max_q=0))]
    for python in (False, True):
        if python:
            monkeypatch.setattr(paged, "_host", lambda: _lib._PythonHost)
        for f, ok, bad in cases:
            f(**ok)
            with pytest.raises(ValueError):
                f(**{**ok, **bad})


@pytest.mark.parametrize("lens,max_q", [([(1, 900)] * 3 + [(1, 17)], 1), ([(1, 5000)], 1), ([(4, 300), (3, 3), (2, 900)], 4), ([(1, 2 + i) for i in range(40)], 1)],
                         ids=lambda v: f"{len(v)}x{v[0][0]}-{v[0][1]}" if isinstance(v, list) else None)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (4, 2, 128), (4, 2, 256), (4, 4, 128), (2, 1, 64)])
def test_probabilities_of_few_rows_are_held_in_17_bits(lens, max_q, hq, hkv, d):
    """Half a step of the result; beside it two bf16 numbers leave 2^-16 of a probability, and scores, sums of magnitudes up to 20 in some
    sixteen 32-bit steps that may cut off a unit, 20 * 16 * 2^-23 < 2^-14 of it: less than 2^-13 together.  (With 8 bits
    results of these lengths are off by 3 to 18 times that.)"""
    from ixrun_b200.paged import AttnPaged

    s = batch(5, lens, hq, hkv, d, 32)
    got = AttnPaged(hq, hkv, d, DEV)(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"], max_q=max_q).double()
    want, mag = attn64(s, hq, hkv, d)
    half = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -100))) - 8)
    assert ((got - want).abs() <= half + 2.0 ** -13 * mag).all()


@pytest.mark.parametrize("rot,norm", [(64, False), (64, True), (36, True)])
def test_steps_and_releases_in_dependent_launches(rot, norm):
    """tables, write (rows that are not aligned among them), attention and release one behind the other without a wait of the host: the bits
    of the same calls made one by one"""
    from ixrun_b200.glue import rope_tables
    from ixrun_b200.p6 import set_pdl
    from ixrun_b200.paged import AttnPaged, PageTables, rope_kv_paged

    hq, hkv, d, page, requests, rows, n_pages, width = 4, 2, 64, 16, 6, 120, 60, 9
    g = torch.Generator(device=DEV).manual_seed(5)
    cos, sin = rope_tables(width * page, rot, 10000.0, DEV)
    x = torch.randn(12, rows, (hq + 2 * hkv) * d, generator=g, device=DEV).bfloat16()
    w = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).bfloat16() if norm else None
    new = [on_gpu([(7 * i + 5 * r) % 19 for r in range(requests)]) for i in range(12)]
    done = [torch.tensor([(i + r) % 4 == 0 for r in range(requests)], device=DEV) for i in range(12)]

    def run(wait):
        t, attn, outs = PageTables(requests, n_pages, page, width, DEV), AttnPaged(hq, hkv, d, DEV), []
        kp, vp = (torch.zeros(n_pages, page, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        st, qs = t.new_step(rows), torch.zeros(rows, hq * d, dtype=torch.bfloat16, device=DEV)
        for i in range(12):
            q, k, v = x[i][:, :hq * d], x[i][:, hq * d:(hq + hkv) * d], x[i][:, (hq + hkv) * d:]
            o = torch.zeros_like(qs)
            wait()
            t.step(new[i], rows, out=st)
            wait()
            rope_kv_paged(q, k, v, st.pos, st.slot, kp, vp, cos, sin, hq, hkv, d, rot_dim=rot, q_norm=w, k_norm=w, out=qs)
            wait()
            attn(qs, kp, vp, t.table, st.length, st.cu_rows, out=o)
            wait()
            outs += [o, t.release(done[i])]
            wait()
            outs += [t.table.clone(), t.free.clone(), t.n_free.clone(), t.length.clone()]
        return outs + [kp, vp]

    want = run(torch.cuda.synchronize)
    assert all(s.tolist()[0] == 0 for s in want[1:-2:6])
    prev = set_pdl(True)
    try:
        for _ in range(5):
            got = run(lambda: None)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    finally:
        torch.cuda.synchronize()
        set_pdl(prev)


@pytest.mark.parametrize("rot,norm", [(64, False), (36, True)])
def test_a_position_outside_the_tables_is_the_nearest_one_in_them(rot, norm):
    from ixrun_b200.glue import rope_tables
    from ixrun_b200.paged import rope_kv_paged

    hq, hkv, d = 2, 1, 64
    g = torch.Generator(device=DEV).manual_seed(2)
    cos, sin = rope_tables(50, rot, 10000.0, DEV)
    w = torch.randn(d, generator=g, device=DEV).bfloat16() if norm else None
    x = [torch.randn(5, n * d, generator=g, device=DEV).bfloat16() for n in (hq, hkv, hkv)]
    got = []
    for pos in ([50, 51, 2**31 - 1, -1, -2**31], [49, 49, 49, 0, 0]):
        kp, vp = (torch.zeros(1, 16, hkv, d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        got.append((rope_kv_paged(*x, on_gpu(pos), on_gpu([0, 1, 2, 3, 4]), kp, vp, cos, sin, hq, hkv, d, rot_dim=rot, q_norm=w, k_norm=w,
                                  out=torch.empty_like(x[0])), kp, vp))
    for a, b in zip(*got):
        assert torch.equal(a, b)
