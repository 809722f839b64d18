"""The paged-cache operators on the GPU against their definitions in 64 bits (tests/paged_forms.py)."""
from __future__ import annotations

import pytest
import torch

import jetsonfabric_amd as jf
from tests.paged_forms import TYPES, Sequences, rotate, rotation_bound

pytestmark = pytest.mark.gpu


def normal(*size, seed=0, std=1.0):
    return torch.randn(*size, generator=torch.Generator().manual_seed(seed)) * std


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def within(got, want, bound):
    off = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    worst = (off - bound).max().item()
    assert worst <= 0, f"off by {off.max().item():.3e}, over the bound by {worst:.3e}"


SCALINGS = [{}, {"scaling": "linear", "factor": 8.0}, {"scaling": "ntk", "factor": 4.0},
            {"scaling": "yarn", "factor": 4.0, "original_context": 32768},
            {"scaling": "yarn", "factor": 40.0, "original_context": 4096, "base": 1.0e4, "attention_factor": 0.7}]


# ---------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rows,heads,dim,n_rot", [(1, 1, 2, 2), (1, 28, 128, 128), (2, 32, 128, 64), (7, 3, 100, 36),
                                                  (3, 5, 80, 80), (33, 4, 96, 48), (1025, 6, 64, 64), (1031, 3, 67, 66),
                                                  (5, 2, 256, 256), (4, 2, 300, 256)])
def test_rotation(rows, heads, dim, n_rot, layout):
    for n, (kw, (xt, yt)) in enumerate(zip(SCALINGS, [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"),
                                                      ("f16", "f32")])):
        if n_rot == 2 and kw.get("scaling") == "ntk":
            continue
        x = normal(rows, heads, dim, seed=n, std=2.0).to(TYPES[xt])
        p = torch.randint(0, 1 << 20, (rows,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
        want, terms = rotate(x, p, n_rot, layout, **kw)
        out = torch.full((rows, heads, dim), 9.0, dtype=TYPES[yt], device="cuda")
        rope = jf.Rope(n_rot, layout=layout, **kw)
        assert rope.rotate(x.cuda(), p.cuda(), out=out) is out
        within(out.cpu(), want, rotation_bound(want, terms, TYPES[yt]))
        assert torch.equal(out[..., n_rot:].cpu(), x[..., n_rot:].to(TYPES[yt]))


def test_rotation_of_far_and_negative_positions():
    p = ints([0, 1, -1, 1 << 20, -(1 << 20), (1 << 23) + 5, -(1 << 24)])
    x = normal(len(p), 2, 128, seed=3)
    want, terms = rotate(x, p, 128)
    got = jf.Rope(128).rotate(x.cuda(), p.cuda())
    within(got.cpu(), want, rotation_bound(want, terms, torch.float32))
    assert torch.equal(got[0].cpu(), x[0])  # position 0 turns nothing
    back = jf.Rope(128).rotate(got, -p.cuda())
    # the first turn is off by 4.6e-7 (|a| + |b|) at most, the second by as much of values up to sqrt 2 larger
    assert (back.cpu() - x).abs().max() < 4.9 * 4.6e-7 * x.abs().max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotation_in_place_and_of_strided_rows(dtype, layout):
    """Queries and keys inside fused rows; the rest of the buffer stays as it was. Odd offsets take the narrow form."""
    for first, pad in ((0, 0), (1, 0), (0, 3)):  # values before the rows, values between rows
        t = TYPES[dtype]
        store = normal(9 * (6 * 64 + pad) + first, seed=5).to(t)
        gpu = store.cuda()

        def view(s):
            return s[first:].reshape(9, 6 * 64 + pad)[:, :4 * 64].unflatten(1, (4, 64))

        p = torch.arange(100, 109, dtype=torch.int32)
        want, terms = rotate(view(store), p, 32, layout)
        x = view(gpu)
        assert x.data_ptr() == gpu.data_ptr() + first * gpu.element_size()
        jf.Rope(32, layout=layout).rotate(x, p.cuda(), out=x)
        within(x.cpu(), want, rotation_bound(want, terms, t))
        assert torch.equal(x[..., 32:].cpu(), view(store)[..., 32:])
        rest = torch.ones(len(store), dtype=torch.bool)
        view(rest)[...] = False
        assert torch.equal(gpu.cpu()[rest], store[rest])


@pytest.mark.parametrize("rows,heads,dim,n_rot,dtype", [(1027, 160, 128, 128, "bf16"), (66001, 2, 128, 64, "f16"),
                                                        (1030, 65, 136, 128, "f32")])
def test_rotation_of_more_rows_than_the_caches_hold(rows, heads, dim, n_rot, dtype):
    """Out of place, in place behind it, and back to back with a reader of the result."""
    t = TYPES[dtype]
    x = normal(rows, heads, dim, seed=2).to(t)
    p = torch.randint(0, 1 << 15, (rows,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    assert x.numel() * x.element_size() > 32 << 20
    want, terms = rotate(x, p, n_rot)
    bound = rotation_bound(want, terms, t)
    rope, gx, gp = jf.Rope(n_rot), x.cuda(), p.cuda()
    got = rope.rotate(gx, gp)
    rope.rotate(gx, gp, out=gx)
    assert torch.equal(got, gx)
    within(got.cpu(), want, bound)


def test_rotation_of_no_rows():
    x = torch.zeros(0, 4, 64, device="cuda")
    assert jf.Rope(64).rotate(x, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


def test_rotation_keeps_nonfinite_values_to_their_pair():
    x = normal(2, 1, 64, seed=1)
    x[0, 0, 5], x[1, 0, 40] = float("inf"), float("nan")
    got = jf.Rope(32).rotate(x.cuda(), ints([3, 4]).cuda()).cpu()
    assert not torch.isfinite(got[0, 0, [5, 21]]).any() and torch.isnan(got[1, 0, 40])
    assert torch.isfinite(got).sum() == got.numel() - 3


# ---------------------------------------------------------------- rows into pages

def appended(seq, k, v, positions, rope_kw, rope):
    """The pool after an append, and the bound of the keys."""
    kp, vp, w, pos = seq.k.double().clone(), seq.v.clone(), seq.weights.clone(), seq.positions.clone()
    bound = torch.zeros_like(kp)
    rk, terms = rotate(k, positions, **rope_kw) if rope else (k.double(), torch.zeros(k.shape, dtype=torch.float64))
    for s in range(len(seq.rows)):
        for row, t in seq.rows_of(s):
            at = seq.slot(s, t)
            if at is None:
                continue
            page, i = at
            kp[page, :, i] = rk[row]
            bound[page, :, i] = rotation_bound(rk[row], terms[row], seq.dtype)
            vp[page, :, i] = v[row].to(seq.dtype)
            w[page, :, i], pos[page, :, i] = 0.0, positions[row]
    return kp, bound, vp, w, pos


APPENDS = [
    # rows, lengths, K/V heads, dim, page, what else
    ([1], [1], 1, 8, 1, {}),
    ([1, 1], [257, 4096], 4, 128, 16, {"absent": [(1, 3)]}),
    ([9, 0, 9], [4100, 5, 9], 8, 128, 16, {"order": "tokens"}),
    ([5, 3], [5, 700], 2, 64, 64, {"order": "padded", "pad_rows": 4}),
    ([33, 1, 700], [40, 33, 1500], 2, 96, 8, {"absent": [(2, 101), (2, 187), (0, 4)], "pad_rows": 3}),
    ([6, 4], [2, 4], 3, 80, 4, {}),  # more rows than slots: the first ones fall out
    ([1100, 77], [1100, 2000], 1, 256, 256, {}),
    ([3], [3], 2, 72, 2, {"wide_table": 5}),
]


@pytest.mark.parametrize("rows,lens,heads,dim,page,more", APPENDS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_append(rows, lens, heads, dim, page, more, kind):
    for n, (rt, layout, kw) in enumerate([(kind, "half", SCALINGS[3]), ("f32", "interleaved", SCALINGS[1]), ("f32", None, {})]):
        seq = Sequences(rows, lens, heads, dim, page, TYPES[kind], seed=n, **more)
        g = normal(seq.total, 2 * heads + 1, dim, seed=20 + n, std=1.5).to(TYPES[rt])
        k, v = g[:, :heads], g[:, heads:2 * heads]
        positions = torch.randint(0, 200000, (seq.total,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
        n_rot = dim if n == 0 else dim // 4 * 2
        rope = jf.Rope(n_rot, layout=layout, **kw) if layout else None
        want, bound, wv, ww, wp = appended(seq, k, v, positions, {"n_rot": n_rot, "layout": layout or "half", **kw}, rope)
        kp, vp, w, pos, table, lengths, starts = seq.to_gpu()
        cache = jf.PagedCache(kp, vp, w, pos)
        batch = jf.PagedBatch(table, lengths, starts, seq.max_rows, seq.max_length)
        gpu = g.cuda()
        cache.append(batch, gpu[:, :heads], gpu[:, heads:2 * heads], positions.cuda(), rope)
        if rope:
            within(kp.cpu(), want, bound)
            untouched = bound == 0
            assert torch.equal(kp.cpu()[untouched], seq.k[untouched])
        else:
            assert torch.equal(kp.cpu(), want.to(seq.dtype))
        assert torch.equal(vp.cpu(), wv) and torch.equal(w.cpu(), ww) and torch.equal(pos.cpu(), wp)
        assert torch.equal(lengths.cpu(), seq.lengths)


def test_append_from_rows_of_odd_offsets_and_without_weights():
    seq = Sequences([4, 2], [20, 33], 2, 64, 16, torch.float16, seed=2)
    flat = normal(seq.total * (4 * 64 + 1) + 1, seed=9).half()
    view = flat[1:].reshape(seq.total, 4 * 64 + 1)[:, :256].unflatten(1, (4, 64))
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    batch = jf.PagedBatch(table, lengths, starts, 4, 33)
    x = flat.cuda()[1:].reshape(seq.total, 4 * 64 + 1)[:, :256].unflatten(1, (4, 64))
    jf.PagedCache(kp, vp).append(batch, x[:, :2], x[:, 2:])
    want, _, wv, _, _ = appended(seq, view[:, :2], view[:, 2:], torch.zeros(seq.total, dtype=torch.int32), {}, None)
    assert torch.equal(kp.cpu(), want.half()) and torch.equal(vp.cpu(), wv)


def test_bounds_leave_out_what_lies_beyond_them():
    """max_rows below a sequence's rows, max_length below a length: the rows and slots beyond them are left out."""
    seq = Sequences([3, 2], [20, 33], 2, 64, 16, torch.float16, seed=4)
    k, v = normal(5, 2, 64, seed=1).half(), normal(5, 2, 64, seed=2).half()
    kp, vp, w, pos, table, lengths, starts = seq.to_gpu()
    cache = jf.PagedCache(kp, vp, w, pos)
    cache.append(jf.PagedBatch(table, lengths, starts, 2, 30), k.cuda(), v.cuda(), ints([1, 2, 3, 4, 5]).cuda())
    want = seq.v.clone()
    for s, row, t in ((0, 0, 18), (0, 1, 19), (1, 3, 28), (1, 4, 29)):
        page, i = seq.slot(s, t)
        want[page, :, i] = v[row]
    assert torch.equal(vp.cpu(), want)


# ---------------------------------------------------------------- attention

def attended(seq, heads, causal=True, scale=None, q=None, lse=True):
    """Attention of random queries over seq's cache, checked; returns (q, out, lse) on the CPU."""
    scale = seq.dim ** -0.5 if scale is None else scale
    q = normal(seq.total, heads, seq.dim, seed=77, std=1.5).to(seq.dtype) if q is None else q
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    cache = jf.PagedCache(kp, vp)
    batch = jf.PagedBatch(table, lengths, starts, seq.max_rows, seq.max_length)
    out = torch.full(q.shape, 7.0, dtype=seq.dtype, device="cuda")
    got, got_lse = cache.attend(batch, q.cuda(), scale, causal, out=out,
                                lse=torch.full(q.shape[:2], 5.0, device="cuda"))
    assert got is out
    want, want_lse, bound, lse_bound = seq.attend(q, scale, causal)
    n = seq.starts[-1]
    within(out[:n].cpu(), want[:n], bound[:n])
    some = want_lse[:n] > -float("inf")
    assert torch.equal(got_lse[:n].cpu()[~some], want_lse[:n].float()[~some])
    within(got_lse[:n].cpu()[some], want_lse[:n][some], lse_bound[:n][some])
    assert (out[n:] == 7).all() and (got_lse[n:] == 5).all()  # rows of no sequence
    return q, out.cpu(), got_lse.cpu()


ATTENDS = [
    # rows, lengths, heads, K/V heads, dim, page, what else
    ([1], [1], 1, 1, 64, 1, {}),
    ([1], [256], 12, 2, 128, 16, {}),
    ([1, 1, 1], [31, 32, 33], 28, 4, 128, 16, {"order": "tokens"}),
    ([1] * 5, [1, 700, 17, 64, 129], 8, 2, 64, 32, {"absent": [(1, 3), (3, 0), (3, 1)]}),
    ([1, 0, 1], [5000, 3, 4097], 40, 8, 128, 64, {"pad_rows": 2}),
    ([9, 9], [1033, 9], 40, 8, 128, 16, {}),
    ([5, 3, 0, 7], [300, 3, 5, 2], 7, 1, 96, 8, {"pad_rows": 3, "order": "padded"}),
    ([4, 2], [2000, 2], 4, 1, 256, 256, {}),
    ([2, 6], [70, 100], 12, 2, 200, 4, {"absent": [(0, 5), (1, 24)]}),
    ([33, 1, 130], [33, 900, 400], 6, 3, 80, 2, {"absent": [(2, 0), (2, 7)], "wide_table": 3}),
    ([100], [100], 28, 4, 128, 16, {}),
    ([77, 200], [1500, 333], 10, 2, 64, 64, {"order": "tokens", "pad_rows": 1}),
    ([3], [40], 16, 16, 8, 8, {}),
    ([1], [9000], 4, 1, 72, 1, {}),
    ([20], [65], 3, 1, 256, 16, {}),
    ([1], [40000], 2, 1, 64, 16, {}),       # more than 64 splits
    ([40, 3], [9000, 5], 2, 1, 64, 32, {}),  # of tiles
    ([3], [20000], 8, 1, 128, 64, {}),
]


@pytest.mark.parametrize("rows,lens,heads,kv,dim,page,more", ATTENDS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention(rows, lens, heads, kv, dim, page, more, kind):
    for causal in (True, False):
        attended(Sequences(rows, lens, kv, dim, page, TYPES[kind], seed=len(rows), **more).poison(), heads, causal)


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_rows_that_see_nothing(rows):
    """Sequences without slots, with fewer slots than rows, with absent pages alone; other rows beside them."""
    seq = Sequences([rows, rows, rows, rows], [0, rows // 2, 48, 50], 2, 64, 16, torch.float16, seed=3,
                    absent=[(2, 0), (2, 1), (2, 2), (2, 3)]).poison()
    q, out, lse = attended(seq, 6)
    assert (out[:rows] == 0).all() and (lse[:rows] == -float("inf")).all()
    assert (out[2 * rows:3 * rows] == 0).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [6, 150])
def test_attention_does_not_take_hidden_infinities(kind, rows):
    """Later rows' K and V are infinite or NaN: rows that do not see them are as if those were numbers."""
    seq = Sequences([rows], [rows + 37], 1, 64, 16, TYPES[kind], seed=8)
    at = {t: seq.slot(0, t) for t in range(37, rows + 37)}
    q = normal(rows, 4, 64, seed=9).to(seq.dtype)
    clean = seq.attend(q, 0.125)
    for t, v in ((39, float("inf")), (40, float("nan")), (rows + 36, -float("inf"))):
        seq.v[at[t][0], 0, at[t][1], 3] = v
    seq.k[at[41][0], 0, at[41][1], 5] = float("nan")
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    out, lse = jf.PagedCache(kp, vp).attend(jf.PagedBatch(table, lengths, starts, rows, rows + 37), q.cuda(), 0.125)
    out = out.cpu()
    seen = torch.arange(64) != 3
    within(out[:4][..., seen], clean[0][:4][..., seen], clean[2][:4][..., seen])
    within(out[:2], clean[0][:2], clean[2][:2])
    assert (out[2, :, 3] == float("inf")).all()       # row 2 sees slot 39
    assert torch.isnan(out[3, :, 3]).all()            # and row 3 a NaN
    assert torch.isnan(out[4:]).all()                 # a NaN score makes the row NaN
    assert torch.isnan(lse[4:]).all() and torch.isfinite(lse[:4]).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,lens,dim", [([5, 6], [700, 7], 64), ([5, 8], [3000, 4100], 128), ([1, 5], [40, 3], 96), ([7, 0], [7, 1], 128)])
def test_attention_with_room_for_long_sequences(rows, lens, dim, kind):
    """Tables and bounds for many more positions than there are: 4 to 32 queries per K/V head, infinities of V that some
    rows do not see."""
    seq = Sequences(rows, lens, 4, dim, 16, TYPES[kind], seed=6).poison()
    q = normal(seq.total, 16, dim, seed=7).to(seq.dtype)
    want, want_lse, bound, lse_bound = seq.attend(q, 0.1)
    at = seq.slot(0, lens[0] - rows[0] // 2 - 1)  # the last rows // 2 + 1 rows see it
    seq.v[at[0], 2, at[1], 5] = float("inf")
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    table = torch.cat([table, torch.full((2, 5000), -1, dtype=torch.int32, device="cuda")], 1)
    batch = jf.PagedBatch(table, lengths, starts, max(rows), table.shape[1] * 16)
    out, lse = jf.PagedCache(kp, vp).attend(batch, q.cuda(), 0.1)
    out, lse = out.cpu(), lse.cpu()
    struck = torch.zeros(out.shape, dtype=torch.bool)
    struck[rows[0] - rows[0] // 2 - 1:rows[0], 8:12, 5] = True
    assert (out[struck] == float("inf")).all()
    within(out[~struck], want[~struck], bound[~struck])
    some = want_lse > -float("inf")
    assert torch.equal(lse[~some], want_lse[~some].float())
    within(lse[some], want_lse[some], lse_bound[some])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,rows,length", [(1, 200, 200), (1, 150, 333), (4, 130, 130)])
def test_attention_takes_the_infinities_that_it_sees(heads, rows, length, dim):
    """Rows far behind an infinite V, which see all of its tile, have it as the rows near it do."""
    seq = Sequences([rows], [length], 1, dim, 16, torch.float16, seed=4)
    q = normal(rows, heads, dim, seed=5).half()
    want, _, bound, _ = seq.attend(q, 0.05)
    odd = {3: (length - rows + 5, float("inf")), 9: (length - rows + 70, -float("inf")), 11: (length - rows + 100, float("nan"))}
    for column, (t, x) in odd.items():
        at = seq.slot(0, t)
        seq.v[at[0], 0, at[1], column] = x
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    out, _ = jf.PagedCache(kp, vp).attend(jf.PagedBatch(table, lengths, starts, rows, length), q.cuda(), 0.05)
    out = out.cpu()
    plain = [c for c in range(dim) if c not in odd]
    within(out[..., plain], want[..., plain], bound[..., plain])
    for column, (t, x) in odd.items():
        first = t - (length - rows)
        within(out[:first, :, column], want[:first, :, column], bound[:first, :, column])
        left = out[first:, :, column]
        assert torch.isnan(left).all() if x != x else (left == x).all()


def test_attention_of_infinite_queries_and_scores():
    seq = Sequences([3, 1], [40, 50], 1, 64, 16, torch.float16, seed=1)
    q = normal(4, 2, 64, seed=2).half()
    want = seq.attend(q, 0.125)
    q[1, 0, 0], q[2, 1, 7] = float("nan"), float("inf")
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    out, _ = jf.PagedCache(kp, vp).attend(jf.PagedBatch(table, lengths, starts, 3, 50), q.cuda(), 0.125)
    out = out.cpu()
    assert torch.isnan(out[1, 0]).all() and torch.isnan(out[2, 1]).all()
    for r, h in ((0, 0), (0, 1), (1, 1), (2, 0), (3, 0), (3, 1)):
        within(out[r, h], want[0][r, h], want[2][r, h])


@pytest.mark.parametrize("rows", [1, 8, 90])
def test_attention_of_large_scores(rows):
    """Scores over hundreds: one slot takes nearly everything; a scale that is not 1 / sqrt(dim)."""
    seq = Sequences([rows], [777], 2, 128, 16, torch.bfloat16, seed=5)
    q = normal(rows, 8, 128, seed=6, std=6.0).bfloat16()
    attended(seq, 8, q=q, scale=0.5)
    attended(seq, 8, q=q, scale=1e-6)


def test_attention_of_strided_rows_on_another_stream():
    seq = Sequences([3, 2], [80, 300], 2, 64, 16, torch.float16, seed=6)
    fused = normal(5, 14 * 64, seed=3).half()
    view = fused.unflatten(1, (14, 64))[:, 2:10]
    want = seq.attend(view, 0.125)
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    cache, batch = jf.PagedCache(kp, vp), jf.PagedBatch(table, lengths, starts, 3, 300)
    gpu = fused.cuda()
    out = torch.zeros(5, 8, 3 * 64, dtype=torch.float16, device="cuda")[..., 64:128]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        cache.attend(batch, gpu.unflatten(1, (14, 64))[:, 2:10], 0.125, out=out)
    stream.synchronize()
    within(out.cpu(), want[0], want[2])


@pytest.mark.parametrize("rows,length", [(1, 40), (2, 5000), (60, 90), (30, 9000)])
def test_attention_in_place(rows, length):
    seq = Sequences([rows], [length], 2, 64, 16, torch.float16, seed=7)
    q = normal(rows, 8, 64, seed=3).half()
    want, _, bound, _ = seq.attend(q, 0.125)
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    gpu = q.cuda()
    out, _ = jf.PagedCache(kp, vp).attend(jf.PagedBatch(table, lengths, starts, rows, length), gpu, out=gpu)
    assert out is gpu
    within(gpu.cpu(), want, bound)


# ---------------------------------------------------------------- attention weights

@pytest.mark.parametrize("rows,lens,heads,kv,dim,page,more", ATTENDS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_weights(rows, lens, heads, kv, dim, page, more, kind):
    seq = Sequences(rows, lens, kv, dim, page, TYPES[kind], seed=len(lens), **more).poison()
    q = normal(seq.total, heads, dim, seed=4, std=1.5).to(seq.dtype)
    scale = dim ** -0.5
    kp, vp, w, _, table, lengths, starts = seq.to_gpu()
    cache, batch = jf.PagedCache(kp, vp, w), jf.PagedBatch(table, lengths, starts, seq.max_rows, seq.max_length)
    for causal in (True, False):
        lse = seq.attend(q, scale, causal)[1].float()
        w.copy_(seq.weights)
        cache.weigh(batch, q.cuda(), lse.cuda(), scale, causal)
        want, bound = seq.weigh(q, lse, scale, causal)
        within(w.cpu(), want, bound)
        assert torch.equal(w.cpu()[bound == 0], seq.weights[bound == 0])
        again = w.clone()
        w.copy_(seq.weights)
        cache.weigh(batch, q.cuda(), lse.cuda(), scale, causal)
        assert torch.equal(w, again)


def test_weights_of_attention_sum_to_its_rows():
    """What a step adds to all positions of a K/V head is its rows times its heads."""
    seq = Sequences([50, 3], [400, 77], 2, 128, 16, torch.float16, seed=4)
    kp, vp, w, _, table, lengths, starts = seq.to_gpu()
    cache, batch = jf.PagedCache(kp, vp, w), jf.PagedBatch(table, lengths, starts, 50, 400)
    q = normal(53, 10, 128, seed=1, std=2.0).half().cuda()
    w.zero_()
    _, lse = cache.attend(batch, q)
    cache.weigh(batch, q, lse)
    per_head = w.double().sum((0, 2)).cpu()
    # lse and the weights carry the same scores: errors of their sums and exponentials, below 400 terms' worst case
    assert (per_head - 53 * 5).abs().max() < 53 * 5 * (400 + 64) * 2.0**-23


def test_weights_of_the_last_rows_alone():
    """A prompt's last rows only: a step of fewer rows over the same lengths."""
    seq = Sequences([8, 8], [300, 90], 1, 64, 16, torch.float16, seed=2)
    q = normal(200, 4, 64, seed=3).half()
    part = torch.cat([q[92:100], q[192:200]])
    lse = seq.attend(part, 0.125)[1].float()
    kp, vp, w, _, table, lengths, starts = seq.to_gpu()
    jf.PagedCache(kp, vp, w).weigh(jf.PagedBatch(table, lengths, starts, 8, 300), part.cuda(), lse.cuda(), 0.125)
    want, bound = seq.weigh(part, lse, 0.125)
    within(w.cpu(), want, bound)


# ---------------------------------------------------------------- cutting

def cut(seq, budget, first, recent):
    kp, vp, w, pos, table, lengths, starts = seq.to_gpu()
    batch = jf.PagedBatch(table, lengths, starts, seq.max_rows, seq.max_length)
    jf.PagedCache(kp, vp, w, pos).evict(batch, budget, first, recent)
    k, v, ww, wp, lens = seq.evict(budget, first, recent)
    assert lengths.cpu().tolist() == lens
    assert torch.equal(pos.cpu(), wp)
    assert torch.equal(w.cpu().view(torch.int32), ww.view(torch.int32))
    for got, want in ((kp, k), (vp, v)):
        assert torch.equal(got.cpu().contiguous().view(torch.int16), want.contiguous().view(torch.int16))
    return w.cpu(), pos.cpu()


CUTS = [
    # lengths, K/V heads, dim, page, budget, first, recent, what else
    ([2], 1, 8, 1, 1, 0, 1, {}),
    ([33, 32, 31], 2, 64, 16, 32, 4, 8, {}),
    ([4097, 4096, 100], 4, 128, 16, 4096, 4, 256, {}),
    ([1000, 3000], 2, 72, 8, 700, 0, 0, {"order": "tokens"}),
    ([1500, 900], 3, 256, 64, 100, 4, 32, {"order": "padded"}),
    ([500, 70], 2, 64, 16, 64, 40, 40, {}),       # more protected than the budget
    ([600], 2, 64, 16, 200, 4, 16, {"absent": [(0, 2), (0, 20), (0, 30)]}),
    ([90], 1, 64, 16, 30, 4, 16, {"absent": [(0, 0), (0, 1)]}),
    ([40000, 33000], 1, 8, 256, 20000, 16, 1000, {}),  # beyond the keys held in LDS
    ([70000], 1, 8, 1024, 66000, 16, 1000, {}),        # more than one round of the lists
    ([2500], 1, 16, 2, 2499, 0, 1, {}),
    ([5, 1, 0], 2, 32, 4, 3, 1, 1, {}),
]


@pytest.mark.parametrize("lens,kv,dim,page,budget,first,recent,more", CUTS)
@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
def test_cut(lens, kv, dim, page, budget, first, recent, more, values):
    seq = Sequences([0] * len(lens), lens, kv, dim, page, torch.float16, seed=budget, **more)
    for s in range(len(lens)):  # positions as a cache has them that was cut before: ascending, with gaps
        for p in range(-(-lens[s] // page)):
            at = seq.slot(s, p * page)
            if at is not None:
                seq.positions[at[0]] = (torch.arange(page, dtype=torch.int32) + p * page) * 2
    if values == "ties":
        seq.weights = (seq.weights * 3).floor() - 1
        seq.weights[seq.weights == 0] *= -1  # -0 and 0 weigh the same
    if values == "odd":
        pick = torch.randint(0, 12, seq.weights.shape, generator=torch.Generator().manual_seed(1))
        for n, x in enumerate((float("nan"), -float("nan"), float("inf"), -float("inf"), -1.0, 1e-42, 3e38)):
            seq.weights[pick == n] = x
    cut(seq, budget, first, recent)


def test_cut_of_a_cache_in_any_order_protects_by_position():
    """The newest and the first positions stay wherever their slots are."""
    seq = Sequences([0], [300], 1, 64, 16, torch.bfloat16, seed=9)
    order = torch.randperm(300, generator=torch.Generator().manual_seed(2)).int()
    for t in range(300):
        at = seq.slot(0, t)
        seq.positions[at[0], 0, at[1]] = order[t] + 1000
    _, pos = cut(seq, 40, 1004, 30)
    left = {int(pos[(*seq.slot(0, t)[:1], 0, seq.slot(0, t)[1])]) for t in range(40)}
    assert left >= set(range(1000, 1004)) | set(range(1270, 1300))


def test_cut_within_the_budget_changes_nothing():
    seq = Sequences([0, 0], [50, 64], 2, 64, 16, torch.float16, seed=1)
    cut(seq, 64, 4, 8)
    cut(seq, 1000, 4, 8)


def test_offsets_beyond_32_bits():
    """Pages further apart than 2^32 values: every operator on them gives what it gives on neighbouring pages."""
    far, shape = (1 << 32) + 1024, (3, 2, 16, 64)
    seq = Sequences([5], [40], 2, 64, 16, torch.float16, seed=3, extra_pages=0)
    near = seq.to_gpu()
    pools = [torch.empty(2 * far + 2 * 16 * 64, dtype=torch.float16, device="cuda").as_strided(shape, (far, 1024, 64, 1))
             for _ in range(2)]
    for x, y in zip(pools, near):
        x.copy_(y)
    rows = normal(5, 12, 64, seed=1).half().cuda()
    positions = torch.arange(35, 40, dtype=torch.int32, device="cuda")
    got = []
    for k, v in (near[:2], pools):
        w, pos, lengths = near[2].clone(), near[3].clone(), near[5].clone()
        cache, batch = jf.PagedCache(k, v, w, pos), jf.PagedBatch(near[4], lengths, near[6], 5, 40)
        cache.append(batch, rows[:, 8:10], rows[:, 10:], positions, jf.Rope(64))
        out, lse = cache.attend(batch, rows[:, :8])
        many, _ = cache.attend(batch, rows[:, :8].repeat(1, 5, 1))
        cache.weigh(batch, rows[:, :8], lse)
        cache.evict(batch, 20, 2, 4)
        got.append([out, lse, many, k.contiguous(), v.contiguous(), w, pos, lengths])
    for x, y in zip(*got):
        assert torch.equal(x, y)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_prompt_cut_and_decoding(kind):
    """A prompt in two chunks, its cache cut by the weights of its last rows, then steps of single tokens with the cache
    held at its budget: every operator on what the ones before it left, each against its definition on those values."""
    dtype, heads, kv, dim, budget, page = TYPES[kind], 10, 2, 64, 96, 16
    kw = {"layout": "half", "scaling": "yarn", "factor": 4.0, "original_context": 64}
    rope = jf.Rope(dim, **kw)
    seq = Sequences([0, 0], [0, 0], kv, dim, page, dtype, seed=12, wide_table=20)
    kp, vp, w, pos, table, lengths, starts = seq.to_gpu()
    cache = jf.PagedCache(kp, vp, w, pos)
    text = [0, 0]
    for step, rows in enumerate([[130, 61], [70, 1], [1, 1], [1, 1], [3, 0], [1, 1]]):
        total = sum(rows)
        qkv = normal(total, heads + 2 * kv, dim, seed=30 + step, std=1.5).to(dtype)
        positions = torch.cat([torch.arange(text[s], text[s] + rows[s], dtype=torch.int32) for s in range(2)])
        seq.rows, seq.starts, seq.total = rows, [0, rows[0], total], total
        seq.lens = [n + r for n, r in zip(seq.lens, rows)]
        text = [n + r for n, r in zip(text, rows)]
        lengths.copy_(ints(seq.lens))
        starts.copy_(ints(seq.starts))
        batch = jf.PagedBatch(table, lengths, starts, max(rows), max(seq.lens))
        gpu = qkv.cuda()
        q = rope.rotate(gpu[:, :heads], positions.cuda())
        want, terms = rotate(qkv[:, :heads], positions, dim, **kw)
        within(q.cpu(), want, rotation_bound(want, terms, dtype))

        want_k, bound, want_v, want_w, want_p = appended(seq, qkv[:, heads:heads + kv], qkv[:, heads + kv:], positions,
                                                         {"n_rot": dim, **kw}, rope)
        cache.append(batch, gpu[:, heads:heads + kv], gpu[:, heads + kv:], positions.cuda(), rope)
        within(kp.cpu(), want_k, bound)
        assert torch.equal(vp.cpu(), want_v) and torch.equal(w.cpu(), want_w) and torch.equal(pos.cpu(), want_p)
        seq.k, seq.v, seq.weights, seq.positions = kp.cpu(), vp.cpu(), w.cpu(), pos.cpu()

        out, lse = cache.attend(batch, q)
        want, want_lse, bound, lse_bound = seq.attend(q.cpu(), dim ** -0.5)
        within(out.cpu(), want, bound)
        within(lse.cpu(), want_lse, lse_bound)

        cache.weigh(batch, q, lse)
        want, bound = seq.weigh(q.cpu(), lse.cpu(), dim ** -0.5)
        within(w.cpu(), want, bound)
        seq.weights = w.cpu()
        if step > 0:
            cache.evict(batch, budget, 4, 32)
            k, v, want_w, want_p, seq.lens = seq.evict(budget, 4, 32)
            assert torch.equal(kp.cpu(), k) and torch.equal(vp.cpu(), v) and torch.equal(w.cpu(), want_w)
            assert torch.equal(pos.cpu(), want_p) and lengths.cpu().tolist() == seq.lens
            seq.k, seq.v, seq.weights, seq.positions = k, v, want_w, want_p


def test_a_captured_step_replays_with_other_contents():
    """A decode step with its cut in a graph: lengths, rows and tables of the same tensors change between replays, and
    eager calls of the same shapes run between them. Every replay equals the eager step."""
    dtype, heads, kv, dim, budget = torch.float16, 8, 2, 64, 1500
    rope = jf.Rope(dim)
    seq = Sequences([1, 1], [1500, 1500], kv, dim, 16, dtype, seed=21, wide_table=10)
    state = [x.clone() for x in seq.to_gpu()[:4]]
    _, _, _, _, table, lengths, starts = seq.to_gpu()
    qkv, positions = torch.zeros(2, heads + 2 * kv, dim, dtype=dtype, device="cuda"), ints([0, 0]).cuda()
    batch = jf.PagedBatch(table, lengths, starts, 1, 1600)

    def step(kp, vp, w, pos):
        cache = jf.PagedCache(kp, vp, w, pos)
        q = rope.rotate(qkv[:, :heads], positions)
        cache.append(batch, qkv[:, heads:heads + kv], qkv[:, heads + kv:], positions, rope)
        out, lse = cache.attend(batch, q)
        cache.weigh(batch, q, lse)
        cache.evict(batch, budget, 4, 64)
        return out, lse

    def contents(n):
        g = torch.Generator().manual_seed(100 + n)
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        positions.fill_(1500 + n)
        lengths.copy_(ints([[1501, 1501], [1501, 700], [3, 1501], [1501, 1501]][n]))

    # positions as the cache's slots
    for s in range(2):
        for p in range(table.shape[1]):
            state[3][int(seq.table[s, p])] = torch.arange(16 * p, 16 * p + 16, dtype=torch.int32, device="cuda")
    mine = [x.clone() for x in state]
    graph = torch.cuda.CUDAGraph()
    contents(0)
    warm = [x.clone() for x in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*warm)
    torch.cuda.current_stream().wait_stream(side)
    contents(0)
    with torch.cuda.graph(graph):
        out, lse = step(*mine)
    for n in range(4):
        contents(n)
        want_out, want_lse = step(*state)
        left = lengths.clone()
        contents(n)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out) and torch.equal(lse, want_lse) and torch.equal(lengths, left)
        for a, b in zip(mine, state):
            assert torch.equal(a, b)


def test_calls_on_two_streams_do_not_disturb_each_other():
    seqs = [Sequences([1], [3000], 2, 64, 16, torch.float16, seed=40 + n) for n in range(2)]
    q = normal(1, 8, 64, seed=1).half()
    parts, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seq in seqs:
        kp, vp, _, _, table, lengths, starts = seq.to_gpu()
        parts.append((jf.PagedCache(kp, vp), jf.PagedBatch(table, lengths, starts, 1, 3000)))
    gpu = q.cuda()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for n in range(2):
            with torch.cuda.stream(streams[n]):
                got[n].append(parts[n][0].attend(parts[n][1], gpu)[0])
    torch.cuda.synchronize()
    for n in range(2):
        want, _, bound, _ = seqs[n].attend(q, 0.125)
        for out in got[n]:
            within(out.cpu(), want, bound)


def test_keys_equal_the_engines():
    """Keys that an engine's prefill caches are those that append writes: the same pairs, angles and rounding. One layer,
    float weights; the projected rows come from the engine's own matmul."""
    import numpy as np

    cfg = jf.ModelConfig(n_layer=1, n_embd=256, n_ff=256, n_head=4, n_head_kv=2, n_vocab=256, n_ctx=128)
    model = jf.Model.synthesize(cfg, type_linear=jf.Q8_0, type_embd=jf.Q8_0, type_output=jf.Q8_0, seed=5)
    engine = jf.NativeEngine(model)
    tokens = [int(t) for t in np.random.default_rng(3).integers(0, 256, 20)]
    session = engine.create_session(32)
    session.prefill_greedy(tokens)
    k, _ = session.read_kv(0, 20)
    want = torch.from_numpy(k.view(np.float16).copy()).transpose(0, 1).double()  # [position, head, dim]

    x = engine.dequantize_rows("token_embd.weight", 0, 256, 256)[tokens].astype(np.float64)
    def vector(name):
        return np.frombuffer(model.tensor_bytes(name), dtype=np.float32).astype(np.float64)
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg.rms_eps) * vector("blk.0.attn_norm.weight")
    rows = engine.matmul("blk.0.attn_k.weight", x.astype(np.float32), 128) + vector("blk.0.attn_k.bias").astype(np.float32)
    rows = torch.from_numpy(rows.astype(np.float32)).reshape(20, 2, 64).cuda()
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.float16, device="cuda")
    cache = jf.PagedCache(pages, torch.zeros_like(pages))
    batch = jf.PagedBatch(ints([[1, 0]]).cuda(), ints([20]).cuda(), ints([0, 20]).cuda(), 20, 20)
    cache.append(batch, rows, rows, torch.arange(20, dtype=torch.int32, device="cuda"), jf.Rope(64, base=cfg.rope_base))
    got = torch.cat([pages[1], pages[0, :, :4]], 1).transpose(0, 1).double().cpu()
    # the engine rounds its activations to 8-bit codes: a normalization in f32 moves a few of them by one of 127
    assert (got - want).norm() < 0.01 * want.norm()
    engine.close()
    model.close()
