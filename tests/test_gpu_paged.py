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
