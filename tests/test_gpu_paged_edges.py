"""The paged-cache operators on the GPU where single slots, weights or bounds decide: each result against its definition in
64 bits (tests/paged_forms.py), with bounds relative to the output."""
from __future__ import annotations

import math

import pytest
import torch

import jetsonfabric_amd as jf
from tests.paged_forms import TYPES, Sequences, half_step

pytestmark = pytest.mark.gpu


def normal(*size, seed=0, std=1.0):
    return torch.randn(*size, generator=torch.Generator().manual_seed(seed)) * std


def put(seq, s, t, k=None, v=None, at=slice(None)):
    """Sets K or V of a sequence's slot (every K/V head, columns `at`)."""
    page, i = seq.slot(s, t)
    if k is not None:
        seq.k[page, :, i, at] = torch.as_tensor(k, dtype=seq.dtype)
    if v is not None:
        seq.v[page, :, i, at] = torch.as_tensor(v, dtype=seq.dtype)


def attend(seq, q, scale, causal=True, room=0):
    """room: pages that the table has beyond the sequences', all absent."""
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    table = torch.cat([table, torch.full((len(table), room), -1, dtype=torch.int32, device="cuda")], 1)
    batch = jf.PagedBatch(table, lengths, starts, seq.max_rows, table.shape[1] * seq.page if room else seq.max_length)
    out, lse = jf.PagedCache(kp, vp).attend(batch, q.cuda(), scale, causal)
    return out.cpu(), lse.cpu()


# rows, heads of the one K/V head, slots: few queries in one part and in many, tiles in one part and in many
FORMS = [(1, 2, 700), (2, 4, 6000), (1, 1, 40000), (40, 2, 700), (40, 2, 6000), (300, 1, 3000)]


@pytest.mark.parametrize("rows,heads,length", FORMS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [20, 24, 28])
def test_a_heavy_slot_does_not_take_the_others_weight(rows, heads, length, kind, bits):
    """One early slot with V = 0 and 2^bits times the weight of each other: the output is the others' alone."""
    seq = Sequences([rows], [length], 1, 64, 16, TYPES[kind], seed=bits)
    seq.k.zero_()
    seq.v = (torch.rand(seq.v.shape, generator=torch.Generator().manual_seed(1)) * 64 + 32).to(seq.dtype)
    less = bits + torch.rand(seq.k.shape[:3], generator=torch.Generator().manual_seed(2))
    seq.k[..., 0] = (4.0 - less / 4.0).to(seq.dtype)
    put(seq, 0, 3, k=4.0, v=0.0)
    put(seq, 0, 3, k=0.0, at=slice(1, 64))
    q = torch.zeros(rows, heads, 64, dtype=seq.dtype)
    q[..., 0] = 4.0
    scale = math.log(2.0)
    want, want_lse, _, _ = seq.attend(q, scale)
    out, lse = attend(seq, q, scale)
    # All terms are positive. Weights are 29 octaves below the largest at most, where either type has its full precision: a
    # half step each, and one of the output; scores of up to 33 in base 2 (2^-24 of it each for product, scale and
    # difference, 7e-6 of the weight), and f32 sums of 40000 / 256 terms a lane and fewer than 2^8 parts (2^-24 each, 3e-5).
    off = ((out.double() - want) / want).abs().max().item()
    assert off <= 2 * half_step(seq.dtype) + 5e-5, off
    assert (lse.double() - want_lse).abs().max() <= 1e-5


@pytest.mark.parametrize("rows,heads,length", FORMS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_a_slot_that_takes_all_weight_gives_its_value(rows, heads, length, kind):
    """The other slots' weights are below 2^-60 together: the output is V of the one, to the bit."""
    for slot in (0, length - rows, (length - rows) // 2 + 1):
        seq = Sequences([rows], [length], 1, 64, 16, TYPES[kind], seed=slot)
        seq.k *= 0.01
        put(seq, 0, slot, k=normal(64, seed=slot + 1, std=3.0))
        page, i = seq.slot(0, slot)
        q = (seq.k[page, 0, i].float() + normal(rows, heads, 64, seed=2, std=0.3)).to(seq.dtype)
        out, _ = attend(seq, q, 0.25)
        assert torch.equal(out, seq.v[page, 0, i].expand_as(out))


@pytest.mark.parametrize("rows,heads,length", FORMS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [0.3, 3.4, 7.6])
def test_the_heaviest_weight_is_not_rounded(rows, heads, length, kind, bits):
    """Behind many slots with V = 0 comes one of 2^bits times their weight: its value over the sum of weights, rounded once."""
    seq = Sequences([rows], [length], 1, 64, 16, TYPES[kind], seed=5)
    heavy = length - rows
    seq.k.zero_()
    seq.v.zero_()
    seq.k[..., 0] = 4.0 - bits / 8.0
    put(seq, 0, heavy, k=4.0, v=normal(64, seed=3))
    put(seq, 0, heavy, k=0.0, at=slice(1, 64))
    q = torch.zeros(rows, heads, 64, dtype=seq.dtype)
    q[..., 0] = 8.0
    want, _, _, _ = seq.attend(q, math.log(2.0))
    out, _ = attend(seq, q, math.log(2.0))
    # one rounding, scores of up to 32 (2^-24 of it each for product, scale and difference), f32 sums as above
    off = (out.double() - want).abs()
    bound = (half_step(seq.dtype) + 5e-5) * want.abs() + torch.finfo(seq.dtype).tiny * torch.finfo(seq.dtype).eps
    assert (off <= bound).all(), (off / want.abs()).nan_to_num().max().item()


@pytest.mark.parametrize("rows,lens,heads,kv,dim,room", [
    ([1], [1], 1, 1, 64, 0), ([1, 2], [40, 17], 8, 2, 128, 0), ([3], [300], 5, 1, 256, 0), ([2, 1], [90, 33], 6, 2, 200, 0),
    ([1], [2000], 28, 4, 128, 0), ([4], [9000], 4, 1, 72, 0), ([8, 5], [60, 500], 16, 4, 128, 1 << 13),
    ([9], [70], 3, 1, 48, 1 << 15)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_of_few_queries_rounds_once(rows, lens, heads, kv, dim, room, kind):
    """Queries and keys whose scores are exact in f32: what is left is the output's rounding."""
    seq = Sequences(rows, lens, kv, dim, 16, TYPES[kind], seed=3)
    g = torch.Generator().manual_seed(7)
    seq.k = (torch.randint(-8, 9, seq.k.shape, generator=g) / 8).to(seq.dtype)
    q = (torch.randint(-8, 9, (seq.total, heads, dim), generator=g) / 8).to(seq.dtype)
    scale = dim ** -0.5
    want, _, _, _ = seq.attend(q, scale)
    out, _ = attend(seq, q, scale, room=room)
    values = seq.v
    seq.v = values.abs()
    size = seq.attend(q, scale)[0]
    # Products of eighths add up exactly, to scores of 6 at most after the scale (2^-24 of it for product, scale and
    # difference each, 1.1e-6), exp2 2^-23; a weight's two values leave half a step of half a step; f32 sums of 9000 / 64
    # products of 32 a wave, 8 waves and 40 parts, 1.2e-5.
    step = half_step(seq.dtype)
    bound = size * (step * step + 1.4e-5) + step * (want.abs() + size * 2e-5) + torch.finfo(seq.dtype).tiny * torch.finfo(seq.dtype).eps
    off = (out.double() - want).abs()
    assert (off <= bound).all(), ((off - bound) / size).max().item()


@pytest.mark.parametrize("rows,heads,length", FORMS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [1, 60, 140, 240])
def test_infinities_reach_every_row_that_sees_them(rows, heads, length, kind, bits):
    """Infinite and NaN V of slots with 2^-bits of the other slots' weight: early ones that all rows see, at places of a tile
    that they see whole, and one among the new rows. Whatever the weight rounds to, rows that see them have them."""
    seq = Sequences([rows], [length], 1, 64, 16, TYPES[kind], seed=bits)
    seq.k.zero_()
    seq.k[..., 0] = 4.0
    first = length - rows
    odd = {2: (0, math.inf), 5: (first // 2, -math.inf), 7: (100, math.nan), 11: (first - 1, math.inf), 13: (first + rows // 2, math.inf)}
    for t, _ in odd.values():
        put(seq, 0, t, k=4.0 - bits / 16.0, at=0)
    q = torch.zeros(rows, heads, 64, dtype=seq.dtype)
    q[..., 0] = 16.0
    want, _, bound, _ = seq.attend(q, math.log(2.0))
    for column, (t, x) in odd.items():
        put(seq, 0, t, v=x, at=column)
    out, lse = attend(seq, q, math.log(2.0))
    assert torch.isfinite(lse).all()
    for column, (t, x) in odd.items():
        sees = max(0, t - first)  # the first row that sees it
        off = (out[:sees, :, column].double() - want[:sees, :, column]).abs()
        assert (off <= bound[:sees, :, column]).all()
        got = out[sees:, :, column]
        assert torch.isnan(got).all() if x != x else (got == x).all(), (column, t, x)
    plain = [c for c in range(64) if c not in odd]
    assert ((out.double() - want).abs() <= bound)[..., plain].all()


@pytest.mark.parametrize("rows,heads,length", FORMS)
@pytest.mark.parametrize("dim", [40, 96, 128, 200])
def test_infinities_of_both_signs_make_nan(rows, heads, length, dim):
    seq = Sequences([rows], [length], 2, dim, 16, torch.float16, seed=3)
    want, _, bound, _ = seq.attend(q := normal(rows, 2 * heads, dim, seed=4).half(), 0.125)
    put(seq, 0, 0, v=math.inf, at=9)
    put(seq, 0, length - rows - 1, v=-math.inf, at=9)
    out, _ = attend(seq, q, 0.125)
    assert torch.isnan(out[..., 9]).all()
    plain = torch.arange(dim) != 9
    assert ((out.double() - want).abs() <= bound)[..., plain].all()


# ---------------------------------------------------------------- rows and lengths beyond a batch's bounds

BOUNDS = [([3, 2, 1], [20, 33, 100], 2, 30), ([1, 1, 1], [30, 31, 29], 1, 30), ([40, 30, 3], [60, 300, 700], 35, 290),
          ([70, 5, 2], [20, 5, 500], 60, 400)]


def step(seq, heads, rows, length):
    """A cache on the GPU, a batch of max_rows and max_length, and random queries."""
    kp, vp, w, pos, table, lengths, starts = seq.to_gpu()
    return jf.PagedCache(kp, vp, w, pos), jf.PagedBatch(table, lengths, starts, rows, length), normal(seq.total, heads, seq.dim, seed=9).half()


@pytest.mark.parametrize("rows,lens,max_rows,max_length", BOUNDS)
def test_appended_rows_beyond_the_bounds_are_not_written(rows, lens, max_rows, max_length):
    """Those within them go to the slots where they would go without: a longer sequence loses nothing that it has."""
    seq = Sequences(rows, lens, 2, 64, 16, torch.float16, seed=4)
    cache, batch, x = step(seq, 4, max_rows, max_length)
    positions = torch.arange(1, seq.total + 1, dtype=torch.int32)
    cache.append(batch, x[:, :2].cuda(), x[:, 2:].cuda(), positions.cuda())
    for s in range(len(rows)):
        for i in range(min(rows[s], max_rows)):
            t = lens[s] - rows[s] + i
            if 0 <= t < max_length:
                page, place = seq.slot(s, t)
                row = seq.starts[s] + i
                seq.k[page, :, place], seq.v[page, :, place] = x[row, :2], x[row, 2:]
                seq.weights[page, :, place], seq.positions[page, :, place] = 0.0, positions[row]
    assert torch.equal(cache.k.cpu(), seq.k) and torch.equal(cache.v.cpu(), seq.v)
    assert torch.equal(cache.weights.cpu(), seq.weights) and torch.equal(cache.positions.cpu(), seq.positions)


@pytest.mark.parametrize("rows,lens,max_rows,max_length", BOUNDS)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_and_weights_within_bounds(rows, lens, max_rows, max_length, causal):
    """Rows beyond max_rows are left out; the others see what they see without bounds, of the first max_length slots."""
    seq = Sequences(rows, lens, 2, 64, 16, torch.float16, seed=5)
    cache, batch, q = step(seq, 8, max_rows, max_length)
    whole = seq.sees
    seq.sees = lambda s, causal, there: (whole(s, causal, there) & (torch.arange(seq.lens[s]) < max_length)
                                         & (torch.arange(seq.rows[s]) < max_rows)[:, None])
    want, want_lse, bound, lse_bound = seq.attend(q, 0.125, causal)
    out, lse = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda"), torch.full(q.shape[:2], 5.0, device="cuda")
    cache.attend(batch, q.cuda(), 0.125, causal, out=out, lse=lse)
    out, lse = out.cpu(), lse.cpu()
    for s in range(len(rows)):
        r0, r1, r2 = seq.starts[s], seq.starts[s] + min(rows[s], max_rows), seq.starts[s + 1]
        assert ((out[r0:r1].double() - want[r0:r1]).abs() <= bound[r0:r1]).all()
        some = want_lse[r0:r1] > -math.inf
        assert (lse[r0:r1][~some] == -math.inf).all()
        assert ((lse[r0:r1].double() - want_lse[r0:r1]).abs()[some] <= lse_bound[r0:r1][some]).all()
        assert (out[r1:r2] == 7).all() and (lse[r1:r2] == 5).all()
    given = want_lse.float()
    cache.weigh(batch, q.cuda(), given.cuda(), 0.125, causal)
    want, bound = seq.weigh(q, given, 0.125, causal)
    assert ((cache.weights.cpu().double() - want).abs() <= bound).all()


# ---------------------------------------------------------------- handles and tensors

def test_a_closed_rotation_appends_nothing():
    seq = Sequences([3], [20], 2, 64, 16, torch.float16, seed=1)
    cache, batch, x = step(seq, 4, 3, 20)
    x, positions, rope = x.cuda(), torch.arange(3, dtype=torch.int32, device="cuda"), jf.Rope(64)
    rope.close()
    with pytest.raises(jf.InvalidArgument, match="closed"):
        cache.append(batch, x[:, :2], x[:, 2:], positions, rope)
    with pytest.raises(jf.InvalidArgument, match="rotation is required"):
        rope.rotate(x, positions)
    assert torch.equal(cache.k.cpu(), seq.k) and torch.equal(cache.v.cpu(), seq.v)


def test_handles_keep_their_tensors():
    seq = Sequences([2], [20], 2, 64, 16, torch.float16, seed=1)
    kp, vp, w, pos, table, lengths, starts = seq.to_gpu()
    cache, batch = jf.PagedCache(kp, vp, w, pos), jf.PagedBatch(table, lengths, starts, 2, 20)
    assert cache.k is kp and cache.v is vp and cache.weights is w and cache.positions is pos and cache.device == 0
    assert batch.table is table and batch.lengths is lengths and batch.row_starts is starts and batch.device == 0
    for handle, name in ((cache, "k"), (cache, "weights"), (batch, "lengths"), (batch, "table")):
        with pytest.raises(AttributeError):
            setattr(handle, name, getattr(handle, name).clone())
    assert jf.PagedCache(kp, vp).weights is None


def test_tensors_that_require_gradients_are_refused():
    seq = Sequences([2], [20], 2, 64, 16, torch.float16, seed=1)
    cache, batch, q = step(seq, 4, 2, 20)
    kp, q, positions = cache.k.clone().requires_grad_(), q.cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    grad = q.clone().requires_grad_()
    out, lse = cache.attend(batch, q)
    calls = [("x", lambda: jf.Rope(64).rotate(grad, positions)), ("out", lambda: jf.Rope(64).rotate(q, positions, out=grad)),
             ("k", lambda: cache.append(batch, grad[:, :2], q[:, 2:], positions)),
             ("v", lambda: cache.append(batch, q[:, :2], grad[:, 2:], positions)),
             ("q", lambda: cache.attend(batch, grad)), ("lse", lambda: cache.attend(batch, q, lse=lse.clone().requires_grad_())),
             ("q", lambda: cache.weigh(batch, grad, lse)), ("k", lambda: jf.PagedCache(kp, cache.v)),
             ("v", lambda: jf.PagedCache(cache.k, kp))]
    for name, call in calls:
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            call()
    with torch.no_grad():
        again, _ = cache.attend(batch, grad)
    assert torch.equal(again, out)


def test_numbers_beyond_32_bits_are_refused_not_cut():
    seq = Sequences([0], [40], 2, 64, 16, torch.float16, seed=1)
    cache, batch, _ = step(seq, 4, 1, 40)
    far = 1 << 32
    for args in ((far + 20,), (20 - far,), (20, far + 4), (20, 4, far + 1), (20, -1), (-5,)):
        with pytest.raises(jf.InvalidArgument, match="must be 0 to"):
            cache.evict(batch, *args)
    assert batch.lengths.tolist() == [40]
    for rows, length in ((far + 1, 40), (1, far + 40), (-1, 40), (1, -1)):
        with pytest.raises(jf.InvalidArgument, match="must be 0 to"):
            jf.PagedBatch(batch.table, batch.lengths, batch.row_starts, rows, length)
    cache.evict(batch, 20)
    assert batch.lengths.tolist() == [20]


# ---------------------------------------------------------------- attention weights

@pytest.mark.parametrize("max_rows", [1, 100])
@pytest.mark.parametrize("low", [-40.0, 12.0, 60.0])
def test_weights_keep_the_bits_of_lse(max_rows, low):
    """Scores of 0: each slot gets exp(-lse) of its sequence's one row, in either form."""
    n = 100
    seq = Sequences([1] * n, [1] * n, 1, 64, 1, torch.float16, seed=1)
    seq.k.zero_()
    seq.weights.zero_()
    cache, batch, q = step(seq, 1, max_rows, 1)
    lse = torch.rand(n, 1, generator=torch.Generator().manual_seed(3)) * 20 + low
    cache.weigh(batch, q.cuda(), lse.cuda())
    got = torch.stack([cache.weights[seq.slot(s, 0)[0], 0, 0] for s in range(n)]).cpu().double()
    want = torch.exp(-lse[:, 0].double())
    # the lse's two parts leave 2^-48 of it, exp2 is off by 2^-23, the factor of the second part and the sum by 2^-24 each
    off = ((got - want) / want).abs().max().item()
    assert off <= 2.0**-22, off


def test_weights_of_rows_without_a_finite_lse():
    """-inf: the row saw nothing and adds nothing; inf: its weights are 0; NaN: what it sees becomes NaN, nothing else."""
    for rows, heads in ((5, 2), (70, 2)):
        seq = Sequences([rows], [rows + 9], 1, 64, 16, torch.float16, seed=2)
        cache, batch, q = step(seq, heads, rows, rows + 9)
        lse = seq.attend(q, 0.125)[1].float()
        lse[1, 0], lse[2, 1] = -math.inf, math.inf
        some = lse.clone()
        some[2, 1] = -math.inf  # adds as little
        want, bound = seq.weigh(q, some, 0.125)
        cache.weigh(batch, q.cuda(), lse.cuda(), 0.125)
        assert ((cache.weights.cpu().double() - want).abs() <= bound).all()
        lse[3, 1] = math.nan
        cache.weigh(batch, q.cuda(), lse.cuda(), 0.125)
        for t in range(rows + 9):
            page, i = seq.slot(0, t)
            assert torch.isnan(cache.weights[page, 0, i]).item() == (t <= 9 + 3)


# ---------------------------------------------------------------- every slot

@pytest.mark.parametrize("rows,heads,length,dim,room", [
    (1, 16, 40000, 64, 0), (1, 4, 2049, 128, 0), (4, 4, 5000, 72, 0), (2, 8, 4097, 200, 0), (1, 16, 3000, 256, 0),
    (2, 16, 9000, 128, 1 << 15), (40, 2, 6001, 64, 0), (9, 5, 4096, 128, 0), (33, 4, 20000, 96, 0), (20, 2, 2500, 256, 0),
    (300, 1, 3000, 128, 0), (130, 7, 257, 136, 0)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_every_slot_is_seen_once(rows, heads, length, dim, room, kind):
    """Keys of random signs, each row's query one of the keys that it sees: that slot takes all weight, so a slot that is
    lost, or counted twice, at any seam of tiles, waves, parts or the causal end shows at once."""
    seq = Sequences([rows], [length], 1, dim, 16, TYPES[kind], seed=dim)
    g = torch.Generator().manual_seed(5)
    seq.k = (torch.randint(0, 2, seq.k.shape, generator=g) * 2 - 1).to(seq.dtype)
    kp, vp, _, _, table, lengths, starts = seq.to_gpu()
    slots = torch.arange(length, device="cuda")
    page, place = table[0, slots // 16].long(), slots % 16
    k, v = kp[page, 0, place], vp[page, 0, place]
    wide = torch.cat([table, torch.full((1, room), -1, dtype=torch.int32, device="cuda")], 1)
    cache = jf.PagedCache(kp, vp)
    batch = jf.PagedBatch(wide, lengths, starts, rows, wide.shape[1] * 16 if room else length)
    scale = 192.0 / dim  # a score of 192
    sees = length - rows + 1 + torch.arange(rows, device="cuda")[:, None]
    query = torch.arange(rows * heads, device="cuda").reshape(rows, heads)
    some = min(2000, length)
    most = (k.float()[:some] @ k.float().T - 2 * dim * torch.eye(some, length, device="cuda")).max().item()
    assert (dim - most) * scale > 40  # others' weights are below e^-40 each
    for call in range(-(-length // (rows * heads))):
        target = (query + call * rows * heads) % sees
        out, lse = cache.attend(batch, k[target], scale)
        assert torch.equal(out, v[target]), call
        # a second count of the slot would add ln 2; the score and its logarithm keep 2^-22 of 192
        assert (lse - 192.0).abs().max() < 1e-3
    if rows > 1:  # the slot behind a row's own is not seen
        target = torch.cat([sees[:-1], sees[:1] - 1]).expand(rows, heads)
        out, lse = cache.attend(batch, k[target], scale)
        assert (lse[:-1] < 192 - 40).all() and (lse[-1] - 192.0).abs().max() < 1e-3
        assert torch.isfinite(out.float()).all()


def test_threads_share_a_batch():
    """Four threads, each on a stream of its own, with one cache and one batch."""
    import threading

    seq = Sequences([1, 3], [5000, 700], 2, 64, 16, torch.float16, seed=4)
    cache, batch, q = step(seq, 8, 3, 5000)
    queries = [normal(4, 8, 64, seed=50 + n).half().cuda() for n in range(4)]
    want = [cache.attend(batch, x)[0] for x in queries]
    torch.cuda.synchronize()
    failed = []

    def run(n):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [cache.attend(batch, queries[n])[0] for _ in range(50)]
        stream.synchronize()
        if not all(torch.equal(x, want[n]) for x in got):
            failed.append(n)

    threads = [threading.Thread(target=run, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("heads,kv", [(100, 1), (71, 1), (130, 2)])
@pytest.mark.parametrize("rows,lens", [([1, 1], [300, 40]), ([3, 70], [300, 90])])
def test_more_heads_of_a_kv_head_than_a_tile_of_queries(heads, kv, rows, lens):
    """A row's heads span tiles: 64 queries of the weights, 128 and 32 of attention."""
    seq = Sequences(rows, lens, kv, 64, 16, torch.float16, seed=heads)
    cache, batch, q = step(seq, heads, seq.max_rows, seq.max_length)
    want, want_lse, bound, lse_bound = seq.attend(q, 0.125)
    out, lse = cache.attend(batch, q.cuda(), 0.125)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert ((lse.cpu().double() - want_lse).abs() <= lse_bound).all()
    cache.weigh(batch, q.cuda(), lse, 0.125)
    want, bound = seq.weigh(q, lse.cpu(), 0.125)
    assert ((cache.weights.cpu().double() - want).abs() <= bound).all()


def test_expanded_rows_are_read():
    """One row for all, one head for all: stride 0 in what a call reads."""
    seq = Sequences([4], [50], 2, 64, 16, torch.float16, seed=6)
    cache, batch, x = step(seq, 4, 4, 50)
    one = x[:1, :1].expand(4, 4, 64)
    want, _, bound, _ = seq.attend(one, 0.125)
    out, _ = cache.attend(batch, x.cuda()[:1, :1].expand(4, 4, 64), 0.125)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    gpu, positions = x.cuda(), torch.arange(46, 50, dtype=torch.int32, device="cuda")
    rope = jf.Rope(64)
    wide = rope.rotate(gpu[:1, :1].expand(4, 2, 64), positions)
    assert torch.equal(wide, rope.rotate(gpu[:1, :1].expand(4, 2, 64).contiguous(), positions))
    cache.append(batch, gpu[:1, :1].expand(4, 2, 64), gpu[:, :1].expand(4, 2, 64), positions, rope)
    for i in range(4):
        page, place = seq.slot(0, 46 + i)
        assert torch.equal(cache.k[page, :, place], wide[i]) and torch.equal(cache.v[page, :, place], gpu[i, :1].expand(2, 64))
