"""GPU: the cache of 8-bit rows where its operators meet what surrounds them: arrays that the launch before makes, loud and tiny
neighbours, what lies beside a sequence's own rows, arguments between the kernels' ranges.  Formulas and bounds as in
test_scaled_cache_gpu.py."""

import pytest
import torch

from test_scaled_cache_gpu import DEV, FMT, PAGE, Cache, attend, check, kernels, quantise, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [5, 200])
def test_positions_that_the_launch_before_makes(T):
    """Sequences and positions come out of an argmax right ahead of the write, over arrays that held other valid places."""
    G, D, lengths = 2, 64, [150, 150]
    c = Cache(lengths, G, D, "int8")
    V = 40000
    logits = torch.zeros(2 * T, V, device=DEV)
    places = torch.zeros(2 * T, dtype=torch.int32, device=DEV)
    g = torch.Generator(DEV).manual_seed(1)
    for turn in range(4):
        where = torch.randperm(300, generator=g, device=DEV)[:T]
        seq, pos = (where // 150).int(), (where % 150).int()
        logits.zero_()
        logits[torch.arange(2 * T, device=DEV), torch.cat([seq, pos]).long()] = 1.0
        places[:T], places[T:] = 0, torch.arange(T, device=DEV) % 150
        for scale in (c.ks, c.vs):
            scale.fill_(7.0)
        qkv = torch.randn(T, 3 * G * D, generator=g, device=DEV)
        q = torch.empty(T, G * D, device=DEV)
        torch.cuda.synchronize()
        kernels().argmax(logits, places)
        kernels().scaled_cache_write(qkv, q, *c.args(), places[:T], places[T:], None, None, 0.0, None, None, 0, G, G, D)
        torch.cuda.synchronize()
        for store, scale, part in ((c.k, c.ks, qkv[:, G * D : 2 * G * D]), (c.v, c.vs, qkv[:, 2 * G * D :])):
            held, s = quantise(part.reshape(T, G, D), "int8")
            assert torch.equal(rows_of(store, c, seq, pos), held) and torch.equal(rows_of(scale, c, seq, pos), s)
            assert int((scale != 7.0).sum()) == T * G          # and nowhere else
    kernels().check_status()


def attention_calls(D):
    """(name, types of queries, call(q, out, cache, positions of sequences of one token)): single tokens and both kernels of several."""
    def chunk(tc):
        def run(q, out, c, pos, H, shares):
            start = torch.arange(len(q) + 1, dtype=torch.int32, device=DEV)
            kernels().scaled_attention_chunk(q, out, *c.args(), start, pos, len(q), 1, H, c.G, c.D, None, c.D ** -0.5, n_shares=shares, tc=tc)
        return run

    def decode(q, out, c, pos, H, shares):
        kernels().scaled_attention_decode(q, out, *c.args(), pos, H, c.G, c.D, None, c.D ** -0.5, n_shares=shares)

    both = (torch.bfloat16, torch.float32)
    return [("decode", both, decode), ("chunk", both, chunk(False))] + ([("tcgen05", both[:1], chunk(True))] if D in (64, 128) else [])


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("D", [64, 80, 128])
def test_value_scales_of_next_to_nothing(D, fmt):
    """A first page of scales of 2^-120 (no writer makes them, any caller may) ahead of ordinary ones: what they stand for is
    nothing beside the rest, whatever the largest scale was when they were met."""
    H, G, L = 4, 2, 200
    c = Cache([L], G, D, fmt).fill()
    page = int(c.table[0, 0])
    c.V[0][:PAGE] *= 2.0 ** -120 / c.vs[page].T.double().unsqueeze(-1)
    c.vs[page] = 2.0 ** -120
    pos = torch.tensor([L - 1], dtype=torch.int32, device=DEV)
    for name, dtypes, call in attention_calls(D):
        for dtype in dtypes:
            q = torch.randn(1, H * D, generator=torch.Generator(DEV).manual_seed(2), device=DEV).to(dtype)
            want = attend(q.double().view(1, H, D), c.K[0], c.V[0], pos, None, 0, 0, D ** -0.5)
            for shares in (1, 3):
                out = torch.empty_like(q)
                call(q, out, c, pos, H, shares)
                check(out.view(1, H, D), *want, dtype, L)


@pytest.mark.parametrize("D", [64, 80, 128])
def test_queries_of_next_to_nothing(D):
    """Queries of 2^-116 on keys of 2^115: their scores are ordinary."""
    H, G, L = 4, 2, 100
    c = Cache([L], G, D, "int8").fill()
    for page in c.table[0].tolist():
        c.ks[page] *= 2.0 ** 115
    c.K[0] *= 2.0 ** 115
    pos = torch.tensor([L - 1], dtype=torch.int32, device=DEV)
    for name, dtypes, call in attention_calls(D):
        for dtype in dtypes:
            q = (torch.randn(1, H * D, generator=torch.Generator(DEV).manual_seed(2), device=DEV) * 2.0 ** -116).to(dtype)
            want = attend(q.double().view(1, H, D), c.K[0], c.V[0], pos, None, 0, 0, D ** -0.5)
            out = torch.empty_like(q)
            call(q, out, c, pos, H, 1)
            check(out.view(1, H, D), *want, dtype, L)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("D, tc", [(64, False), (80, False), (128, False), (64, True), (128, True)])
def test_a_loud_row_is_nothing_to_those_that_do_not_see_it(D, tc, window, fmt):
    """One value row of a scale 2^40 above the others: whoever does not see it gets, bit for bit, what it got without it."""
    H, G, L, n = 4, 2, 330, 300
    c = Cache([L], G, D, fmt).fill()
    start, past = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, n], [L - n]))
    for dtype in (torch.bfloat16,) if tc else (torch.bfloat16, torch.float32):
        q = torch.randn(n, H * D, generator=torch.Generator(DEV).manual_seed(5), device=DEV).to(dtype)
        run = lambda out: kernels().scaled_attention_chunk(q, out, *c.args(), start, past, 1, n, H, G, D, window, D ** -0.5, n_shares=1, tc=tc)
        clean = torch.empty_like(q)
        run(clean)
        for bad in (60, 191, 300, L - 1):
            page, row = int(c.table[0, bad // PAGE]), bad % PAGE
            scale, values = c.vs[page, :, row].clone(), c.V[0][bad].clone()
            c.vs[page, :, row] *= 2.0 ** 40
            c.V[0][bad] *= 2.0 ** 40
            out = torch.empty_like(q)
            run(out)
            want = attend(q.double().view(n, H, D), c.K[0], c.V[0], torch.arange(L - n, L, device=DEV), window, 0, 0, D ** -0.5)
            c.vs[page, :, row], c.V[0][bad] = scale, values
            at = torch.arange(L - n, L, device=DEV)
            sees = (at >= bad) & (at < bad + (window or L))
            assert torch.equal(out[~sees], clean[~sees]), (bad, dtype)
            if sees.any():
                check(out[sees].view(-1, H, D), *(x[sees] for x in want), dtype, L)


@pytest.mark.parametrize("fmt", list(FMT))
@pytest.mark.parametrize("D", [64, 80, 128])
def test_a_loud_row_that_nobody_weighs(D, fmt):
    """A visible value row 2^30 above the others under a key whose weight is about 2^-60 of the others': they keep their digits.
    What a weight loses at float16's end goes by the row's largest product of probability and value, not by the largest value:
    2^-38 of it, and for several tokens, whose largest weight is kept above 2^10 and not 2^13, 2^-35."""
    H, G, L, loud = 4, 2, 700, 130
    c = Cache([L], G, D, fmt).fill(strength=0.5)
    q0 = torch.randn(D, generator=torch.Generator(DEV).manual_seed(8), device=DEV)
    page, row = int(c.table[0, loud // PAGE]), loud % PAGE
    key = (-42.0 * D ** 0.5 / (q0 @ q0) * q0).expand(G, D)
    held, scale = quantise(key, fmt)
    c.k.view(torch.int8)[page, :, row], c.ks[page, :, row] = held.view(torch.int8), scale
    c.K[0][loud] = held.float().double() * scale.double().unsqueeze(-1)
    c.vs[page, :, row] *= 2.0 ** 30
    c.V[0][loud] *= 2.0 ** 30
    pos = torch.tensor([L - 1], dtype=torch.int32, device=DEV)
    for name, dtypes, call in attention_calls(D):
        for dtype in dtypes:
            q = q0.expand(H, D).reshape(1, H * D).to(dtype)
            x = q.double().view(1, H, D)
            out64, mag, score, _ = attend(x, c.K[0], c.V[0], pos, None, 0, 0, D ** -0.5)
            p = [torch.softmax(c.K[0][:, h // (H // G)] @ x[0, h] * D ** -0.5, 0) for h in range(H)]
            assert all(2.0 ** -68 < float(y[loud] / y.max()) < 2.0 ** -50 for y in p)
            largest = torch.stack([(y * c.V[0][:, h // (H // G)].abs().amax(-1)).max() for h, y in enumerate(p)]).view(1, H, 1)
            for shares in (1, 3):
                out = torch.empty_like(q)
                call(q, out, c, pos, H, shares)
                check(out.view(1, H, D), out64, mag, score, largest * (1 if name == "decode" else 8), dtype, L)


@pytest.mark.parametrize("dtype, tc", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
@pytest.mark.parametrize("shares", [1, 3])
def test_sequences_outside_the_arrays_are_reported(dtype, tc, shares):
    """Starts past the queries, in no order or negative, more tokens than ``max_new`` says, positions before 0 or past the block
    table: nothing outside the arrays is read or written, the other sequence is right, and the host hears of it."""
    from llmoxide_b200.errors import KernelError
    H, G, D = 4, 2, 64
    c = Cache([100, 70], G, D, "int8").fill()
    T, n = 60, 30
    q = torch.randn(T, H * D, generator=torch.Generator(DEV).manual_seed(6), device=DEV).to(dtype)
    want = attend(q[:n].double().view(n, H, D), c.K[0], c.V[0], torch.arange(70, 100, device=DEV), None, 0, 0, D ** -0.5)
    library = "scaled_attention_tc" if tc else "scaled_attention"
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    for start, past, max_new in (([0, n, T + 1], [70, 39], n + 1), ([0, n, 1 << 30], [70, 0], n), ([0, n, n - 5], [70, 40], n),
                                 ([0, n, -7], [70, 40], n), ([0, n, T], [70, -1], n), ([0, n, T], [70, 99], n),
                                 ([0, n, T], [70, (1 << 31) - 8], n), ([0, n, T], [70, -(1 << 31)], n)):
        store = torch.full((T + 64, H * D), 7.0, dtype=dtype, device=DEV)
        kernels().scaled_attention_chunk(q, store[:T], *c.args(), ints(start), ints(past), 2, max_new, H, G, D, None, D ** -0.5,
                                         n_shares=shares, tc=tc)
        torch.cuda.synchronize()
        with pytest.raises(KernelError, match=library + ": a sequence's tokens or positions"):
            kernels().check_status()
        check(store[:n].view(n, H, D), *want, dtype, 100)
        assert (store[T:] == 7.0).all()
    # more tokens than max_new says
    out = torch.full_like(q, 7.0)
    kernels().scaled_attention_chunk(q, out, *c.args(), ints([0, n, T]), ints([70, 40]), 2, n - 1, H, G, D, None, D ** -0.5, n_shares=shares, tc=tc)
    torch.cuda.synchronize()
    with pytest.raises(KernelError, match="a sequence's tokens or positions"):
        kernels().check_status()
    kernels().scaled_attention_chunk(q, out, *c.args(), ints([0, n, T]), ints([70, 40]), 2, n, H, G, D, None, D ** -0.5, n_shares=shares, tc=tc)
    kernels().check_status()
    check(out[:n].view(n, H, D), *want, dtype, 100)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shares", [1, 3, 12])
def test_a_position_past_the_block_table_is_reported(dtype, shares):
    """A single token's: no key is walked to, and the other sequence is right."""
    from llmoxide_b200.errors import KernelError
    H, G, D = 4, 2, 64
    c = Cache([100, 70], G, D, "int8").fill()
    q = torch.randn(2, H * D, generator=torch.Generator(DEV).manual_seed(6), device=DEV).to(dtype)
    for past in (128, 1 << 20, (1 << 31) - 1):
        pos = torch.tensor([99, past], dtype=torch.int32, device=DEV)
        out = torch.full_like(q, 7.0)
        kernels().scaled_attention_decode(q, out, *c.args(), pos, H, G, D, None, D ** -0.5, n_shares=shares)
        torch.cuda.synchronize()
        with pytest.raises(KernelError, match="scaled_attention: a visible key's page"):
            kernels().check_status()
        check(out[:1].view(1, H, D), *attend(q[:1].double().view(1, H, D), c.K[0], c.V[0], pos[:1], None, 0, 0, D ** -0.5), dtype, 100)
        assert (out[1] == 0).all()


@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_what_lies_past_a_sequences_end_is_nobodys(D):
    """Pages that no writer has touched past a sequence's last row, here all bits set: NaN codes in e4m3, under NaN scales."""
    H, G = 4, 2
    past, new = [64, 0, 90, 129], [30, 5, 1, 64]
    for fmt in FMT:
        c = Cache([p + n for p, n in zip(past, new)], G, D, fmt).fill()
        for b, n in enumerate(c.lengths):
            page, row = int(c.table[b, (n - 1) // PAGE]), (n - 1) % PAGE + 1
            for store in (c.k, c.v):
                store.view(torch.int8)[page, :, row:] = -1
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        start, T = [sum(new[:i]) for i in range(len(new) + 1)], sum(new)
        for dtype in (torch.bfloat16, torch.float32):
            q = torch.randn(T, H * D, generator=torch.Generator(DEV).manual_seed(7), device=DEV).to(dtype)
            want = [attend(q[start[b] : start[b] + n].double().view(n, H, D), c.K[b], c.V[b], torch.arange(p, p + n, device=DEV), None, 0, 0,
                           D ** -0.5) for b, (p, n) in enumerate(zip(past, new))]
            for tc in (False, True) if dtype == torch.bfloat16 and D in (64, 128) else (False,):
                for shares in (1, 3):
                    out = torch.empty_like(q)
                    kernels().scaled_attention_chunk(q, out, *c.args(), ints(start), ints(past), len(new), max(new), H, G, D, None, D ** -0.5,
                                                     n_shares=shares, tc=tc)
                    for b, n in enumerate(new):
                        check(out[start[b] : start[b] + n].view(n, H, D), *want[b], dtype, past[b] + n)
            last = torch.tensor(start[1:], device=DEV) - 1
            for shares in (1, 3):
                out = torch.empty(len(new), H * D, dtype=dtype, device=DEV)
                kernels().scaled_attention_decode(q[last], out, *c.args(), ints([n - 1 for n in c.lengths]), H, G, D, None, D ** -0.5,
                                                  n_shares=shares)
                for b in range(len(new)):
                    check(out[b].view(1, H, D), *(x[-1:] for x in want[b]), dtype, c.lengths[b])
    kernels().check_status()


@pytest.mark.parametrize("dtype, tc", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_rows_of_no_sequence_are_left_alone(dtype, tc):
    """Queries before the first sequence's and behind the last one's, as a padded step has them, in one share or several."""
    H, G, D = 4, 2, 64
    c = Cache([700, 70], G, D, "int8").fill()
    T, lo, mid, hi = 40, 3, 13, 20
    q = torch.randn(T, H * D, generator=torch.Generator(DEV).manual_seed(6), device=DEV).to(dtype)
    start, past = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([lo, mid, hi], [690, 63]))
    for shares in (1, 3, 11):
        out = torch.full_like(q, 7.0)
        kernels().scaled_attention_chunk(q, out, *c.args(), start, past, 2, 10, H, G, D, None, D ** -0.5, n_shares=shares, tc=tc)
        assert (out[:lo] == 7.0).all() and (out[hi:] == 7.0).all()
        for b, rows in enumerate((slice(lo, mid), slice(mid, hi))):
            n = rows.stop - rows.start
            at = int(past[b]) + torch.arange(n, device=DEV)
            check(out[rows].view(n, H, D), *attend(q[rows].double().view(n, H, D), c.K[b], c.V[b], at, None, 0, 0, D ** -0.5), dtype, c.lengths[b])
    kernels().check_status()


@pytest.mark.parametrize("name", ["D", "E"])
def test_an_engine_without_tcgen05(tmp_path, monkeypatch, name):
    """``tensor_cores=False``: prompts over 8-bit rows go by the other kernel, and the tcgen05 one is not even loaded.  Bound: as in
    test_scaled_engine_gpu.py, the wide cache's tolerance and twice what rounding the cache does."""
    import numpy as np
    from replay_util import TOL
    from test_scaled_engine_gpu import folder_of, load
    from tiny_configs import ALL
    folder = folder_of(tmp_path, name, "bfloat16")
    toks = np.random.default_rng(3).integers(0, ALL[name]["vocab_size"], 150).tolist()
    called, find = [], kernels()._scaled_fn
    monkeypatch.setattr(kernels(), "_scaled_fn", lambda key: (called.append(key), find(key))[1])
    logits, by = [], []
    for fmt, tensor_cores in (("", True), ("int8", True), ("int8", False)):
        eng = load(folder, "bfloat16", fmt, tensor_cores=tensor_cores)
        del called[:]
        slot = eng.acquire()
        logits.append(torch.cat([eng.step([(slot, toks[:149])], [list(range(149))]), eng.step([(slot, toks[149:])])]).double())
        eng.check_status()
        by.append((set(lib for lib, _ in called), eng.model.libraries()))
    assert "scaled_attention_tc" in by[1][0] and "scaled_attention_tc" in by[1][1]
    assert "scaled_attention_tc" not in by[2][0] and "scaled_attention_tc" not in by[2][1] and "scaled_attention" in by[2][0]
    off = lambda a, b: float((logits[a] - logits[b]).abs().max() / logits[0].abs().max())
    assert off(1, 2) <= TOL["bfloat16"] + 2 * off(0, 1)


@pytest.mark.parametrize("D", [64, 128])
def test_queries_that_start_between_vectors(D):
    """bfloat16 queries and results on 8-byte boundaries: the kernel of 16-byte loads does not take them, the other does."""
    H, G, n = 4, 2, 20
    c = Cache([100], G, D, "int8").fill()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    base = torch.randn(n * H * D + 8, generator=torch.Generator(DEV).manual_seed(6), device=DEV).to(torch.bfloat16)
    q = base[4 : 4 + n * H * D].view(n, H * D)
    want = attend(q.double().view(n, H, D), c.K[0], c.V[0], torch.arange(80, 100, device=DEV), None, 0, 0, D ** -0.5)
    for q_at, out_at in ((4, 0), (0, 4), (4, 4)):
        x = base[:n * H * D].clone().view(n, H * D).copy_(q) if q_at == 0 else q
        store = torch.full((n * H * D + 8,), 7.0, dtype=torch.bfloat16, device=DEV)
        out = store[out_at : out_at + n * H * D].view(n, H * D)
        kernels().scaled_attention_chunk(x, out, *c.args(), ints([0, n]), ints([80]), 1, n, H, G, D, None, D ** -0.5)
        check(out.view(n, H, D), *want, torch.bfloat16, 100)
        one = torch.empty(8 + H * D, dtype=torch.bfloat16, device=DEV)[out_at : out_at + H * D].view(1, H * D)
        kernels().scaled_attention_decode(x[-1:], one, *c.args(), ints([99]), H, G, D, None, D ** -0.5)
        check(one.view(1, H, D), *(y[-1:] for y in want), torch.bfloat16, 100)
    kernels().check_status()
