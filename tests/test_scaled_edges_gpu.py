"""GPU: the cache of 8-bit rows where its operators meet what surrounds them: arrays that the launch before makes, loud and tiny
neighbours, what lies beside a sequence's own rows, arguments between the kernels' ranges.  Formulas and bounds as in
test_scaled_cache_gpu.py."""

import pytest
import torch

from test_scaled_cache_gpu import DEV, Cache, kernels, quantise, rows_of

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
