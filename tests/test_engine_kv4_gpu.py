"""The decoding step over the 4-bit paged cache (Engine(kv="int4")): what a layer writes and attends, a shared prompt,
the captured step and the decoding loop, a pool that is too small."""
import pytest
import torch

import kv4_ref as ref
from oumu_b200 import engine, ops

pytestmark = pytest.mark.gpu

SMALL = dict(base_layers=2, res_layers=1, enc_layers=1, dit_layers=1)


def make(B, **kw):
    return engine.Engine(B, **{**dict(maxlen=320, max_steps=8, kv="int4"), **SMALL, **kw})


def slots(e, layer, ahead=0):
    """What the takes hold, as bf16 slots; after a step lens is one `ahead` of it."""
    kc = torch.zeros(e.B, engine.NK, e.maxlen, engine.HD, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    ops.kv4_read(e.kv4.pools[layer], e.kv4.table, e.lens - ahead, kc, vc, engine.NK, engine.HD)
    return kc, vc


def test_a_layer_writes_and_attends_over_the_cache(cuda):
    B, lens = 4, [70, 1, 64, 200]
    e = make(B)
    e.prime(lens)
    before = [slots(e, l) for l in range(3)]
    e.step()
    torch.cuda.synchronize()
    sc = e._scratch[(B, engine.LM)]  # what the last layer, the residual LM's (no rope), left
    x = sc["qkv"].cpu().double().view(B, -1, engine.HD)
    pool, rows = e.kv4.pools[2].cpu(), e.kv4.table.tolist()
    kc, vc = slots(e, 2, 1)
    for s, n in enumerate(lens):
        k, v, _ = ref.take_values(pool, rows[s], n, engine.NK, engine.HD)
        new = ref.held(x[s, engine.NQ:])[3]
        assert torch.equal(k[:, n - 1], new[:engine.NK]) and torch.equal(v[:, n - 1], new[engine.NK:])
        assert torch.equal(kc[s, :, :n - 1], before[2][0][s, :, :n - 1])
        assert torch.equal(vc[s, :, :n - 1], before[2][1][s, :, :n - 1])
        got = sc["att"][s].cpu().double().view(engine.NQ, engine.HD)
        want = ref.attend(x[s, :engine.NQ], k, v, engine.HD ** -0.5)
        # p s in fp16 (2^-11) times codes of at most 15: 15 s <= the spread (1 + 2^-7); the output's bf16 rounding
        spread = (v.amax((1, 2)) - v.amin((1, 2))).repeat_interleave(8)[:, None]
        tol = want.abs() * 2 ** -8 + spread * (1 + 2 ** -7) * (2 ** -11 + 2 ** -14) + v.abs().max() * 2 ** -14
        assert bool(((got - want).abs() <= tol).all())
    for l in range(2):  # the layers before wrote their newest position too, and nothing else
        kc, vc = slots(e, l, 1)
        for s, n in enumerate(lens):
            assert torch.equal(kc[s, :, :n - 1], before[l][0][s, :, :n - 1])
            assert not torch.equal(vc[s, :, n - 1], before[l][1][s, :, n - 1])
    assert e.lens.tolist() == [n + 1 for n in lens] and ops.device_error() == 0


def test_a_shared_prompt_is_held_once(cuda):
    B, prompt = 5, 150
    e = make(B)
    e.prime([prompt + 1 + 3 * s for s in range(B)], prompt=prompt)
    used = int((e.kv4.ref > 0).sum())
    assert used == 2 + B  # two full pages for all, a page of its own for each take's rest
    assert e.kv4.ref.max().item() == B
    for l in range(3):
        for c in slots(e, l):
            assert bool((c[:, :, :prompt] == c[:1, :, :prompt]).all())
    before = [slots(e, l) for l in range(3)]
    for _ in range(4):
        e.step()
    torch.cuda.synchronize()
    for l in range(3):
        for a, b in zip(before[l], slots(e, l, 1)):
            assert torch.equal(a[:, :, :prompt], b[:, :, :prompt])
    with pytest.raises(ValueError):
        e.set_lens([prompt] * B)
    e.prime([20] * B)  # the next text: everything is given back first
    assert int((e.kv4.ref > 0).sum()) == B and ops.device_error() == 0


def test_bf16_slots_with_a_shared_prompt(cuda):
    e = make(3, kv="bf16")
    e.prime([100, 120, 140], prompt=90)
    for c in e.base.kc + e.res.vc:
        assert bool((c[:, :, :90] == c[:1, :, :90]).all())
        assert not torch.equal(c[0, :, 90:100], c[1, :, 90:100])


def test_captured_step_and_loop_match_eager_steps(cuda):
    B, lens, steps = 3, [60, 127, 190], 7

    def run(how):
        e = make(B, max_steps=steps + 1, min_len=10 ** 6, seed=3)
        if how != "eager":
            e.prime(lens)
            g = e.capture(keep_graph=how == "loop")
        e.prime(lens)
        if how == "eager":
            for _ in range(steps + 1):
                e.step()
        elif how == "replay":
            for _ in range(steps + 1):
                g.replay()
        else:
            assert e.decode(g, device_loop=True) == [steps + 1] * B
        torch.cuda.synchronize()
        assert ops.device_error() == 0
        return e.patches.clone(), e.lens.tolist(), [torch.cat(slots(e, l, 1)) for l in range(3)]

    eager, replay, loop = (run(h) for h in ("eager", "replay", "loop"))
    for got in (replay, loop):
        assert torch.equal(got[0], eager[0]) and got[1] == eager[1]
        assert all(torch.equal(a, b) for a, b in zip(got[2], eager[2]))


def test_a_pool_that_is_too_small_is_an_error(cuda):
    e = make(4, kv_pages=7, min_len=10 ** 6)  # no take stops: the fourth reaches its 65th position
    with pytest.raises(RuntimeError, match="1 pages are missing"):
        e.prime([100] * 4)
    e.prime([100, 100, 100, 60])
    g = e.capture()  # the capture's own eager step
    e.set_lens([100, 100, 100, 60])
    with pytest.raises(RuntimeError, match="missing"):
        e.decode(g, device_loop=False)
    ops.device_error(reset=True)
    with pytest.raises(ValueError):
        make(2, kv="int8")
