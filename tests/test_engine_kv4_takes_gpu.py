"""Takes of Engine(kv="int4") that stop or are freed while others go on, or are given lengths they do not hold."""
import pytest
import torch

from oumu_b200 import engine, ops
from test_engine_kv4_gpu import make, slots

pytestmark = pytest.mark.gpu


def test_a_stopped_take_takes_no_more_pages(cuda):
    """Take 0 has stopped at 59 positions: it stays there (the step's own position behind them apart), and the pool, which
    has no page for its 65th, lasts for the takes that go on."""
    e = make(3, kv_pages=5, min_len=10 ** 6)
    e.prime([60, 100, 110])
    e.stop[0] = 0
    before = [slots(e, l) for l in range(3)]
    for _ in range(8):
        e.step()
    torch.cuda.synchronize()
    assert e.lens.tolist() == [60, 108, 118]
    e.kv4.extend()
    assert int(e.kv4.status[0]) == 0 and ops.device_error() == 0
    for l in range(3):
        for a, b in zip(before[l], slots(e, l)):
            assert torch.equal(a[0, :, :59], b[0, :, :59])
    g = e.capture()  # and a step of its own
    g.replay()
    torch.cuda.synchronize()
    assert e.lens.tolist() == [60, 110, 120] and int(e.kv4.status[0]) == 0 and ops.device_error() == 0


def test_what_a_take_holds_when_it_stops_is_kept(cuda):
    """The stop logits ask every take to stop after 2 patches: the position of that step is the last that counts, and no
    later step writes it again."""
    B = 2
    e = make(B, min_len=1)
    e.prime([70, 90])
    e.stop_head = lambda x, out: out[:, 1].fill_(1.0)  # the stop logits, whatever the state says
    e.stop_l.zero_()
    for _ in range(3):
        e.step()
    torch.cuda.synchronize()
    assert e.stop.tolist() == [2, 2]  # the third patch is number 2, more than min_len
    held = e.lens.tolist()
    assert held == [73, 93]
    kept = [slots(e, l, 1) for l in range(3)]
    for _ in range(4):
        e.step()
    torch.cuda.synchronize()
    assert e.lens.tolist() == held
    for l in range(3):
        for a, b in zip(kept[l], slots(e, l, 1)):
            assert torch.equal(a, b)
    assert ops.device_error() == 0


def test_a_freed_take_stays_free(cuda):
    e = make(3, min_len=10 ** 6)
    e.prime([65, 70, 80])
    used = int((e.kv4.ref > 0).sum())
    e.step()
    e.kv4.free([1])
    for _ in range(3):
        e.step()
    torch.cuda.synchronize()
    assert e.lens.tolist() == [69, 0, 84]
    assert e.kv4.table[1].max().item() == -1 and int((e.kv4.ref > 0).sum()) == used - 2
    assert ops.device_error() == 0
    # decode on: the other takes from where they are
    e.set_lens([60, 0, 80])
    e.step()
    torch.cuda.synchronize()
    assert e.lens.tolist() == [61, 0, 81] and ops.device_error() == 0


def test_set_lens_refuses_positions_that_no_take_holds(cuda):
    e = make(2)
    e.prime([70, 100])
    with pytest.raises(ValueError):
        e.set_lens([71, 100])  # position 70 would be read as the page was left
    with pytest.raises(ValueError):
        e.set_lens([70, 300])
    with pytest.raises(ValueError):
        e.set_lens([0, 100])
    e.set_lens([70, 100])
    e.step()
    torch.cuda.synchronize()
    assert e.lens.tolist() == [71, 101]
    e.set_lens([71, 90])
    e.step()
    torch.cuda.synchronize()
    assert e.lens.tolist() == [72, 91] and ops.device_error() == 0
    b = make(2, kv="bf16")
    b.prime([70, 100])
    b.set_lens([200, 300])  # bf16 slots are filled to their ends


def test_set_lens_refuses_positions_that_takes_share(cuda):
    e = make(2)
    e.prime([130, 70])
    e.kv4.fork([0], [1])  # positions 0..127 on shared pages
    with pytest.raises(ValueError):
        e.set_lens([100, 130])
    with pytest.raises(ValueError):
        e.set_lens([130, 128])
    e.set_lens([129, 130])
    with pytest.raises(ValueError):
        e.set_lens([129])


def test_a_pool_that_runs_out_is_noticed_at_once(cuda):
    """The loop that steps from the host raises at the step that lacks a page, not at the end."""
    e = make(2, kv_pages=3, min_len=10 ** 6, max_steps=200)
    e.prime([60, 100])
    g = e.capture()
    e.set_lens([60, 100])
    with pytest.raises(RuntimeError, match="missing"):
        e.decode(g, device_loop=False)
    torch.cuda.synchronize()
    assert int(e.ctr[1]) < 10
    ops.device_error(reset=True)


def test_step_end_live_exact(cuda):
    B, max_steps = 7, 5
    logits = torch.tensor([[0, 1], [1, 0], [0, 1], [1, 0], [0, 1], [1, 0], [0, 1]], dtype=torch.bfloat16, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    patch, patches = logits.new_ones(B, 256), logits.new_zeros(B, max_steps, 256)
    stop, ctr, lens = i32([-1, -1, 1, 1, -1, -1, 2]), i32([100, 3, 0, 0]), i32([50, 51, 52, 53, 0, 0, 1])
    ops.step_end(logits, patch, patches, stop, ctr, lens, B, 2, max_steps, live=True)
    assert stop.tolist() == [3, -1, 1, 1, 3, -1, 2]
    assert lens.tolist() == [51, 52, 52, 53, 0, 0, 1] and ctr.tolist()[:2] == [101, 4]
    assert bool((patches[:, 3] == 1).all()) and int(patches.float().sum()) == B * 256
    with pytest.raises(RuntimeError):
        ops.step_end(logits, patch, patches, stop, ctr, None, B, 2, max_steps, live=True)
