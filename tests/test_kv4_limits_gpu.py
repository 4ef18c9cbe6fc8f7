"""The 4-bit paged cache at its limits: lengths that its tables do not hold, pools that run out."""
import pytest
import torch

from oumu_b200 import ops
from oumu_b200.kv4 import KV4Cache
from test_kv4_gpu import LENGTH, attn_case, i32, randn, run_attn

pytestmark = pytest.mark.gpu


# ---- lengths that the tables do not hold ----

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("what", ["table", "rotary", "position"])
def test_a_step_past_the_end_writes_nothing(cuda, what, hd):
    """Three takes share two full pages; one is stepped past what its table row, or the rotary tables, can hold: the
    pool keeps its bytes and the other takes their outputs."""
    nq, nk, B = 8, 2, 3
    qkv, pool, rows, table, ln = attn_case([128], nq, nk, hd, seed=90)
    table = table.repeat(B, 1).contiguous()
    qkv = randn(91, B, (nq + 2 * nk) * hd)
    cs, sn = (t.cuda() for t in ops.rotary_tables(100 if what == "rotary" else 128, hd))
    before, want = pool.clone(), run_attn(qkv, pool, table, i32([128] * B), B, nq, nk, hd)
    ws = ops.decode_kv4_workspace(B, nq, nk, hd, 2)
    out = torch.empty(B, nq * hd, dtype=torch.bfloat16, device="cuda")
    lens = None if what == "position" else i32([0, 120 if what == "rotary" else 129, 0])
    pos = i32([128]) if what == "position" else None
    ops.attn_decode_kv4_step(qkv, pool, out, ws, cs, sn, table, pos, lens, B, nq, nk, hd, hd ** -0.5)
    assert ops.device_error(reset=True) == LENGTH
    assert torch.equal(pool, before)
    assert torch.equal(run_attn(qkv, pool, table, i32([128] * B), B, nq, nk, hd), want)


# ---- the cache's own calls ----

def test_pages_a_fork_lacked_stay_visible(cuda):
    """A fork that finds no page leaves its takes empty; the extend behind it, which then lacks nothing, and a second
    fork do not hide that."""
    c = KV4Cache(1, 4, 8, 2, 64, 4, 256)
    c.lens[0] = 100
    c.extend()
    c.fork([0, 0, 0], [1, 2, 3])  # a page each for their second pages: two there are
    c.extend()
    assert c.missing() == 1
    assert c.lens.tolist() == [100, 100, 100, 0]
    assert c.missing() == 0
    c.fork([0], [3])
    c.free([1])
    c.fork([0], [1])
    c.extend()
    assert c.missing() == 1 and c.missing() == 0


def test_pages_an_extend_lacked_stay_visible(cuda):
    c = KV4Cache(1, 3, 8, 2, 64, 3, 256)
    c.lens.copy_(i32([64, 128, 64]))
    c.extend()
    c.free([0])
    c.extend()  # now there is a page, but the positions in between were not written
    assert c.missing() == 1 and c.missing() == 0
