"""The 4-bit paged cache at its limits: lengths that its tables do not hold."""
import pytest
import torch

from oumu_b200 import ops
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
