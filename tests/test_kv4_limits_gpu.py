"""The 4-bit paged cache at its limits: lengths that its tables do not hold, V and q of any size a
bf16 has, spreads next to fp32's largest, pools that run out."""
import pytest
import torch

import kv4_ref as ref
from oumu_b200 import ops
from oumu_b200.kv4 import KV4Cache
from test_kv4_gpu import LENGTH, attn_case, check_attn, i32, randn, run_attn

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


# ---- V of any size ----

def sized(kind, T, nk, hd, dev="cuda"):
    """T rows of k and v [T][2][nk][hd]."""
    kv = randn(95, T, 2 * nk * hd).float().view(T, 2, nk, hd)
    v = kv[:, 1]
    part, _, arg = kind.partition(":")
    x = float(arg) if arg else 0.0
    if part == "all":
        v *= x
    elif part == "group":            # one group of every position
        v[..., 32:64] *= x
    elif part == "constant":
        v[:] = x
    elif part == "constant_and":     # a constant group beside one of another size
        v[..., :32] = 1e20
        v[..., 32:64] *= x
    elif part == "late":             # a group that is 0 at first
        v[..., 32:64] *= x
        v[:T // 2, :, 32:64] = 0
    elif part == "growing":          # from 1e-20 to 1e10 along the positions
        v *= 10.0 ** torch.linspace(-20, 10, T, device=dev).view(T, 1, 1)
    elif part == "falling":
        v *= 10.0 ** torch.linspace(10, -20, T, device=dev).view(T, 1, 1)
    elif part == "some":             # one position in 50 is larger in one group
        v[::50, :, 32:64] *= x
    return kv.bfloat16().view(T, -1)


KINDS = ["all:1e-25", "all:1e-28", "all:1e-32", "all:1e-35", "all:1e30", "all:1e33", "all:3e37", "group:1e-9", "group:1e-12",
         "group:1e-25", "group:1e12", "group:1e25", "constant:1e20", "constant:-1e30", "constant:-3e38", "constant:1e-30",
         "constant_and:1e-9", "constant_and:1e9", "late:1e-15", "late:1e15", "growing", "falling", "some:1e6", "some:1e-12"]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_with_v_of_any_size(cuda, kind, hd):
    """The bound of check_attn, each channel's own: what one group holds costs another nothing."""
    nq, nk, lens = 8, 2, [500, 97]
    kv = torch.cat([sized(kind, 500, nk, hd), sized(kind, 500, nk, hd).flip(0)])
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=96, kv=kv)
    check_attn(run_attn(qkv, pool, table, ln, 2, nq, nk, hd), qkv, pool, rows, lens, nq, nk, hd)


@pytest.mark.parametrize("kind", ["group:1e-12", "all:1e-30", "all:3e37", "constant_and:1e-9", "constant:3e38", "growing",
                                  "falling"])
def test_split_attention_with_v_of_any_size(cuda, kind):
    nq, nk, hd, lens = 16, 2, 128, [20000]
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=97, kv=sized(kind, 20000, nk, hd))
    check_attn(run_attn(qkv, pool, table, ln, 1, nq, nk, hd), qkv, pool, rows, lens, nq, nk, hd)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [0, 1])
def test_nan_in_a_group_of_v_stays_in_it(cuda, hd, group):
    nq, nk, n = 4, 2, 300
    kv = randn(101, n, 2 * nk * hd).view(n, 2, nk, hd)
    bad = kv.clone()
    bad[[0, 5, 250], 1, 1, 32 * group + 7] = float("nan")
    good, out = [], []
    for x, to in ((kv, good), (bad, out)):
        qkv, pool, rows, table, ln = attn_case([n], nq, nk, hd, seed=102, kv=x.view(n, -1))
        to.append(run_attn(qkv, pool, table, ln, 1, nq, nk, hd).view(nq, hd).float())
    good, out = good[0], out[0]
    hit = torch.zeros(nq, hd, dtype=torch.bool, device="cuda")
    hit[2:, 32 * group:32 * group + 32] = True
    assert bool(torch.isnan(out[hit]).all()) and not bool(torch.isnan(out[~hit]).any())
    # the bound of check_attn, of both, with 15 s <= the spread (1 + 2^-7), which is at most twice the largest |V|
    big = float(kv[:, 1].abs().max())
    tol = 2 * (good.abs() * 2 ** -8 + 2 * big * (1 + 2 ** -7) * (2 ** -11 + 2 ** -14) + big * 2 ** -14)
    assert bool(((out - good).abs() <= tol)[~hit].all())


# ---- q of any size ----

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_size,k_size", [(1e30, 1e-30), (1e32, 1e-32), (1e34, 1e-34), (1e33, 1.0),
                                           (1e36, 1e-2), (1e5, 1.0), (1e8, 1.0), (1.0, 1e30), (1e-30, 1e30),
                                           (1e-36, 1e36), (1e-38, 1.0)])
def test_attention_with_q_of_any_size(cuda, q_size, k_size, hd):
    nq, nk, lens = 8, 2, [300, 33]
    kv = randn(98, 600, 2 * nk * hd).float().view(600, 2, nk, hd)
    kv[:, 0] *= k_size
    q = (randn(99, 2, nq * hd).float() * q_size).bfloat16()
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=98, kv=kv.bfloat16().view(600, -1), q=q)
    check_attn(run_attn(qkv, pool, table, ln, 2, nq, nk, hd), qkv, pool, rows, lens, nq, nk, hd)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_at_a_tiny_scale(cuda, hd):
    """A scale that leaves nothing of the logits: the average of V, for q of 0 too."""
    nq, nk, n = 4, 2, 45
    qkv, pool, rows, table, ln = attn_case([n], nq, nk, hd, seed=100)
    qkv[:, :hd] = 0
    out = torch.empty(1, nq * hd, dtype=torch.bfloat16, device="cuda")
    for scale in (1e-18, 1e-30, 1e-38):
        ops.attn_decode_kv4(qkv, pool, out, ops.decode_kv4_workspace(1, nq, nk, hd, 1), table, None, ln, 1, nq, nk, hd,
                            scale)
        k, v, vs = ref.take_values(pool.cpu(), rows[0], n, nk, hd)
        want = v.mean(1).repeat_interleave(2, 0)
        # the bound of check_attn
        tol = 15 * vs.amax(1) * (2 ** -11 + 2 ** -14) + v.abs().amax(1) * 2 ** -14
        tol = want.abs() * 2 ** -8 + tol.repeat_interleave(2, 0)
        assert bool(((out.cpu().double().view(nq, hd) - want).abs() <= tol).all())


# ---- spreads next to fp32's largest ----

def test_groups_whose_spread_fp32_just_holds(cuda):
    """max - min = 2^128 - 2^112: fp32 has it, so the group is held like any other."""
    nk, hd = 1, 64
    top, low = 2.0 ** 128 - 2.0 ** 120, -(2.0 ** 120 - 2.0 ** 112)
    x = torch.linspace(0, 1, 32, dtype=torch.float64) * 2.0 ** 127
    x[3], x[17] = top, low
    x = x.float().bfloat16().repeat(4)
    pool = torch.full((1, ref.page_bytes(nk, hd)), 255, dtype=torch.uint8, device="cuda")
    ops.kv4_write(x.cuda(), pool, i32([[0]]), None, None, 1, 1, 0, nk, hd)
    k, _, v, _ = ref.pool_values(pool.cpu(), nk, hd)
    want = ref.held(x.view(2, 64).double())[3]
    assert bool(torch.isfinite(want).all())
    assert torch.equal(k[0, 0, 0], want[0]) and torch.equal(v[0, 0, 0], want[1])


# ---- workspaces ----

@pytest.mark.parametrize("hd", [64, 128])
def test_one_workspace_for_batches_of_several_sizes(cuda, hd):
    """Records of a smaller batch do not lie where a larger one has its counters."""
    nq, nk = 8, 2
    most = 1200
    sizes = {2: [4000, 4007], most: [1 + s % 90 for s in range(most)], 40: [200 + 7 * s for s in range(40)]}
    ws = ops.decode_kv4_workspace(most, nq, nk, hd, 64)
    for B, lens in list(sizes.items()) * 2:
        qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=B)
        out = torch.full((B, nq * hd), float("nan"), dtype=torch.bfloat16, device="cuda")
        ops.attn_decode_kv4(qkv, pool, out, ws, table, None, ln, B, nq, nk, hd, hd ** -0.5)
        assert torch.equal(out, run_attn(qkv, pool, table, ln, B, nq, nk, hd))
        assert int(ws[:4 * most * nk].int().sum()) == 0


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


def test_lists_of_takes_do_not_wait_for_the_gpu(cuda):
    c = KV4Cache(1, 4, 8, 2, 64, 16, 256)
    c.lens[0] = 70
    c.extend()
    c.fork([0], [1])
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(400_000_000)  # some 0.2 s
    c.fork([0], [2])
    c.free([1])
    done.record()
    assert not done.query()
    torch.cuda.synchronize()
    assert c.lens.tolist() == [70, 0, 70, 0] and ops.device_error() == 0


def test_a_cache_gives_its_free_pages_back_and_grows(cuda):
    """Three of five takes are freed and the cache cut to what is left: its bytes shrink, the other takes' outputs stay; it
    grows again when a take needs more."""
    nq, nk, hd, layers, B = 8, 2, 64, 3, 5
    c = KV4Cache(layers, B, nq, nk, hd, 24, 512)
    c.lens.copy_(i32([300, 64, 130, 250, 190]))
    c.extend()
    for l in range(layers):
        c.write(l, randn(110 + l, B * 300, 2 * nk * hd), 300, nq=0, count=c.lens)
    qkv = randn(120, B, (nq + 2 * nk) * hd)

    def outputs():
        out = torch.empty(layers, B, nq * hd, dtype=torch.bfloat16, device="cuda")
        for l in range(layers):
            c.attend(l, qkv, out[l])
        return out[:, [2, 4]]

    c.free([0, 1, 3])
    want, before = outputs(), c.nbytes()  # (the split of the work, and with it last bits, go by every take's length)
    with pytest.raises(ValueError):
        c.resize(5)  # 3 pages of each take are in use
    assert torch.equal(outputs(), want)
    c.resize(6)
    assert c.npages == 6 and c.nbytes() * 4 == before and int((c.ref > 0).sum()) == 6
    assert torch.equal(outputs(), want)
    c.lens[2] = 193
    c.extend()
    assert c.missing() == 1
    c.resize(9)
    c.extend()
    assert c.missing() == 0 and c.table[2].max().item() == 6
    c.lens[2] = 130
    assert torch.equal(outputs(), want) and ops.device_error() == 0


def test_extend_and_fork_then_step_with_programmatic_launches(cuda):
    """No launch of the caller's between page calls and steps: the cache's own is one."""
    nq, nk, hd, layers, B = 16, 2, 128, 2, 6
    cs, sn = (t.cuda() for t in ops.rotary_tables(512, hd))
    qkv = randn(130, 12, B, (nq + 2 * nk) * hd)
    src, dst = i32([0, 0]), i32([4, 5])
    results = []
    for pdl in (False, True):
        c = KV4Cache(layers, B, nq, nk, hd, 60, 512)
        c.lens.copy_(i32([127, 64, 1, 300, 0, 0]))
        c.extend()
        for l in range(layers):
            c.write(l, randn(131 + l, B * 300, 2 * nk * hd), 300, nq=0, count=c.lens)
        out = torch.zeros(12, layers, B, nq * hd, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        prev = ops.set_pdl(pdl)
        try:
            for i in range(12):
                if i == 5:
                    c.fork(src, dst)
                c.lens.add_((c.lens > 0).int())
                c.extend()
                for l in range(layers):
                    c.step(l, qkv[i], out[i, l], cs, sn)
        finally:
            ops.set_pdl(prev)
        assert c.missing() == 0 and ops.device_error() == 0
        results.append((out, c.table.clone(), c.lens.tolist()))
    assert all(torch.equal(a, b) for a, b in zip(results[0][:2], results[1][:2])) and results[0][2] == results[1][2]
