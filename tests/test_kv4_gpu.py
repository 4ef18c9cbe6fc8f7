"""The 4-bit paged cache on the GPU against its 64-bit restatement (kv4_ref): writes and reads exactly, attention within
the roundings it makes, the fused step bit for bit against the launches it stands for, page tables against a model in
Python lists, and a run of all of them together as a decode makes it."""
import random

import pytest
import torch

import kv4_ref as ref
from oumu_b200 import ops

pytestmark = pytest.mark.gpu

TIMEOUT, LENGTH, PAGE_ERR = 1, 2, 4


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(seed, *shape):
    return torch.randn(shape, generator=gen(seed), device="cuda").bfloat16()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def poisoned(npages, nk, hd):
    """A pool whose every scale and zero is a NaN until it is written."""
    return torch.full((npages, ref.page_bytes(nk, hd)), 255, dtype=torch.uint8, device="cuda")


def tables(lens, maxpages, npages, seed):
    ids = random.Random(seed).sample(range(npages), sum(-(-n // 64) for n in lens))
    rows = []
    for n in lens:
        rows.append([ids.pop() for _ in range(-(-n // 64))])
        rows[-1] += [-1] * (maxpages - len(rows[-1]))
    return rows


def attn_case(lens, nq, nk, hd, seed=0, kv=None, q=None):
    """qkv, pool, table rows and lengths: K and V written by kv4_write, unused pages and positions left as NaN."""
    B, maxpages = len(lens), max(1, -(-max(lens) // 64))
    npages = sum(-(-n // 64) for n in lens) + 2
    rows = tables(lens, maxpages, npages, seed)
    pool = poisoned(npages, nk, hd)
    T = max(max(lens), 1)
    if kv is None:
        kv = randn(seed + 1, B * T, 2 * nk * hd)
    table, ln = i32(rows), i32(lens)
    ops.kv4_write(kv, pool, table, None, ln, B, T, 0, nk, hd)
    qkv = randn(seed + 2, B, (nq + 2 * nk) * hd)
    if q is not None:
        qkv[:, :nq * hd] = q
    return qkv, pool, rows, table, ln


def run_attn(qkv, pool, table, ln, B, nq, nk, hd, pos=None):
    out = torch.full((B, nq * hd), float("nan"), dtype=torch.bfloat16, device="cuda")
    ws = ops.decode_kv4_workspace(B, nq, nk, hd, table.shape[1])
    ops.attn_decode_kv4(qkv, pool, out, ws, table, pos, ln, B, nq, nk, hd, hd ** -0.5)
    assert int(ws[:4 * B * nk].int().abs().sum()) == 0  # counters left at zero
    return out


def check_attn(out, qkv, pool, rows, lens, nq, nk, hd):
    """Bound: the output's rounding to bf16 (2^-8 of the value); p s rounded to fp16 (2^-11 of it, times a code of at
    most 15 of either sign: 15 s 2^-11 of the weighted mean of s, so of the largest); p from fp32 logits, of which a
    relative 2^-14 is more than their sums of at most 2^12 terms of fp32 rounding allow (again on 15 s, and on |z|
    through the zeros' fp32 sums)."""
    pool, x = pool.cpu(), qkv.cpu().double()
    for s, n in enumerate(lens):
        got = out[s].cpu().double().view(nq, hd)
        if n == 0:
            assert bool((got == 0).all())
            continue
        k, v, vs = ref.take_values(pool, rows[s], n, nk, hd)
        want = ref.attend(x[s].view(-1, hd)[:nq], k, v, hd ** -0.5)
        top = vs.amax(1).repeat_interleave(nq // nk, 0)
        big = v.abs().amax(1).repeat_interleave(nq // nk, 0)
        tol = want.abs() * 2 ** -8 + 15 * top * (2 ** -11 + 2 ** -14) + big * 2 ** -14
        assert bool(((got - want).abs() <= tol).all()), (s, n, float(((got - want).abs() / tol).max()))


# ---- writes and reads ----

@pytest.mark.parametrize("nk,nq,hd,starts,counts", [
    (2, 16, 128, [0], [1]), (2, 16, 128, [63], [1]), (2, 16, 128, [5, 0, 64, 31], [70, 0, 3, 33]),
    (1, 7, 64, [1, 2, 7], [1, 2, 9]), (3, 0, 64, [0, 127], [200, 65]), (4, 4, 128, [8], [129]),
])
def test_write_then_read(cuda, nk, nq, hd, starts, counts):
    B, rows = len(starts), max(max(counts), 1) + 2  # padded: two rows behind the longest
    ends = [a + n for a, n in zip(starts, counts)]
    maxpages = -(-max(ends) // 64) + 1
    tab = tables([max(e, 1) for e in ends], maxpages, 4 * B * maxpages, 3)
    g = gen(17)
    pool = torch.randint(0, 128, (4 * B * maxpages, ref.page_bytes(nk, hd)), dtype=torch.uint8, generator=g,
                         device="cuda")  # finite scales everywhere
    before = [x.clone() for x in ref.pool_values(pool.cpu(), nk, hd)]
    qkv = randn(4, B * rows, (nq + 2 * nk) * hd)
    ops.kv4_write(qkv, pool, i32(tab), i32(starts), i32(counts), B, rows, nq, nk, hd)
    after = ref.pool_values(pool.cpu(), nk, hd)
    x = qkv.cpu().double().view(B, rows, nq + 2 * nk, hd)
    touched = torch.zeros(pool.shape[0], 64, dtype=torch.bool)
    maxlen = maxpages * 64 - 3
    kc = torch.full((B, nk, maxlen, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    ops.kv4_read(pool, i32(tab), i32(ends), kc, vc, nk, hd)
    kc, vc = kc.cpu(), vc.cpu()
    for s in range(B):
        for i in range(counts[s]):
            p = starts[s] + i
            page = tab[s][p // 64]
            touched[page, p % 64] = True
            for j, (vals, slot) in enumerate(((after[0], kc), (after[2], vc))):
                want = ref.held(x[s, i, nq + j * nk:nq + (j + 1) * nk])[3]
                assert torch.equal(vals[page, :, p % 64], want)
                assert torch.equal(slot[s, :, p], want.float().bfloat16())
        assert bool((kc[s, :, ends[s]:] == 7).all()) and bool((vc[s, :, ends[s]:] == 7).all())
    for b, a in zip(before, after):
        m = ~touched[:, None, :, None].expand_as(a)
        assert torch.equal(a[m], b[m])
    assert ops.device_error() == 0


def test_write_of_ties_constants_and_extremes(cuda):
    nk, hd = 1, 64
    ramp = torch.arange(32).double() / 2  # 0 .. 15.5: with 15 as its maximum every half is a tie at scale 1
    ramp[31] = 15
    tiny = torch.arange(32).double() * 2.0 ** -133  # bf16 subnormals
    far = torch.cat((torch.tensor([-15.0]), torch.full((30,), 2.0 ** -60), torch.tensor([15.0])))  # ties, but for 2^-60
    groups = [ramp, torch.full((32,), 3.25), tiny, ramp * 2.0 ** 100, -ramp,
              torch.randn(32, generator=torch.Generator().manual_seed(6)) * 1e-39, far, ramp * 2.0 ** -130]
    groups += [torch.where(torch.arange(32) == 9, torch.inf, ramp), torch.where(torch.arange(32) == 0, torch.nan, ramp)]
    x = torch.stack(groups).bfloat16()
    x = torch.stack((x, x.roll(1, 0)), 1).reshape(-1, hd)  # rows of two groups each
    qkv = torch.cat((x, x.flip(0)), 1).contiguous().cuda()  # k | v
    pool, n = poisoned(1, nk, hd), x.shape[0]
    ops.kv4_write(qkv, pool, i32([[0]]), None, None, 1, n, 0, nk, hd)
    k, _, v, _ = ref.pool_values(pool.cpu(), nk, hd)
    for got, want in ((k, x), (v, x.flip(0))):
        want = ref.held(want.double())[3]
        assert torch.equal(torch.isnan(got[0, 0, :n]), torch.isnan(want))
        assert torch.equal(got[0, 0, :n].nan_to_num(), want.nan_to_num())


def special_groups():
    """Groups in which the difference to the minimum is not exact in fp32, or a scale's reciprocal not a normal number:
    0 on a border with tiny values beside it, minima tiny beside the scale, subnormal and constant groups."""
    g = torch.Generator().manual_seed(11)
    out = []
    for m in range(15):  # -z = (m + 1/2) s: 0 lies on a border, s = 2
        v = torch.empty(32).uniform_(-2.0 * m - 1, 29.0 - 2 * m, generator=g).double()
        v[:8] = torch.tensor([2.0 ** -60, -(2.0 ** -60), 0.0, 2.0 ** -11, -(2.0 ** -11), 2.0 ** -13, -(2.0 ** -13), 1e-38])
        v[30], v[31] = -2.0 * m - 1, 29.0 - 2 * m
        out.append(v)
    for e in (-4, -11, -12, -13, -20, -40, -100):  # borders of s = 2 behind a minimum that hides in rounding
        out.append(torch.cat((torch.arange(1, 31, 2).double(), torch.arange(0, 32, 2).double(), -torch.tensor([2.0 ** e]))))
    ramp = torch.arange(32).double() / 2
    out += [ramp * 2.0 ** -e for e in (90, 100, 120, 127, 130, 133)] + [torch.zeros(32), torch.full((32,), -1e-30)]
    return torch.stack(out).bfloat16()


@pytest.mark.parametrize("hd", [64, 128])
def test_write_and_step_of_special_groups(cuda, hd):
    W = hd // 32
    x = special_groups()
    x = torch.cat((x, x.flip(1), -x))
    rows = torch.stack([x.roll(-3 * i, 0) for i in range(2 * W)], 1).reshape(x.shape[0], 2 * hd)  # k | v, one kv head
    n = rows.shape[0]
    pool = poisoned(-(-n // 64), 1, hd)
    ops.kv4_write(rows.cuda().contiguous(), pool, i32([list(range(pool.shape[0]))]), None, None, 1, n, 0, 1, hd)
    k, _, v, _ = ref.pool_values(pool.cpu(), 1, hd)
    want = ref.held(rows.double())[3]
    assert torch.equal(k.reshape(-1, hd)[:n], want[:, :hd]) and torch.equal(v.reshape(-1, hd)[:n], want[:, hd:])
    # the same rows as the first positions of n takes, by the fused step
    pool1, pool2 = poisoned(n, 1, hd), poisoned(n, 1, hd)
    table, ones = i32([[i] for i in range(n)]), i32([1] * n)
    qkv = torch.cat((randn(9, n, hd).cpu(), rows), 1).cuda().contiguous()
    out, ws = torch.empty(n, hd, dtype=torch.bfloat16, device="cuda"), ops.decode_kv4_workspace(n, 1, 1, hd, 1)
    held = torch.empty(n, 2 * hd, dtype=torch.bfloat16, device="cuda")
    ops.attn_decode_kv4_step(qkv, pool1, out, ws, None, None, table, None, ones, n, 1, 1, hd, 0.1, held=held)
    ops.kv4_write(qkv, pool2, table, None, None, n, 1, 1, 1, hd)
    assert torch.equal(pool1, pool2)
    assert torch.equal(held.cpu(), want.float().bfloat16())


# ---- attention ----

@pytest.mark.parametrize("nq,nk,hd", [(16, 2, 128), (8, 2, 64), (4, 4, 128), (7, 1, 64), (10, 2, 128), (3, 1, 128)])
@pytest.mark.parametrize("lens", [[1], [2, 31, 32, 33], [63, 64, 65, 0, 127, 129], [0, 0, 5], [700, 3, 1025]])
def test_attention(cuda, nq, nk, hd, lens):
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=len(lens))
    out = run_attn(qkv, pool, table, ln, len(lens), nq, nk, hd)
    check_attn(out, qkv, pool, rows, lens, nq, nk, hd)
    assert torch.equal(out, run_attn(qkv, pool, table, ln, len(lens), nq, nk, hd))
    assert ops.device_error() == 0


def test_attention_all_takes_empty(cuda):
    qkv, pool, rows, table, ln = attn_case([3, 4], 16, 2, 128)
    assert bool((run_attn(qkv, pool, table, i32([0, 0]), 2, 16, 2, 128) == 0).all())


def test_attention_at_a_shared_position(cuda):
    lens = [130, 130, 130]
    qkv, pool, rows, table, ln = attn_case(lens, 16, 2, 128, seed=8)
    a = run_attn(qkv, pool, table, ln, 3, 16, 2, 128)
    b = run_attn(qkv, pool, table, None, 3, 16, 2, 128, pos=i32([129, 5]))
    assert torch.equal(a, b)


@pytest.mark.parametrize("B,L,nq,nk,hd", [(1, 30000, 16, 2, 128), (2, 9001, 8, 1, 64), (40, 333, 16, 2, 128),
                                          (600, 40, 4, 4, 64), (1500, 9, 2, 1, 128), (70, 1300, 16, 4, 64)])
def test_attention_split_over_the_gpu(cuda, B, L, nq, nk, hd):
    r = random.Random(B)
    lens = [max(0, L - r.randint(0, L // 3)) for _ in range(B)]
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=B)
    out = run_attn(qkv, pool, table, ln, B, nq, nk, hd)
    some = sorted(r.sample(range(B), min(B, 12)))
    check_attn(out[some], qkv[some], pool, [rows[i] for i in some], [lens[i] for i in some], nq, nk, hd)
    assert torch.equal(out, run_attn(qkv, pool, table, ln, B, nq, nk, hd))


@pytest.mark.parametrize("kind", ["peaked", "large_v", "tiny_v", "one_large_v", "constant_v", "zero_k", "tiny_q",
                                  "rising"])
def test_attention_over_wide_ranges(cuda, kind):
    nq, nk, hd, lens = 16, 2, 128, [500, 97]
    T = 500
    kv = randn(31, 2 * T, 2 * nk * hd).float().view(2 * T, 2, nk, hd)
    q = randn(32, 2, nq * hd).float()
    if kind == "peaked":
        q *= 30
    elif kind == "large_v":
        kv[:, 1] *= 1e25
    elif kind == "tiny_v":
        kv[:, 1] *= 1e-12
    elif kind == "one_large_v":
        kv[77, 1] *= 1e6
    elif kind == "constant_v":
        kv[:, 1] = 2.5
        kv[400:440, 1] = 100.0
    elif kind == "zero_k":
        kv[:, 0] = 0
    elif kind == "tiny_q":
        q *= 1e-30
    elif kind == "rising":  # every later position beats the ones before: the reference exponent moves all along
        kv[:, 0] = torch.arange(2 * T, device="cuda").view(-1, 1, 1) % T * 0.05
        q = q.abs()
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, kv=kv.bfloat16().view(2 * T, -1), q=q.bfloat16())
    out = run_attn(qkv, pool, table, ln, 2, nq, nk, hd)
    check_attn(out, qkv, pool, rows, lens, nq, nk, hd)


def test_nan_in_a_take_stays_in_it(cuda):
    nq, nk, hd, lens = 16, 2, 128, [100, 100, 100]
    kv = randn(41, 300, 2 * nk * hd)
    kv[150, 3] = float("nan")  # k of take 1, kv head 0
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, kv=kv)
    out = run_attn(qkv, pool, table, ln, 3, nq, nk, hd).view(3, nk, -1)
    assert bool(torch.isnan(out[1, 0]).all()) and not bool(torch.isnan(out[[0, 2]]).any())
    assert not bool(torch.isnan(out[1, 1]).any())


def test_bad_pages_and_lengths_are_reported(cuda):
    nq, nk, hd, lens = 16, 2, 128, [200, 100, 70]
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=5)
    want = run_attn(qkv, pool, table, ln, 3, nq, nk, hd)
    ops.device_error(reset=True)
    for entry in (-1, pool.shape[0], 1 << 30):
        bad = table.clone()
        bad[1, 1] = entry
        out = run_attn(qkv, pool, bad, ln, 3, nq, nk, hd)
        assert ops.device_error(reset=True) == PAGE_ERR
        assert torch.equal(out[[0, 2]], want[[0, 2]])
        ops.kv4_write(randn(1, 3, 4 * 128), pool, bad, i32([300, 64, 300]), i32([0, 1, 0]), 3, 1, 0, nk, hd)
        assert ops.device_error(reset=True) == PAGE_ERR
    for n in (-5, table.shape[1] * 64 + 1):
        run_attn(qkv, pool, table, i32([lens[0], n, lens[2]]), 3, nq, nk, hd)
        assert ops.device_error(reset=True) & LENGTH
    assert torch.equal(run_attn(qkv, pool, table, ln, 3, nq, nk, hd), want)
    assert ops.device_error() == 0


# ---- the fused step ----

@pytest.mark.parametrize("nq,nk,hd", [(16, 2, 128), (8, 2, 64), (5, 1, 128), (4, 4, 64)])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("lens", [[1], [64, 65, 1, 33, 0, 96], [1000, 2, 513], [300] * 90])
def test_step_is_rope_write_attend(cuda, nq, nk, hd, rope, lens):
    B = len(lens)
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=B + nq)
    cs, sn = (t.cuda() for t in ops.rotary_tables(max(lens), hd))
    if not rope:
        cs = sn = None
    pool2, q2, kept = pool.clone(), qkv.clone(), qkv.clone()
    ws = ops.decode_kv4_workspace(B, nq, nk, hd, table.shape[1])
    out, held = randn(1, B, nq * hd), randn(2, B, 2 * nk * hd)
    ops.attn_decode_kv4_step(qkv, pool, out, ws, cs, sn, table, None, ln, B, nq, nk, hd, hd ** -0.5, held=held)
    assert torch.equal(qkv, kept)
    if rope:
        for s, n in enumerate(lens):
            if n:
                ops.rope(q2[s:s + 1], cs, sn, i32([n - 1]), 1, 0, nq, nk, hd)
    ops.kv4_write(q2, pool2, table, (ln - 1).clamp(min=0), (ln > 0).int(), B, 1, nq, nk, hd)
    assert torch.equal(pool, pool2)
    assert torch.equal(out, run_attn(q2, pool2, table, ln, B, nq, nk, hd))
    x = q2.cpu().double().view(B, -1, hd)[:, nq:]
    want = ref.held(x)[3].float().bfloat16() * (ln.cpu() > 0).view(B, 1, 1)
    assert torch.equal(held.cpu().view(B, -1, hd), want)
    check_attn(out, q2, pool, rows, lens, nq, nk, hd)
    again = torch.empty_like(out)
    ops.attn_decode_kv4_step(qkv, pool, again, ws, cs, sn, table, None, ln, B, nq, nk, hd, hd ** -0.5)
    assert torch.equal(again, out)
    assert ops.device_error() == 0


# ---- pages ----

class Model:
    def __init__(self, B, npages, maxpages, layers=2, size=48, seed=0):
        self.m = ref.Pages(B, npages, maxpages)
        self.table = torch.full((B, maxpages), -1, dtype=torch.int32, device="cuda")
        self.ref = torch.zeros(npages, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(2, dtype=torch.int32, device="cuda")
        self.pools = torch.randint(0, 256, (layers, npages, size), dtype=torch.uint8, generator=gen(seed), device="cuda")
        self.bytes = self.pools.cpu()
        self.ws = ops.pages_workspace(npages)

    def check(self):
        for a, b in self.m.moved:
            self.bytes[:, b] = self.bytes[:, a]
        self.m.moved = []
        assert self.table.tolist() == self.m.table
        assert self.ref.tolist() == self.m.ref
        assert self.lens.tolist() == self.m.lens
        assert torch.equal(self.pools.cpu(), self.bytes)

    def set_len(self, s, n):
        self.m.lens[s] = n
        self.lens[s] = n

    def extend(self, extra):
        ops.pages_extend(self.table, self.ref, self.lens, extra, self.status)
        assert int(self.status[0]) == self.m.extend(extra)
        self.check()

    def fork(self, src, dst):
        ops.pages_fork(self.pools, self.table, self.ref, self.lens, i32(src), i32(dst), self.status)
        missing, ok = self.m.fork(src, dst)
        assert int(self.status[0]) == missing
        assert ops.device_error(reset=True) == (0 if ok else PAGE_ERR)
        self.check()

    def free(self, takes):
        ops.pages_free(self.table, self.ref, self.lens, i32(takes))
        for s in takes:
            self.m.release(s)
        self.check()

    def compact(self):
        ops.pages_compact(self.pools, self.table, self.ref, self.ws, self.status)
        assert tuple(self.status.tolist()) == self.m.compact()
        self.check()


@pytest.mark.parametrize("seed", range(6))
def test_pages_like_their_model(cuda, seed):
    r = random.Random(seed)
    B, maxpages = r.randint(2, 12), r.randint(1, 40)
    p = Model(B, r.randint(3, 60), maxpages, layers=r.randint(1, 3), size=16 * r.randint(1, 90), seed=seed)
    for _ in range(40):
        do = r.choice(["extend", "extend", "fork", "free", "compact"])
        if do == "extend":
            s = r.randrange(B)
            if all(x >= 0 for x in p.m.table[s][:-(-p.m.lens[s] // 64)]):
                p.set_len(s, r.randint(p.m.lens[s], min(64 * maxpages, p.m.lens[s] + 200)))
            p.extend(0)
            for s in range(B):  # what no page was left for ends where its pages end
                have = sum(x >= 0 for x in p.m.table[s])
                if p.m.lens[s] > 64 * have:
                    p.set_len(s, 64 * have)
        elif do == "fork":
            n = r.randint(0, B - 1)
            dst = r.sample(range(B), n)
            rest = [s for s in range(B) if s not in dst]
            p.fork([r.choice(rest) for _ in dst], dst)
        elif do == "free":
            p.free([r.randrange(B) for _ in range(r.randint(0, B))])
        else:
            p.compact()


def test_fork_refuses_takes_that_cannot_be(cuda):
    p = Model(6, 40, 8)
    for s, n in enumerate([100, 64, 0, 200, 1, 130]):
        p.set_len(s, n)
    p.extend(0)
    p.fork([0, 0, 0, 1, 9, 0, 3, 5], [2, 2, 0, 6, 4, -1, 3, 1])  # twice, itself, out of range; 1 -> 6 and 5 -> 1
    p.fork([0, 1], [1, 4])                                        # reads what the same call fills
    p.fork([], [])


def test_fork_and_extend_when_pages_run_out(cuda):
    p = Model(8, 9, 6)
    p.set_len(0, 64 * 3 + 5)
    p.extend(0)          # 4 pages
    p.fork([0] * 7, list(range(1, 8)))  # 5 copies fit, two takes end up empty
    assert p.m.lens.count(0) == 2
    p.extend(64)
    p.free([1, 1, 2])
    p.extend(64)
    p.compact()


def test_many_pages(cuda):
    p = Model(3, 30000, 12000, layers=1, size=16)
    p.set_len(0, 64 * 9000)
    p.set_len(1, 64 * 11000 - 7)
    p.extend(0)
    p.fork([1], [2])
    p.free([0])
    p.compact()


# ---- together, as a decode uses them ----

def test_a_decode_from_a_shared_prompt(cuda):
    """A prompt stored once, forked to the takes, then steps that append across page ends (captured and replayed),
    a take that ends, a new one from the prompt, a compaction in between: every step's output against the 64-bit
    attention over what the takes wrote."""
    nq, nk, hd, B, layers, T, maxpages, npages = 16, 2, 128, 5, 2, 125, 4, 24
    cs, sn = (t.cuda() for t in ops.rotary_tables(64 * maxpages, hd))
    pools = torch.full((layers, npages, ops.kv4_page_bytes(nk, hd)), 255, dtype=torch.uint8, device="cuda")
    table, rf = torch.full((B, maxpages), -1, dtype=torch.int32, device="cuda"), i32([0] * npages)
    lens, status = i32([T, 0, 0, 0, 0]), i32([0, 0])
    prompt = randn(3, layers, T, (nq + 2 * nk) * hd)
    ops.pages_extend(table, rf, lens, 0, status)
    for l in range(layers):
        ops.kv4_write(prompt[l], pools[l], table, None, lens[:1], 1, T, nq, nk, hd)
    ops.pages_fork(pools, table, rf, lens, i32([0] * 4), i32([1, 2, 3, 4]), status)
    qkv = randn(4, layers, B, (nq + 2 * nk) * hd)
    out = torch.zeros(layers, B, nq * hd, dtype=torch.bfloat16, device="cuda")
    ws, pws = ops.decode_kv4_workspace(B, nq, nk, hd, maxpages), ops.pages_workspace(npages)

    def step():
        lens.add_((lens > 0).int())
        ops.pages_extend(table, rf, lens, 0, status)
        for l in range(layers):
            ops.attn_decode_kv4_step(qkv[l], pools[l], out[l], ws, cs, sn, table, None, lens, B, nq, nk, hd, hd ** -0.5)

    def rotated(x, p):
        y = x.view(1, -1).clone()
        ops.rope(y, cs, sn, i32([p]), 1, 0, nq, nk, hd)
        return y[0].cpu().double().view(-1, hd)

    hist = [[[ref.held(prompt[l].cpu().double().view(T, -1, hd)[:, nq + j * nk:nq + (j + 1) * nk])[3]
              for j in range(2)] for l in range(layers)]] * B
    hist = [[[x.clone() for x in l] for l in t] for t in hist]
    live = [True] * B
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(9):
        qkv.copy_(randn(50 + i, layers, B, (nq + 2 * nk) * hd))
        if i == 4:
            ops.pages_free(table, rf, lens, i32([2, 3]))
            ops.pages_compact(pools, table, rf, pws, status)
            live[2] = live[3] = False
        if i == 6:
            ops.pages_fork(pools, table, rf, lens, i32([1]), i32([3]), status)
            live[3], hist[3] = True, [[x.clone() for x in l] for l in hist[1]]
        graph.replay() if i % 2 else step()
        n = lens.tolist()
        for s in range(B):
            for l in range(layers):
                got = out[l, s].cpu().double().view(nq, hd)
                if not live[s]:
                    assert n[s] == 0 and bool((got == 0).all())
                    continue
                x = rotated(qkv[l, s], n[s] - 1)
                for j in range(2):
                    hist[s][l][j] = torch.cat((hist[s][l][j], ref.held(x[nq + j * nk:nq + (j + 1) * nk])[3][None]))
                k, v = (h.transpose(0, 1) for h in hist[s][l])
                want = ref.attend(x[:nq], k, v, hd ** -0.5)
                # the bound of check_attn with V's largest scale from its spread: s <= (max - min) / 15 (1 + 2^-7)
                spread = (v.amax((1, 2)) - v.amin((1, 2))).repeat_interleave(nq // nk)[:, None]
                tol = want.abs() * 2 ** -8 + spread * (1 + 2 ** -7) * (2 ** -11 + 2 ** -14) + v.abs().max() * 2 ** -14
                assert n[s] == k.shape[1] and bool(((got - want).abs() <= tol).all())
    assert int(status[0]) == 0 and ops.device_error() == 0
    used = {p for row in table.tolist() for p in row if p >= 0}
    assert [int(r > 0) for r in rf.tolist()] == [int(p in used) for p in range(npages)]


def test_two_streams_with_their_own_workspaces(cuda):
    nq, nk, hd = 16, 2, 128
    cases = [attn_case([400 + 7 * i, 90, 1200], nq, nk, hd, seed=60 + i) for i in range(2)]
    want = [run_attn(c[0], c[1], c[3], c[4], 3, nq, nk, hd) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [torch.zeros_like(w) for w in want]
    wss = [ops.decode_kv4_workspace(3, nq, nk, hd, c[3].shape[1]) for c in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, o, w in zip(cases, streams, outs, wss):
            with torch.cuda.stream(s):
                ops.attn_decode_kv4(c[0], c[1], o, w, c[3], None, c[4], 3, nq, nk, hd, hd ** -0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("maxpages", [1, 4])  # 8 warps, and 12
def test_the_most_takes(cuda, hd, maxpages):
    B, nq, nk = 4096, 2, 1
    r = random.Random(maxpages)
    lens = [r.choice((0, 1, 7, 33, 64 * maxpages)) for _ in range(B)]
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=maxpages)
    out = run_attn(qkv, pool, table, ln, B, nq, nk, hd)
    some = sorted(r.sample(range(B), 40)) + [B - 1]
    check_attn(out[some], qkv[some], pool, [rows[i] for i in some], [lens[i] for i in some], nq, nk, hd)
    with pytest.raises(ValueError):
        ops.decode_kv4_workspace(B + 1, nq, nk, hd, maxpages)


def test_rows_may_be_bf16_bits_but_no_other_16_bit_type(cuda):
    qkv, pool, rows, table, ln = attn_case([70], 16, 2, 128)
    out, ws = torch.empty(1, 2048, dtype=torch.bfloat16, device="cuda"), ops.decode_kv4_workspace(1, 16, 2, 128, 2)
    bits = torch.zeros_like(out, dtype=torch.int16)
    ops.attn_decode_kv4(qkv, pool, out, ws, table, None, ln, 1, 16, 2, 128, 0.1)
    ops.attn_decode_kv4(qkv.view(torch.int16), pool, bits, ws, table, None, ln, 1, 16, 2, 128, 0.1)
    assert torch.equal(out.view(torch.int16), bits)
    with pytest.raises(ValueError):
        ops.attn_decode_kv4(qkv.view(torch.float16), pool, out, ws, table, None, ln, 1, 16, 2, 128, 0.1)
    with pytest.raises(ValueError):
        ops.attn_decode_kv4(qkv, pool, out.view(torch.float16), ws, table, None, ln, 1, 16, 2, 128, 0.1)
    with pytest.raises(ValueError):
        ops.kv4_write(qkv.view(torch.float16), pool, table, None, None, 1, 1, 16, 2, 128)


def test_tensors_the_entry_points_cannot_take_are_refused(cuda):
    nq, nk, hd = 16, 2, 128
    qkv, pool, rows, table, ln = attn_case([70], nq, nk, hd)
    out, ws = torch.empty(1, nq * hd, dtype=torch.bfloat16, device="cuda"), ops.decode_kv4_workspace(1, nq, nk, hd, 2)
    call = lambda **k: ops.attn_decode_kv4(*({**dict(qkv=qkv, pool=pool, out=out, ws=ws, table=table, pos=None,  # noqa
                                                     lens=ln, B=1, nq=nq, nk=nk, hd=hd, scale=0.1), **k}.values()))
    call()
    for k in (dict(table=table.long()), dict(lens=ln.long()), dict(pool=pool[:, :-16]), dict(pool=pool.view(torch.int8)),
              dict(nk=1), dict(hd=64), dict(B=2), dict(qkv=qkv.float()), dict(out=out[:, ::2]), dict(table=table.cpu()),
              dict(lens=ln.cpu()), dict(qkv=qkv.cpu()), dict(out=out.cpu()), dict(ws=ws.cpu()), dict(ws=ws.float()),
              dict(lens=ln[:0])):
        with pytest.raises(ValueError):
            call(**k)


def test_a_small_workspace_runs_on_fewer_ctas(cuda):
    nq, nk, hd, lens = 16, 2, 128, [900, 2500, 0, 77]
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=70)
    record = 2 * (16 + 8 * hd) * 4
    for ctas in (1, 3):
        ws = torch.zeros(256 + ctas * record, dtype=torch.uint8, device="cuda")
        out = torch.empty(4, nq * hd, dtype=torch.bfloat16, device="cuda")
        for _ in range(2):
            ops.attn_decode_kv4(qkv, pool, out, ws, table, None, ln, 4, nq, nk, hd, hd ** -0.5)
            check_attn(out, qkv, pool, rows, lens, nq, nk, hd)
    with pytest.raises(RuntimeError):
        ops.attn_decode_kv4(qkv, pool, out, ws[:256 + record - 16], table, None, ln, 4, nq, nk, hd, hd ** -0.5)


def test_step_past_the_rotary_tables_is_reported(cuda):
    nq, nk, hd, lens = 16, 2, 128, [100, 40]
    qkv, pool, rows, table, ln = attn_case(lens, nq, nk, hd, seed=71)
    cs, sn = (t.cuda() for t in ops.rotary_tables(64, hd))
    ws = ops.decode_kv4_workspace(2, nq, nk, hd, table.shape[1])
    out = [torch.empty(2, nq * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.attn_decode_kv4_step(qkv, pool, out[0], ws, cs, sn, table, None, ln, 2, nq, nk, hd, hd ** -0.5)
    assert ops.device_error(reset=True) == LENGTH
    ops.attn_decode_kv4_step(qkv, pool, out[1], ws, cs, sn, table, None, i32([64, 40]), 2, nq, nk, hd, hd ** -0.5)
    assert ops.device_error() == 0 and torch.equal(out[0], out[1])  # cut to what the tables hold


def test_page_calls_captured_and_replayed(cuda):
    """Free, fork, extend and compact in one graph, replayed as the takes grow, against the model."""
    p = Model(5, 40, 6)
    p.set_len(0, 150)
    p.extend(0)
    src, dst, gone = i32([0, 0]), i32([1, 3]), i32([3, 2, 3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.pages_free(p.table, p.ref, p.lens, gone)
        ops.pages_fork(p.pools, p.table, p.ref, p.lens, src, dst, p.status)
        ops.pages_extend(p.table, p.ref, p.lens, 70, p.status)
        ops.pages_compact(p.pools, p.table, p.ref, p.ws, p.status)
    for grow in (0, 13, 64, 30):
        if grow:
            p.set_len(0, p.m.lens[0] + grow)
            p.extend(0)
        graph.replay()
        for s in (3, 2, 3):
            p.m.release(s)
        p.m.fork([0, 0], [1, 3])
        p.m.extend(70)
        p.m.compact()
        p.check()


def test_step_with_programmatic_launches(cuda):
    """A chain of steps and their page calls with programmatic dependent launches on gives what it gives without."""
    nq, nk, hd, B, layers = 16, 2, 128, 6, 4
    cs, sn = (t.cuda() for t in ops.rotary_tables(512, hd))
    lens0 = [64, 1, 200, 127, 0, 333]
    results = []
    for pdl in (False, True):
        pools = torch.zeros(layers, 40, ops.kv4_page_bytes(nk, hd), dtype=torch.uint8, device="cuda")
        table, rf = torch.full((B, 8), -1, dtype=torch.int32, device="cuda"), i32([0] * 40)
        lens, status = i32(lens0), i32([0, 0])
        ws = ops.decode_kv4_workspace(B, nq, nk, hd, 8)
        ops.pages_extend(table, rf, lens, 0, status)
        kv = randn(80, layers, B * 333, 2 * nk * hd)
        for l in range(layers):
            ops.kv4_write(kv[l], pools[l], table, None, lens, B, 333, 0, nk, hd)
        qkv = randn(81, B, (nq + 2 * nk) * hd)
        outs = []
        prev = ops.set_pdl(pdl)
        try:
            for _ in range(5):
                lens.add_((lens > 0).int())
                ops.pages_extend(table, rf, lens, 0, status)
                x = qkv.clone()
                for l in range(layers):
                    out = torch.empty(B, nq * hd, dtype=torch.bfloat16, device="cuda")
                    ops.attn_decode_kv4_step(x, pools[l], out, ws, cs, sn, table, None, lens, B, nq, nk, hd, hd ** -0.5)
                    x = torch.cat((out, x[:, nq * hd:]), 1)  # the next layer's q is this one's output
                    outs.append(out)
        finally:
            ops.set_pdl(prev)
        results.append((torch.stack(outs), pools.clone()))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert ops.device_error() == 0
