"""The operators of the 4-bit paged KV cache, as they are measured: their cases, their plain forms and their calls.

The cache. A page holds 64 positions of every kv head, K and V; takes name their pages in a table [B][maxpages] that
every layer shares. A value is held in 4 bits, in groups of 32 channels of one position: z = the group's minimum
(bf16), s = the smallest bf16 >= (max - min) / 15, n = (x - z) / s rounded to the nearest whole number (half to even),
and it stands for s * n + z. A page's bytes are [nk][2 halves of 32 positions][K codes, V codes, K scales and
zeros, V scales and zeros]; `_pack` below gives the order of the codes.

`run` computes an operator either in elementary torch operations (own = False) or through the package's entry
points (own = True), on the same state."""
import torch

own = False

PAGE = 64
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one take of one text early in its decode: the smallest call, where latency counts
        dict(name="attn-1x512", op="attn", B=1, lo=512, hi=512, empty=0, nq=16, nk=2, hd=128),
        # a batch of takes at their own lengths, the decode benchmark's shape
        dict(name="attn-64x4096", op="attn", B=64, lo=330, hi=4096, empty=0, nq=16, nk=2, hd=128),
        # two takes near the longest slot the engine allows: work split over a long axis
        dict(name="attn-2x65536", op="attn", B=2, lo=65531, hi=65536, empty=0, nq=16, nk=2, hd=128),
        # an odd batch of short takes with 64-wide heads, some takes already freed (length 0)
        dict(name="attn-19x1500-hd64", op="attn", B=19, lo=1, hi=1500, empty=3, nq=8, nk=2, hd=64),
        # one decode layer of the whole engine: rope, quantise, append, attend for 32 takes
        dict(name="step-32x4096", op="step", B=32, lo=330, hi=4096, empty=0, nq=16, nk=2, hd=128, rope=True),
        # the largest batch: 256 takes on one GPU, a layer without rope (the residual model's)
        dict(name="step-256x4096", op="step", B=256, lo=330, hi=4096, empty=0, nq=16, nk=2, hd=128, rope=False),
        # a prompt stored once and read back as bf16 rows
        dict(name="store-1x1024", op="store", B=1, rows=1024, lo=1024, hi=1024, start=0, nq=16, nk=2, hd=128),
        # a padded batch of ragged prompts that continue takes at odd positions
        dict(name="store-48x4096", op="store", B=48, rows=4096, lo=301, hi=4096, start=77, nq=16, nk=2, hd=128),
        # a short prompt shared by a few takes, the residual model's layers
        dict(name="fork-4x330", op="fork", B=4, prompt=330, layers=8, nk=2, hd=128),
        # a text's prompt shared by 64 takes over every layer of the engine
        dict(name="fork-64x1000", op="fork", B=64, prompt=1000, layers=36, nk=2, hd=128),
        # a small pool after some takes have ended
        dict(name="compact-200x8", op="compact", npages=200, live=110, B=8, layers=8, nk=2, hd=128),
        # the engine's pool, fragmented, packed together so that its end can be given back
        dict(name="compact-1000x36", op="compact", npages=1000, live=550, B=32, layers=36, nk=2, hd=128),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attn", "attn", "step", "step", "store", "fork", "compact"])
    nq, nk, hd = rng.choice([(16, 2, 128), (16, 2, 128), (8, 2, 64), (12, 2, 128), (4, 4, 128), (7, 1, 64)])
    if op in ("attn", "step"):
        B = _log(rng, 1, 200)
        hi = _log(rng, 3, min(65536, 500000 * 256 // (B * nk * hd)))
        c = dict(op=op, B=B, lo=max(1, int(hi * rng.random())), hi=hi, empty=rng.choice([0, 0, B // 5]), nq=nq, nk=nk,
                 hd=hd)
        if op == "step":
            c["rope"] = rng.random() < 0.7
        return c
    if op == "store":
        B = _log(rng, 1, 40)
        rows = _log(rng, 2, min(16384, 90000 * 256 // (B * nk * hd)))
        return dict(op=op, B=B, rows=rows, lo=rng.randint(0, rows), hi=rows, start=rng.choice([0, rng.randint(1, 200)]),
                    nq=nq, nk=nk, hd=hd)
    if op == "fork":
        return dict(op=op, B=_log(rng, 2, 64), prompt=_log(rng, 1, 4000), layers=rng.randint(1, 36), nk=nk,
                    hd=hd)
    npages = _log(rng, 20, 900)
    return dict(op=op, npages=npages, live=max(1, int(npages * rng.uniform(0.2, 0.9))), B=rng.randint(1, 40),
                layers=rng.randint(1, min(36, 36 * 256 // (nk * hd))), nk=nk, hd=hd)


def work(c):
    W = c["hd"] // 32
    row = 2 * (c["hd"] // 2 + 4 * W)  # bytes of K and V of one position and kv head
    if c["op"] in ("attn", "step"):
        pos = sum(_lens(c))
        io = c["B"] * c["hd"] * 4 * c["nq"]
        if c["op"] == "step":  # k and v in, what the cache holds of them out and into the page
            io += c["B"] * c["nk"] * (8 * c["hd"] + row)
        return dict(bytes=pos * c["nk"] * row + io, flops=4 * pos * c["nq"] * c["hd"])
    if c["op"] == "store":
        pos, held = sum(_counts(c)), sum(_counts(c)) + c["B"] * c["start"]
        return dict(bytes=pos * c["nk"] * (4 * c["hd"] + row) + held * c["nk"] * (4 * c["hd"] + row), flops=0)
    page = c["layers"] * PAGE * c["nk"] * row
    if c["op"] == "fork":
        part = 1 if c["prompt"] % PAGE else 0
        ints = 4 * c["B"] * (2 * -(-c["prompt"] // PAGE) + 6)
        return dict(bytes=part * c["B"] * page + ints, flops=0)
    # pages at or past `live` move once: read and written
    ids = _live_ids(c)
    return dict(bytes=2 * page * sum(i >= c["live"] for i in ids) + 16 * c["npages"], flops=0)


# lengths and live pages are part of the case, the same for every seed: the work of a pass goes by them

def _mix(i, salt):
    x = (i * 0x9E3779B1 + salt * 0x85EBCA77 + 0x165667B1) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x2C1B3C6D) & 0xFFFFFFFF
    x = ((x ^ (x >> 12)) * 0x297A2D39) & 0xFFFFFFFF
    return x ^ (x >> 15)


def _lens(c):
    n = [c["lo"] + _mix(i, 1) % (c["hi"] - c["lo"] + 1) for i in range(c["B"])]
    for k in range(c["empty"]):
        n[(3 + 5 * k) % c["B"]] = 0
    return n


def _counts(c):
    return [c["lo"] + _mix(i, 2) % (c["hi"] - c["lo"] + 1) for i in range(c["B"])]


def _live_ids(c):
    return sorted(sorted(range(c["npages"]), key=lambda i: _mix(i, 3))[:c["live"]])


# ------------------------------------------------------------------------------------------------ inputs

def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pages(n):
    return -(-n // PAGE)


def _table(lens, maxpages, g, spare):
    """Every take's pages, scattered over the pool as after some time of serving."""
    total = sum(_pages(n) for n in lens)
    ids = torch.randperm(total + spare, generator=g, device=DEV)[:total].to(torch.int32)
    table, at = torch.full((len(lens), maxpages), -1, dtype=torch.int32, device=DEV), 0
    for s, n in enumerate(lens):
        table[s, :_pages(n)] = ids[at:at + _pages(n)]
        at += _pages(n)
    return table, total + spare


def _pool(npages, nk, hd, g):
    """Pages as the path fills them: K with channels of different size, a few of them large; V without."""
    ch = torch.exp(0.4 * torch.randn(nk, 1, hd, generator=g, device=DEV))
    ch[:, :, torch.randint(0, hd, (3,), generator=g, device=DEV)] *= 4
    parts = []
    for a in range(0, npages, 512):
        n = min(512, npages - a)
        k = torch.randn(n, nk, PAGE, hd, generator=g, device=DEV) * ch
        v = torch.randn(n, nk, PAGE, hd, generator=g, device=DEV)
        parts.append(_pack(*_quantise(k.bfloat16().float()), *_quantise(v.bfloat16().float())))
    return torch.cat(parts)


def _rotary(maxlen, hd):
    f = torch.arange(maxlen, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, hd, 2).double() / hd)
    return f.cos().bfloat16().float().to(DEV), f.sin().bfloat16().float().to(DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = dict(case=c)
    nk, hd = c["nk"], c["hd"]
    if c["op"] in ("attn", "step"):
        lens = _lens(c)
        st["maxpages"] = max(1, _pages(c["hi"]) + 1)
        st["table"], npages = _table(lens, st["maxpages"], g, 3)
        st["pool"] = _pool(npages, nk, hd, g)
        st["lens"] = _int(lens)
        st["qkv"] = torch.randn(c["B"], (c["nq"] + 2 * nk) * hd, generator=g, device=DEV).bfloat16()
        st["out"] = torch.empty(c["B"], c["nq"] * hd, dtype=torch.bfloat16, device=DEV)
        st["longest"] = max(lens)
        if c["op"] == "step":
            st["held"] = torch.empty(c["B"], 2 * nk * hd, dtype=torch.bfloat16, device=DEV)
            st["cos"], st["sin"] = _rotary(c["hi"], hd) if c["rope"] else (None, None)
    elif c["op"] == "store":
        counts = _counts(c)
        ends = [n + c["start"] for n in counts]
        st["maxpages"] = _pages(c["rows"] + c["start"]) or 1
        st["table"], npages = _table(ends, st["maxpages"], g, 1)
        st["pool"] = _pool(npages, nk, hd, g)
        st["start"], st["count"], st["lens"] = _int([c["start"]] * c["B"]), _int(counts), _int(ends)
        st["qkv"] = torch.randn(c["B"] * c["rows"], (c["nq"] + 2 * nk) * hd, generator=g, device=DEV).bfloat16()
        st["maxlen"] = c["rows"] + c["start"]
        st["kc"] = torch.zeros(c["B"], nk, st["maxlen"], hd, dtype=torch.bfloat16, device=DEV)
        st["vc"] = torch.zeros_like(st["kc"])
    elif c["op"] == "fork":
        # the takes still hold the pages of the text before; take 0 holds the new prompt
        lens = [c["prompt"]] + [1 + _mix(i, 4) % 300 for i in range(1, c["B"])]
        st["maxpages"] = max(_pages(n) for n in lens) + 2
        st["table"], npages = _table(lens, st["maxpages"], g, 2 * c["B"] + 2)
        st["lens"] = _int(lens)
        st["ref"] = torch.zeros(npages, dtype=torch.int32, device=DEV)
        st["ref"][st["table"][st["table"] >= 0].long()] = 1
        st["src"], st["dst"] = _int([0] * (c["B"] - 1)), _int(list(range(1, c["B"])))
        st["pools"] = _bytes(c, npages, g)
        st["status"] = torch.zeros(2, dtype=torch.int32, device=DEV)
    else:
        ids = _live_ids(c)
        st["maxpages"] = _pages(PAGE * -(-len(ids) // c["B"]))
        perm = torch.tensor(ids, device=DEV)[torch.randperm(len(ids), generator=g, device=DEV)].to(torch.int32)
        table = torch.full((c["B"] * st["maxpages"],), -1, dtype=torch.int32, device=DEV)
        table[:len(ids)] = perm
        st["table0"] = table.view(c["B"], st["maxpages"])
        st["ref0"] = torch.zeros(c["npages"], dtype=torch.int32, device=DEV)
        st["ref0"][perm.long()] = 1
        if c["B"] > 1 and st["maxpages"] > 1:  # the last take shares the first one's first page
            st["table0"][-1] = -1
            st["ref0"][:] = 0
            st["ref0"][st["table0"][st["table0"] >= 0].long()] = 1
            st["table0"][-1, 0] = st["table0"][0, 0]
            st["ref0"][st["table0"][0, 0].long()] += 1
        st["table"], st["ref"] = st["table0"].clone(), st["ref0"].clone()
        st["pools"] = _bytes(c, c["npages"], g)
        st["status"] = torch.zeros(2, dtype=torch.int32, device=DEV)
    return st


def _bytes(c, npages, g):
    n = PAGE * c["nk"] * 2 * (c["hd"] // 2 + c["hd"] // 8)
    return torch.randint(0, 256, (c["layers"], npages, n), dtype=torch.uint8, generator=g, device=DEV)


# ------------------------------------------------------------------------------------------------ the format, plain

def _quantise(x):
    """Codes, scales and zeros of x [..., hd] (scales and zeros [..., hd / 32]), computed in x's type."""
    x = x.unflatten(-1, (-1, 32))
    z = x.amin(-1)
    r = (x.amax(-1) - z) / 15
    b = (r.float().view(torch.int32) & -65536).view(torch.float32)  # the bf16 at or below r (or r's rounding up)
    up = (b.view(torch.int32) + 65536).view(torch.float32)
    s = torch.where(b.to(x.dtype) < r, up, b).to(x.dtype)
    n = torch.round((x - z[..., None]) / torch.where(s > 0, s, torch.ones_like(s))[..., None])
    return n.to(torch.uint8).flatten(-2), s, z


def _pack(kn, ks, kz, vn, vs, vz):
    """Pages [n][nk * bytes] of codes [n][nk][64][hd] and their scales and zeros."""
    n, nk, _, hd = kn.shape
    W = hd // 32
    # K: half, block of 8, position, w, t, pair of pairs, pair, parity -> a lane's words, low halves first
    k = kn.view(n, nk, 2, 4, 8, W, 4, 2, 2, 2).permute(0, 1, 2, 3, 4, 6, 5, 9, 7, 8)
    # V: half, block of 8, pair of positions, parity, w, lane row, pair, parity of the channel
    v = vn.view(n, nk, 2, 4, 4, 2, W, 8, 2, 2).permute(0, 1, 2, 3, 7, 4, 6, 5, 8, 9)
    k, v = ((x[..., 0] | (x[..., 1] << 4)).reshape(n, nk, 2, -1) for x in (k, v))
    meta = [torch.cat((a, b), -1).bfloat16().view(n, nk, 2, -1).view(torch.uint8) for a, b in ((ks, kz), (vs, vz))]
    return torch.cat((k, v, *meta), -1).reshape(n, -1)


def _unpack(pages, nk, hd):
    """K and V [n][nk][64][hd] in 32 bits that pages stand for."""
    n, W = pages.shape[0], hd // 32
    p = pages.view(n, nk, 2, -1)
    k, v, km, vm = p.split([16 * hd, 16 * hd, 128 * W, 128 * W], -1)
    k = torch.stack((k & 15, k >> 4), -1).view(n, nk, 2, 4, 8, 4, W, 2, 2, 2).permute(0, 1, 2, 3, 4, 6, 5, 8, 9, 7)
    v = torch.stack((v & 15, v >> 4), -1).view(n, nk, 2, 4, 8, 4, W, 2, 2, 2).permute(0, 1, 2, 3, 5, 7, 6, 4, 8, 9)
    out = []
    for x, m in ((k, km), (v, vm)):
        s, z = m.contiguous().view(torch.bfloat16).float().view(n, nk, PAGE, 2, W, 1).unbind(3)
        out.append((x.reshape(n, nk, PAGE, W, 32).float() * s + z).flatten(-2))
    return out


def _slots(pool, table, longest, nk, hd):
    """K and V [B][nk][positions][hd] of every take's first `longest` positions (what no page holds is page 0's)."""
    t = table[:, :_pages(longest)].clamp(min=0).long()
    return [x[t].transpose(1, 2).flatten(2, 3) for x in _unpack(pool, nk, hd)]


def _rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).bfloat16().float()


# ------------------------------------------------------------------------------------------------ the operators, plain

def _attend(q, k, v, lens, scale):
    B, nk = k.shape[:2]
    s = torch.einsum("bhgd,bhld->bhgl", q.view(B, nk, -1, q.shape[-1]), k) * scale
    gone = torch.arange(k.shape[2], device=DEV) >= lens.view(B, 1, 1, 1)
    s = s.masked_fill(gone, -torch.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38)).masked_fill(gone, 0.0)
    v = v.masked_fill(gone.view(B, 1, -1, 1), 0.0)
    l = p.sum(-1, keepdim=True)
    return (torch.einsum("bhgl,bhld->bhgd", p, v) / torch.where(l > 0, l, torch.ones_like(l))).bfloat16().view(B, -1)


def _plain_attn(st):
    c = st["case"]
    B, nq, nk, hd = c["B"], c["nq"], c["nk"], c["hd"]
    q, kn, vn = st["qkv"].float().view(B, -1, hd).split([nq, nk, nk], 1)
    k, v = _slots(st["pool"], st["table"], max(1, st["longest"]), nk, hd)
    if c["op"] == "attn":
        return _attend(q, k, v, st["lens"], hd ** -0.5)
    last = (st["lens"] - 1).clamp(min=0).long()
    if c["rope"]:
        cos, sin = st["cos"][last][:, None], st["sin"][last][:, None]
        q, kn = _rotate(q, cos, sin), _rotate(kn, cos, sin)
    held = []
    for x, slots in ((kn, k), (vn, v)):
        n, s, z = _quantise(x.double())
        y = (n.double().unflatten(-1, (-1, 32)) * s[..., None] + z[..., None]).flatten(-2)
        slots[torch.arange(B, device=DEV), :, last] = y.float()
        held.append(y * (st["lens"] > 0).view(B, 1, 1))
    return _attend(q, k, v, st["lens"], hd ** -0.5), torch.cat(held, 1).bfloat16().view(B, -1)


def _plain_store(st):
    c = st["case"]
    B, nq, nk, hd, rows = c["B"], c["nq"], c["nk"], c["hd"], c["rows"]
    x = st["qkv"].view(B, rows, -1, hd)[:, :, nq:].double()
    n, s, z = _quantise(x)
    y = (n.double().unflatten(-1, (-1, 32)) * s[..., None] + z[..., None]).flatten(-2)
    old = _slots(st["pool"], st["table"], st["maxlen"], nk, hd)
    at = torch.arange(st["maxlen"], device=DEV)
    new = (at >= st["start"][:, None]) & (at < st["lens"][:, None])
    row = (at - st["start"][:, None]).clamp(0, rows - 1).long()
    for i, slot in enumerate((st["kc"], st["vc"])):
        z = y[:, :, i * nk:(i + 1) * nk].transpose(1, 2).float()
        z = z.gather(2, row[:, None, :, None].expand(B, nk, st["maxlen"], hd))
        z = torch.where(new[:, None, :, None], z, old[i][:, :, :st["maxlen"]])
        slot.copy_(torch.where((at < st["lens"][:, None])[:, None, :, None], z.bfloat16(), slot))
    return st["kc"], st["vc"]


def _plain_fork(st):
    table, ref, lens, src, dst = st["table"], st["ref"], st["lens"], st["src"].long(), st["dst"].long()
    P = table.shape[1]
    at = torch.arange(P, device=DEV)

    def count(rows, sign):  # rows' pages, each counted up or down in ref
        ref.index_add_(0, rows.clamp(min=0).flatten().long(), sign * (rows >= 0).flatten().int())

    count(table[dst], -1)
    full, part = lens[src] // PAGE, (lens[src] % PAGE > 0).int()
    rows = torch.where(at < full[:, None], table[src], -1)
    count(rows, 1)
    free = torch.argsort((ref != 0).int(), stable=True)
    mine = free[(part.cumsum(0) - 1).clamp(min=0)]
    old = table[src].gather(1, full[:, None].long())[:, 0]
    takes = part.bool()
    rows = torch.where((at == full[:, None]) & takes[:, None], mine[:, None].int(), rows)
    st["pools"][:, mine[takes]] = st["pools"][:, old[takes].long()]
    ref.index_add_(0, mine, part)
    table[dst] = rows
    lens[dst] = lens[src]
    # pages for one position more
    want = torch.where(lens > 0, -torch.div(-(lens + 1), PAGE, rounding_mode="floor"), 0)
    need = (at < want[:, None]) & (table < 0)
    free = torch.argsort((ref != 0).int(), stable=True)
    order = (need.flatten().cumsum(0) - 1).clamp(min=0)
    table.copy_(torch.where(need, free[order].view_as(table).int(), table))
    ref.index_add_(0, free[order], need.flatten().int())
    return table, ref, lens, st["pools"]


def _plain_compact(st):
    table, ref = st["table"].copy_(st["table0"]), st["ref"].copy_(st["ref0"])
    live = ref > 0
    n = int(live.sum())
    to, old = (~live[:n]).nonzero()[:, 0], live[n:].nonzero()[:, 0] + n
    st["pools"][:, to] = st["pools"][:, old]
    new = torch.arange(len(ref), device=DEV, dtype=torch.int32)
    new[old] = to.int()
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()], table))
    ref[to] = ref[old]
    ref[n:] = 0
    return table, ref, st["pools"]


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    st, c = state, state["case"]
    op = c["op"]
    if not own:
        return {"attn": _plain_attn, "step": _plain_attn, "store": _plain_store, "fork": _plain_fork,
                "compact": _plain_compact}[op](st)
    from oumu_b200 import ops
    if op == "fork":
        ops.pages_fork(st["pools"], st["table"], st["ref"], st["lens"], st["src"], st["dst"], st["status"])
        ops.pages_extend(st["table"], st["ref"], st["lens"], 1, st["status"])
        return st["table"], st["ref"], st["lens"], st["pools"]
    if op == "compact":
        if "ws" not in st:
            st["ws"] = ops.pages_workspace(c["npages"], DEV)
        st["table"].copy_(st["table0"])
        st["ref"].copy_(st["ref0"])
        ops.pages_compact(st["pools"], st["table"], st["ref"], st["ws"], st["status"])
        return st["table"], st["ref"], st["pools"]
    B, nq, nk, hd = c["B"], c["nq"], c["nk"], c["hd"]
    if op == "store":
        ops.kv4_write(st["qkv"], st["pool"], st["table"], st["start"], st["count"], B, c["rows"], nq, nk, hd)
        ops.kv4_read(st["pool"], st["table"], st["lens"], st["kc"], st["vc"], nk, hd)
        return st["kc"], st["vc"]
    if "ws" not in st:
        st["ws"] = ops.decode_kv4_workspace(B, nq, nk, hd, st["maxpages"], DEV)
    if op == "attn":
        ops.attn_decode_kv4(st["qkv"], st["pool"], st["out"], st["ws"], st["table"], None, st["lens"], B, nq, nk, hd,
                            hd ** -0.5)
        return st["out"]
    ops.attn_decode_kv4_step(st["qkv"], st["pool"], st["out"], st["ws"], st["cos"], st["sin"], st["table"], None,
                             st["lens"], B, nq, nk, hd, hd ** -0.5, held=st["held"])
    return st["out"], st["held"]


# ------------------------------------------------------------------------------------------------ in 64 bits

def _where(hd, kind):
    """Byte and shift of every (position, channel)'s code inside a (page, head) unit, from the words' definition:
    K: word [position % 8][channel % 32 / 8][channel / 32] of its block, nibble (channel % 8) / 2 of the low (even
    channel) or high half; V: word [channel % 32 / 4][position % 8 / 2][channel / 32], nibble channel % 4 of the low
    (even position) or high half."""
    W = hd // 32
    p = torch.arange(PAGE, device=DEV)[:, None]
    c = torch.arange(hd, device=DEV)[None]
    if kind == "k":
        word, bit = ((p % 8) * 4 + c % 32 // 8) * W + c // 32, 16 * (c % 2) + 4 * (c % 8 // 2) + 0 * p
    else:
        word, bit = (c % 32 // 4 * 4 + p % 8 // 2) * W + c // 32, 16 * (p % 2) + 4 * (c % 4)
    half = 32 * hd + 256 * W
    byte = p // 32 * half + (0 if kind == "k" else 16 * hd) + p % 32 // 8 * (4 * hd) + 4 * word + bit // 8
    meta = p // 32 * half + 32 * hd + (0 if kind == "k" else 128 * W) + p % 32 * 4 * W + 2 * (c // 32)
    return byte.flatten(), (bit % 8).flatten(), meta.flatten(), 2 * W


def _values(units, hd, kind):
    """[n][64][hd] in 64 bits of units [n][bytes]."""
    byte, shift, meta, zero = _where(hd, kind)
    code = (units[:, byte].int() >> shift.int()) & 15

    def bf16(at):
        return ((units[:, at].int() << 16) | (units[:, at + 1].int() << 24)).view(torch.float32).double()

    return (code.double() * bf16(meta) + bf16(meta + zero)).view(-1, PAGE, hd)


def _held64(x):
    """What x [n][hd] (64 bits) is held as, group by group."""
    y = torch.empty_like(x)
    for a in range(0, x.shape[1], 32):
        g = x[:, a:a + 32]
        z, top = g.min(1, keepdim=True).values, g.max(1, keepdim=True).values
        want = (top - z) / 15
        _, e = torch.frexp(want)
        ulp = torch.ldexp(torch.ones_like(want), (e - 8).clamp(min=-133))
        s = torch.ceil(want / ulp) * ulp
        y[:, a:a + 32] = torch.where(s > 0, torch.round((g - z) / torch.where(s > 0, s, 1.0)) * s + z, g)
    return y


def exact(case, seed):
    c = case
    if c["op"] in ("fork", "compact"):
        return None
    st = prepare(c, seed)
    B, nq, nk, hd = c["B"], c["nq"], c["nk"], c["hd"]
    units = st["pool"].view(-1, nk, 2 * (32 * hd + 8 * hd))
    x = st["qkv"].double().view(-1, nq + 2 * nk, hd)
    if c["op"] == "store":
        outs = [torch.zeros(B, nk, st["maxlen"], hd, dtype=torch.float64, device=DEV) for _ in range(2)]
        for s, n in enumerate(_counts(c)):
            end = c["start"] + n
            pages = st["table"][s, :_pages(end)].long()
            for h in range(nk):
                for i, kind in enumerate("kv"):
                    if end:
                        outs[i][s, h, :end] = _values(units[pages, h], hd, kind).view(-1, hd)[:end]
                    outs[i][s, h, c["start"]:end] = _held64(x[s * c["rows"]:s * c["rows"] + n, nq + i * nk + h])
        return tuple(outs)
    out = torch.zeros(B, nq, hd, dtype=torch.float64, device=DEV)
    held = torch.zeros(B, 2 * nk, hd, dtype=torch.float64, device=DEV)
    for s, n in enumerate(_lens(c)):
        if n == 0:
            continue
        pages, row = st["table"][s, :_pages(n)].long(), x[s].clone()
        if c["op"] == "step":
            if c["rope"]:
                a, b = row[:nq + nk, :hd // 2].clone(), row[:nq + nk, hd // 2:].clone()
                cs, sn = st["cos"][n - 1].double(), st["sin"][n - 1].double()
                row[:nq + nk, :hd // 2] = (a * cs - b * sn).bfloat16().double()
                row[:nq + nk, hd // 2:] = (b * cs + a * sn).bfloat16().double()
            held[s] = _held64(row[nq:])
        for h in range(nk):
            k, v = (_values(units[pages, h], hd, kind).view(-1, hd)[:n] for kind in "kv")
            if c["op"] == "step":
                k[n - 1], v[n - 1] = held[s, h], held[s, nk + h]
            heads = slice(h * (nq // nk), (h + 1) * (nq // nk))
            w = torch.softmax(row[heads] @ k.t() * hd ** -0.5, -1)
            out[s, heads] = w @ v
    out, held = out.view(B, -1), held.view(B, -1)
    return (out, held) if c["op"] == "step" else out
