"""The workloads by which the linear-attention and state-page operators are measured.

Operators: linear attention with a decay for each head (``lin_prefill``, the
chunked form for prompts, and ``lin_decode``, the recurrent form for single
tokens), and the pages of a cache of recurrent states (``pages_copy``,
``pages_fork``, ``pages_free``, ``pages_compact``).

    S_t = exp(g_t) S_{t-1} + k_t v_t^T        o_t = scale * S_t^T q_t

With ``own`` false every operator runs in a plain form made of elementary
torch operations in fp32 (decays in fp64); with ``own`` true the calls go to
this repository's package.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
IO = {"bf16": torch.bfloat16, "f16": torch.float16}


def _prefill(name, B, T, Hqk, Hv, dk, dv, io="bf16", gate="token", packed=False, init=False, paged=False):
    # packed: B sequences of ragged lengths, T tokens in all; paged: states live in a pool
    return {"name": name, "kind": "prefill", "B": B, "T": T, "Hqk": Hqk, "Hv": Hv, "dk": dk, "dv": dv, "io": io,
            "gate": gate, "packed": packed, "init": init, "paged": paged}


def _decode(name, B, Hqk, Hv, dk, dv, io="bf16", gate="token", pages=0):
    # pages > 0: a pool of that many pages, rows find theirs by index, some rows are idle
    return {"name": name, "kind": "decode", "B": B, "Hqk": Hqk, "Hv": Hv, "dk": dk, "dv": dv, "io": io, "gate": gate,
            "pages": pages}


def _pages(name, op, P, n, layers, H, dk, dv, ways=1):
    # n: pages copied, forked (into `ways` children each) or freed before compaction
    return {"name": name, "kind": op, "P": P, "n": n, "layers": layers, "H": H, "dk": dk, "dv": dv, "ways": ways}


def listed():
    return [
        # one short prompt of a small model: launch latency
        _prefill("prefill_short", 1, 61, 8, 8, 64, 64),
        # the prefill configuration of this repository's benchmark: four prompts of 4096 tokens
        _prefill("prefill_batch", 4, 4096, 16, 32, 128, 128),
        # a serving step's ragged prompts, packed without padding, continuing from pages of a state pool
        _prefill("prefill_packed", 24, 9001, 4, 32, 128, 64, io="f16", packed=True, init=True, paged=True),
        # one long document: few rows, a long time axis; a fixed decay per head
        _prefill("prefill_long", 1, 32768, 32, 32, 128, 128, gate="head"),
        # decode of a few sequences: latency
        _decode("decode_small", 8, 16, 32, 128, 128),
        # the headline batch of this repository's decode benchmark
        _decode("decode_large", 1024, 16, 32, 128, 128),
        # continuous batching: rows point at pages, some rows idle; a fixed decay per head
        _decode("decode_paged", 301, 16, 16, 64, 128, io="f16", gate="head", pages=384),
        # one sequence forked once: latency
        _pages("fork_one", "fork", 32, 1, 1, 8, 64, 64),
        # parallel sampling: 16 prompts forked into 4 each, two layers
        _pages("fork_samples", "fork", 256, 16, 2, 32, 128, 128, ways=4),
        # pages moved to given places (a swap with a staging area), four layers
        _pages("copy_pages", "copy", 160, 40, 4, 16, 128, 64),
        # finished sequences leave a small batch: freed, then the rest compacted
        _pages("turnover_small", "turnover", 48, 11, 1, 8, 64, 64),
        # the same for a large batch of the benchmark's state size
        _pages("turnover_large", "turnover", 512, 211, 1, 32, 128, 128),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prefill", "prefill", "prefill", "decode", "decode", "fork", "copy", "turnover"])
    if kind == "prefill":
        group = rng.choice([1, 1, 2, 4, 8])
        Hqk = _log_int(rng, 1, 64 // group)
        Hv = Hqk * group
        dk, dv = rng.choice([64, 128]), rng.choice([64, 128, 128, 192, 256])
        packed = rng.random() < 0.4
        tokens = _log_int(rng, 1, min(65536, (1 << 27) // (Hv * max(dk, dv))))
        B = _log_int(rng, 1, 32)
        T = max(tokens, B) if packed else max(1, tokens // B)
        init = rng.random() < 0.5
        c = _prefill("", B, T, Hqk, Hv, dk, dv, io=rng.choice(["bf16", "f16"]), gate=rng.choice(["token", "token", "head"]),
                     packed=packed, init=init, paged=rng.random() < 0.5)
    elif kind == "decode":
        group = rng.choice([1, 1, 2, 4, 8])
        Hqk = _log_int(rng, 1, 64 // group)
        Hv = Hqk * group
        dk, dv = rng.choice([64, 128, 128, 256]), rng.choice([64, 128, 128, 192, 256])
        B = _log_int(rng, 1, min(2048, (1 << 29) // (Hv * dk * dv)))
        pages = B + rng.randrange(0, B + 1) if rng.random() < 0.5 else 0
        c = _decode("", B, Hqk, Hv, dk, dv, io=rng.choice(["bf16", "f16"]), gate=rng.choice(["token", "token", "head"]),
                    pages=pages)
    else:
        H, dk, dv = _log_int(rng, 1, 64), rng.choice([64, 128, 256]), rng.choice([64, 128, 192])
        layers = rng.randrange(1, 7)
        most = max(8, min(1500, (1 << 28) // (H * dk * dv * layers)))
        P = _log_int(rng, 8, most)
        ways = rng.randrange(1, 5) if kind == "fork" else 1
        n = rng.randrange(1, P // (1 + ways) + 1)
        c = _pages("", kind, P, n, layers, H, dk, dv, ways=ways)
    del c["name"]
    return c


def _lengths(c):
    """Ragged lengths that add up to T, by the case alone; some are zero where T allows no more."""
    r = random.Random(c["T"] * 1009 + c["B"])
    cuts = sorted(r.randrange(0, c["T"] + 1) for _ in range(c["B"] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [c["T"]])]


def _gate(c, gen, *shape):
    Hv = c["Hv"]
    if c["gate"] == "head":  # a fixed decay per head, slopes in a geometric series
        h = torch.arange(1, Hv + 1, device=DEV, dtype=torch.float32)
        return -torch.exp2(-8.0 * h / Hv)
    # data-dependent: -A softplus(a + dt), steps between 0.001 and 0.1, A in 1..16
    A = torch.rand(Hv, device=DEV, generator=gen) * 15 + 1
    dt = torch.exp(torch.rand(Hv, device=DEV, generator=gen) * math.log(100) + math.log(1e-3))
    bias = dt + torch.log(-torch.expm1(-dt))
    a = torch.randn(*shape, Hv, device=DEV, generator=gen) * 0.5
    return -A * torch.nn.functional.softplus(a + bias)


def _package():
    import __graft_entry__ as graft

    return graft.package()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=gen).to(dtype)

    s = {"case": c}
    if c["kind"] == "prefill":
        io, B, T = IO[c["io"]], c["B"], c["T"]
        lead = (1, T) if c["packed"] else (B, T)
        s["q"] = randn(*lead, c["Hqk"], c["dk"], dtype=io)
        s["k"] = randn(*lead, c["Hqk"], c["dk"], dtype=io)
        s["v"] = randn(*lead, c["Hv"], c["dv"], dtype=io)
        s["g"] = _gate(c, gen, *lead)
        s["scale"] = c["dk"] ** -0.5
        s["lens"], s["cu"] = None, None
        if c["packed"]:
            s["lens"] = _lengths(c)
            cu = [0]
            for n in s["lens"]:
                cu.append(cu[-1] + n)
            s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEV)
        s["index"] = None
        rows = B
        if c["paged"]:
            rows = B + max(1, B // 4)
            s["index"] = torch.randperm(rows, device=DEV, generator=gen)[:B].to(torch.int32)
        pool = (rows, c["Hv"], c["dk"], c["dv"])
        s["s0"] = randn(*pool) if c["init"] else None
        s["pool"] = randn(*pool) if c["paged"] else torch.zeros(pool, device=DEV)
    elif c["kind"] == "decode":
        io, B = IO[c["io"]], c["B"]
        s["q"], s["k"] = randn(B, c["Hqk"], c["dk"], dtype=io), randn(B, c["Hqk"], c["dk"], dtype=io)
        s["v"] = randn(B, c["Hv"], c["dv"], dtype=io)
        s["g"] = _gate(c, gen, B)
        s["scale"] = c["dk"] ** -0.5
        s["index"] = None
        rows = B
        if c["pages"]:
            rows = c["pages"]
            index = torch.randperm(rows, device=DEV, generator=gen)[:B]
            idle = torch.rand(B, device=DEV, generator=gen) < 1 / 16
            s["index"] = torch.where(idle, -1, index).to(torch.int32)
        s["state"] = randn(rows, c["Hv"], c["dk"], c["dv"])
    else:
        P, n = c["P"], c["n"]
        s["pools"] = [randn(P, c["H"], c["dk"], c["dv"]) for _ in range(c["layers"])]
        order = torch.randperm(P, device=DEV, generator=gen)
        s["used_out"] = torch.zeros(P, dtype=torch.int32, device=DEV)
        if c["kind"] == "fork":  # a third of what the children leave is free as well
            spare = (P - n - n * c["ways"]) // 3
            used = torch.ones(P, dtype=torch.int32, device=DEV)
            used[order[: n * c["ways"] + spare]] = 0
            s["used"] = used
            s["src"] = order[-n:].repeat_interleave(c["ways"]).to(torch.int32)
        elif c["kind"] == "copy":
            s["src"], s["dst"] = order[:n].to(torch.int32), order[n : 2 * n].to(torch.int32)
        else:
            s["used"] = torch.ones(P, dtype=torch.int32, device=DEV)
            s["done"] = order[:n].to(torch.int32)
            s["used_mid"] = torch.zeros(P, dtype=torch.int32, device=DEV)
            s["rows"] = order[n:].to(torch.int32)  # the live sequences' pages, in the order of their rows
    return s


# ---------------------------------------------------------------- plain forms


def _padded(x, lens, fill_to):
    """Packed [1, T, ...] as [N, fill_to, ...], zeros behind each sequence."""
    out = x.new_zeros(len(lens), fill_to, *x.shape[2:])
    t = torch.arange(fill_to, device=x.device)
    n = torch.tensor(lens, device=x.device)
    live = t[None, :] < n[:, None]
    out[live] = x[0]
    return out, live


def _plain_prefill(s):
    c, C = s["case"], 64
    q, k, v, g = s["q"].float(), s["k"].float(), s["v"].float(), s["g"].double()
    if g.dim() == 1:
        g = g.expand(*v.shape[:3])
    live = None
    if s["lens"] is not None:
        most = max(s["lens"])
        (q, live), (k, _), (v, _), (g, _) = (_padded(x, s["lens"], most) for x in (q, k, v, g))
    N, T = v.shape[:2]
    nc = max(1, -(-T // C))
    pad = nc * C - T
    group = c["Hv"] // c["Hqk"]

    def chunks(x):  # [N, T, H, ...] -> [N, H, nc, C, ...]
        x = torch.cat([x, x.new_zeros(N, pad, *x.shape[2:])], 1) if pad else x
        return x.reshape(N, nc, C, *x.shape[2:]).movedim(3, 1)

    q, k = (chunks(x).repeat_interleave(group, 1) for x in (q, k))
    v, G = chunks(v), chunks(g).reshape(N, c["Hv"], nc * C).cumsum(2).reshape(N, c["Hv"], nc, C)
    end = G[..., -1]  # decay up to each chunk's end
    start = torch.cat([torch.zeros_like(end[..., :1]), end[..., :-1]], 2)
    low = torch.ones(C, C, device=q.device, dtype=torch.bool).tril()
    p = q @ k.transpose(-1, -2)
    diff = (G - start[..., None])[..., :, None] - (G - start[..., None])[..., None, :]
    p = p * torch.where(low, diff, -math.inf).float().exp()
    del diff
    o = p @ v
    del p
    local = (k * (end[..., None] - G).exp().float()[..., None]).transpose(-1, -2) @ v  # [N, H, nc, dk, dv]
    carry = torch.ones(nc, nc, device=q.device, dtype=torch.bool).tril(-1)
    w = torch.where(carry, start[..., :, None] - end[..., None, :], -math.inf).exp().float()
    begin = (w @ local.flatten(3)).reshape_as(local)
    last = ((end[..., -1:] - end).exp().float()[..., None, :] @ local.flatten(3)).reshape(N, c["Hv"], c["dk"], c["dv"])
    if s["s0"] is not None:
        s0 = s["s0"] if s["index"] is None else s["s0"][s["index"].long()]
        begin = begin + start.exp().float()[..., None, None] * s0[:, :, None]
        last = last + end[..., -1].exp().float()[..., None, None] * s0
    o = o + (q * (G - start[..., None]).exp().float()[..., None]) @ begin
    o = (o * s["scale"]).movedim(1, 3).reshape(N, nc * C, c["Hv"], c["dv"])[:, :T]
    if live is not None:
        o = o[live][None]
    if s["index"] is None:
        s["pool"].copy_(last)
    else:
        s["pool"][s["index"].long()] = last
    return o.to(s["v"].dtype), s["pool"]


def _plain_decode(s):
    c, group = s["case"], s["case"]["Hv"] // s["case"]["Hqk"]
    q, k = (x.float().repeat_interleave(group, 1) for x in (s["q"], s["k"]))
    v = s["v"].float()
    a = s["g"].float().exp().expand(c["B"], c["Hv"])
    if s["index"] is None:
        new = s["state"] * a[..., None, None] + k[..., None] * v[..., None, :]
        s["state"].copy_(new)
        o = (q[..., None, :] @ new)[..., 0, :] * s["scale"]
    else:
        row = (s["index"] >= 0).nonzero()[:, 0]
        page = s["index"][row].long()
        new = s["state"][page] * a[row][..., None, None] + k[row][..., None] * v[row][..., None, :]
        s["state"][page] = new
        o = torch.zeros_like(v)
        o[row] = (q[row][..., None, :] @ new)[..., 0, :] * s["scale"]
    return o.to(s["v"].dtype), s["state"]


def _plain_fork(s):
    used = s["used"]
    free_first = used.argsort(stable=True)  # free pages come first, the lowest ones in front
    dst = free_first[: s["src"].numel()]
    s["used_out"].copy_(used)
    s["used_out"][dst] = 1
    for pool in s["pools"]:
        pool[dst] = pool[s["src"].long()]
    return dst.to(torch.int32), s["used_out"], s["pools"]


def _plain_copy(s):
    for pool in s["pools"]:
        pool[s["dst"].long()] = pool[s["src"].long()]
    return s["pools"]


def _plain_turnover(s):
    used = s["used"].clone()
    used[s["done"].long()] = 0
    page = torch.arange(used.numel(), device=used.device)
    count = used.sum()
    hole = ((used == 0) & (page < count)).nonzero()[:, 0]
    mover = ((used != 0) & (page >= count)).nonzero()[:, 0]
    remap = torch.where(used != 0, page, -1)
    remap[mover] = hole
    for pool in s["pools"]:
        pool[hole] = pool[mover]
    s["used_out"].copy_(page < count)
    return remap.to(torch.int32), count.to(torch.int32)[None], remap[s["rows"].long()].to(torch.int32), s["used_out"], s["pools"]


# ---------------------------------------------------------------- one pass


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return {"prefill": _plain_prefill, "decode": _plain_decode, "fork": _plain_fork, "copy": _plain_copy,
                "turnover": _plain_turnover}[kind](s)
    pkg = _package()
    if kind == "prefill":
        return pkg.lin_prefill(s["q"], s["k"], s["v"], s["g"], s["s0"], scale=s["scale"], cu_seqlens=s["cu"],
                               index=s["index"], final_state=s["pool"])
    if kind == "decode":
        return pkg.lin_decode(s["q"], s["k"], s["v"], s["g"], s["state"], scale=s["scale"], index=s["index"]), s["state"]
    if kind == "fork":
        dst = pkg.pages_fork(s["pools"], s["used"], s["src"], used_out=s["used_out"])
        return dst, s["used_out"], s["pools"]
    if kind == "copy":
        pkg.pages_copy(s["pools"], s["src"], s["dst"])
        return s["pools"]
    pkg.pages_free(s["used"], s["done"], used_out=s["used_mid"])
    remap, count, rows = pkg.pages_compact(s["pools"], s["used_mid"], index=s["rows"], used_out=s["used_out"])
    return remap, count, rows, s["used_out"], s["pools"]


# ---------------------------------------------------------------- floors


def work(case):
    c = case
    if c["kind"] == "prefill":
        tokens = c["T"] if c["packed"] else c["B"] * c["T"]
        page = c["Hv"] * c["dk"] * c["dv"]
        data = tokens * 2 * (2 * c["Hqk"] * c["dk"] + 2 * c["Hv"] * c["dv"])
        gate = 4 * c["Hv"] * (tokens if c["gate"] == "token" else 1)
        return {"bytes": data + gate + 4 * c["B"] * page * (2 if c["init"] else 1), "flops": 4 * tokens * page}
    if c["kind"] == "decode":
        page = c["Hv"] * c["dk"] * c["dv"]
        live = c["B"] * (15 / 16 if c["pages"] else 1)
        rows = c["B"] * 2 * (2 * c["Hqk"] * c["dk"] + 2 * c["Hv"] * c["dv"])
        gate = 4 * c["Hv"] * (c["B"] if c["gate"] == "token" else 1)
        return {"bytes": rows + gate + 8 * live * page, "flops": 5 * live * page}
    page = 4 * c["H"] * c["dk"] * c["dv"] * c["layers"]
    if c["kind"] == "fork":
        return {"bytes": c["n"] * (1 + c["ways"]) * page + 8 * c["P"] + 8 * c["n"] * c["ways"], "flops": 0}
    if c["kind"] == "copy":
        return {"bytes": 2 * c["n"] * page + 8 * c["n"], "flops": 0}
    live = c["P"] - c["n"]  # of the live pages the share n / P lies behind the first `live` places
    return {"bytes": 2 * page * live * c["n"] / c["P"] + 4 * (5 * c["P"] + 3 * c["n"]), "flops": 0}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_steps(q, k, v, g, S, scale):
    """One sequence or a batch of equal ones, token by token: q, k, v [B, T, H, d], g [B, T, H], S [B, H, dk, dv]."""
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    S = S.reshape(B * H, dk, dv).clone()
    q, k, v = (x.transpose(0, 1).flatten(1, 2) for x in (q, k, v))
    a = g.exp().transpose(0, 1).reshape(T, B * H, 1, 1)
    o = torch.empty(T, B * H, dv, dtype=torch.float64, device=q.device)
    for t in range(T):
        S.mul_(a[t]).baddbmm_(k[t][:, :, None], v[t][:, None, :])
        torch.bmm(q[t][:, None, :], S, out=o[t][:, None, :])
    return (o * scale).reshape(T, B, H, dv).transpose(0, 1), S.reshape(B, H, dk, dv)


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["kind"] == "prefill":
        group = c["Hv"] // c["Hqk"]
        q, k, v = (s[x].double() for x in "qkv")
        q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
        g = s["g"].double().expand(*v.shape[:3])
        pool = s["pool"].double()
        pages = s["index"].tolist() if s["index"] is not None else list(range(c["B"]))
        zero = torch.zeros(c["B"], *pool.shape[1:], dtype=torch.float64, device=DEV)
        S = zero if s["s0"] is None else s["s0"].double()[pages]
        if c["packed"]:
            o, at = torch.empty_like(v), 0
            for i, n in enumerate(s["lens"]):
                part = [x[:, at : at + n] for x in (q, k, v, g)]
                o[:, at : at + n], S[i : i + 1] = _exact_steps(*part, S[i : i + 1], s["scale"])
                at += n
        else:
            o, S = _exact_steps(q, k, v, g, S, s["scale"])
        pool[pages] = S
        return o, pool
    if c["kind"] == "decode":
        pool = s["state"].double()
        rows = list(range(c["B"])) if s["index"] is None else s["index"].tolist()
        group = c["Hv"] // c["Hqk"]
        live = [i for i, p in enumerate(rows) if p >= 0]
        pages = [rows[i] for i in live]
        o = torch.zeros(c["B"], c["Hv"], c["dv"], dtype=torch.float64, device=DEV)
        g = s["g"].double().expand(c["B"], c["Hv"])
        for lo in range(0, len(live), 128):  # a few rows at a time: 64-bit copies of the states are large
            i, p = live[lo : lo + 128], pages[lo : lo + 128]
            k, q = (s[x][i].double().repeat_interleave(group, 1) for x in "kq")
            S = torch.einsum("bh,bhkv->bhkv", g[i].exp(), pool[p]) + torch.einsum("bhk,bhv->bhkv", k, s["v"][i].double())
            pool[p] = S
            o[i] = torch.einsum("bhk,bhkv->bhv", q, S) * s["scale"]
        return o, pool
    pools = [p.double() for p in s["pools"]]
    if c["kind"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            for p in pools:
                p[b] = p[a]
        return pools
    used = s["used"].tolist()
    if c["kind"] == "fork":
        dst = []
        for a in s["src"].tolist():
            b = used.index(0)
            used[b] = 1
            dst.append(b)
            for p in pools:
                p[b] = p[a]
        return torch.tensor(dst, dtype=torch.int32), torch.tensor(used, dtype=torch.int32), pools
    for b in s["done"].tolist():
        used[b] = 0
    count = sum(used)
    remap = [i if u else -1 for i, u in enumerate(used)]
    for a in range(count, c["P"]):
        if used[a]:
            b = used.index(0)
            used[a], used[b], remap[a] = 0, 1, b
            for p in pools:
                p[b] = p[a]
    i32 = torch.int32
    rows = [remap[r] for r in s["rows"].tolist()]
    return torch.tensor(remap, dtype=i32), torch.tensor([count], dtype=i32), torch.tensor(rows, dtype=i32), torch.tensor(used, dtype=i32), pools
