"""The 4-bit MLA cache (fp4_ds_mla): its operators in plain form, and the calls a user makes of them.

A cache row holds one token in 416 bytes: 512 e2m1 codes of the latent (two per byte, the
lower index in the low nibble), 32 e4m3 scales (one per 16 latent values), 64 bf16 rope values.
A latent value is code * scale.  The operators:

  write    quantise new tokens into their slots, and read those rows back
  gather   read whole sequences back through their block tables, as prefill over a cached
           context does
  sparse   attention of each query token over the slots that an index row names
           ("paged": over positions of its request, through the block table)
  dense    attention of each query token over the first context_len positions of its request
"""

import random

import torch

own = False

NOPE, ROPE, GROUP, ROW = 512, 64, 16, 416
SM_SCALE = 192 ** -0.5
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one new token of one sequence: the write of a decode step, where latency counts
        {"name": "write_1", "op": "write", "n": 1, "slots": 4096, "pad": 0.0},
        # a prefill chunk of odd length, a twentieth of it padding
        {"name": "write_4099_padded", "op": "write", "n": 4099, "slots": 8192, "pad": 0.05},
        # the cache writer's benchmark size
        {"name": "write_65536", "op": "write", "n": 65536, "slots": 131072, "pad": 0.0},
        # the cached context of a prefill batch, lengths from none to 8191
        {"name": "gather_48_ragged", "op": "gather", "B": 48, "len": 8191, "page": 64, "start": 0},
        # two long contexts read from an offset, pages of 16
        {"name": "gather_2_long", "op": "gather", "B": 2, "len": 131071, "page": 16, "start": 37},
        # the smallest decode shape: 4 requests, 16 heads, one index in ten masked
        {"name": "sparse_c1", "op": "sparse", "T": 4, "H": 16, "G": 1, "topk": 256, "slots": 4096, "page": 0, "mask": 0.1},
        # many requests of a tensor-parallel rank with few heads over a large shared pool
        {"name": "sparse_c3", "op": "sparse", "T": 256, "H": 16, "G": 1, "topk": 2048, "slots": 3500032, "page": 0, "mask": 0.0},
        # all 128 heads on one GPU, positions turned into slots through the block table
        {"name": "paged_c2", "op": "sparse", "T": 64, "H": 128, "G": 1, "topk": 2048, "slots": 2097152, "page": 64, "mask": 0.0},
        # 64 heads, a quarter of the indices masked
        {"name": "sparse_c4", "op": "sparse", "T": 32, "H": 64, "G": 1, "topk": 2048, "slots": 1048576, "page": 0, "mask": 0.25},
        # one request with a long context: every SM works on one token
        {"name": "dense_1_long", "op": "dense", "T": 1, "H": 128, "len": 131071, "page": 64, "next_n": 1},
        # a decode batch of ragged contexts on a rank with 16 heads, empty ones among them
        {"name": "dense_64_ragged", "op": "dense", "T": 64, "H": 16, "len": 16384, "page": 64, "next_n": 1},
        # two query tokens a request (a draft token beside the last one), 128 heads
        {"name": "dense_32_mtp", "op": "dense", "T": 32, "H": 128, "len": 8192, "page": 64, "next_n": 2},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["write", "gather", "sparse", "sparse", "dense", "dense"])
    if op == "write":
        n = _log(rng, 1, 65536)
        return {"op": op, "n": n, "slots": n + _log(rng, 1, 65536), "pad": rng.choice([0.0, 0.1, 0.5])}
    page = rng.choice([16, 64, 64, 100, 128])
    if op == "gather":
        B = _log(rng, 1, 64)
        return {"op": op, "B": B, "len": _log(rng, 1, 131071 // B), "page": page, "start": rng.choice([0, 0, _log(rng, 1, 500)])}
    H = rng.choice([1, 4, 8, 16, 16, 24, 32, 40, 64, 96, 128, 128])
    if op == "sparse":
        T = _log(rng, 1, 256)
        topk = _log(rng, 1, min(2048, 64 * 128 * 2048 // (T * H)))
        return {"op": op, "T": T, "H": H, "G": rng.choice([1, 1, 1, 2]) if H % 2 == 0 else 1, "topk": topk,
                "slots": page * (topk // page + 1) * T + page * _log(rng, 1, 4096), "page": rng.choice([0, page]), "mask": rng.choice([0.0, 0.1, 0.6])}
    n = rng.choice([1, 1, 2])
    T = n * _log(rng, 1, 64 // n)
    return {"op": op, "T": T, "H": H, "len": _log(rng, 1, min(131071, 128 * 131071 // (T * H), 262144 // T)), "page": page, "next_n": n}


def _lens(case, B):
    """Lengths of B sequences up to case["len"]: the first has it all, the second none, the third one token."""
    pick = random.Random(B * 1000003 + case["len"])
    lens = [pick.randint(0, case["len"]) for _ in range(B)]
    lens[0] = case["len"]
    if B > 2:
        lens[1], lens[2] = 0, 1
    return lens


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def _pool(g, slots):
    """A cache of `slots` rows, holding quantised tokens."""
    cache = torch.empty(slots, ROW, dtype=torch.uint8, device="cuda")
    for at in range(0, slots, 1 << 18):
        n = min(1 << 18, slots - at)
        cache[at:at + n] = _quantise(_normal(g, n, NOPE), _normal(g, n, ROPE))
    return cache


def _tables(g, pages_each, reqs, pages):
    """Block tables [reqs, pages_each] over distinct pages."""
    return torch.randperm(pages, generator=g, device="cuda")[:reqs * pages_each].view(reqs, pages_each).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "write":
        n, slots = case["n"], case["slots"]
        where = torch.randperm(slots, generator=g, device="cuda")[:n]
        where[torch.rand(n, generator=g, device="cuda") < case["pad"]] = -1
        return {"op": op, "kv_c": _normal(g, n, NOPE), "k_pe": _normal(g, n, ROPE), "slots": where,
                "cache": torch.zeros(slots, ROW, dtype=torch.uint8, device="cuda")}
    if op == "gather":
        lens, page = _lens(case, case["B"]), case["page"]
        each = (case["len"] + case["start"] + page - 1) // page
        cum = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        return {"op": op, "cache": _pool(g, page * each * case["B"]), "table": _tables(g, each, case["B"], each * case["B"]), "page": page,
                "cum": cum, "rows": sum(lens), "starts": torch.full((case["B"],), case["start"], dtype=torch.int32, device="cuda")}
    T, H = case["T"], case["H"]
    state = {"op": op, "q": _normal(g, T, H, NOPE + ROPE), "page": case["page"]}
    if op == "sparse":
        G, topk, slots, page = case["G"], case["topk"], case["slots"], case["page"]
        state["cache"] = _pool(g, slots)
        if page:
            each = slots // page // T
            state["table"] = _tables(g, each, T, slots // page)
            state["req"] = torch.arange(T, dtype=torch.int32, device="cuda")
        reach = each * page if page else slots
        # distinct indices of a row: one from each of topk equal stretches of the reach
        at = torch.arange(topk, device="cuda") * (reach / topk)
        idx = (at + torch.rand(T, G, topk, generator=g, device="cuda", dtype=torch.float64) * (reach / topk)).long().clamp(max=reach - 1)
        idx = idx.gather(2, torch.rand(T, G, topk, generator=g, device="cuda").argsort(2))
        idx[torch.rand(T, G, topk, generator=g, device="cuda") < case["mask"]] = -1
        state["idx"] = idx.to(torch.int32)
        return state
    reqs, page = T // case["next_n"], case["page"]
    lens = _lens(case, reqs)
    each = (case["len"] + page - 1) // page
    state["cache"] = _pool(g, page * each * reqs)
    state["table"] = _tables(g, each, reqs, each * reqs)
    state["req"] = torch.arange(reqs, device="cuda").repeat_interleave(case["next_n"]).to(torch.int32)
    back = torch.arange(case["next_n"] - 1, -1, -1, device="cuda").repeat(reqs)
    state["lens"] = (torch.tensor(lens, device="cuda").repeat_interleave(case["next_n"]) - back).clamp(min=0).to(torch.int32)
    state["most"] = case["len"]
    return state


# ---- plain forms ------------------------------------------------------------------------

def _quantise(kv_c, k_pe):
    """bf16 latents [n, 512] and ropes [n, 64] as packed rows [n, 416]."""
    x = kv_c.float().view(-1, NOPE // GROUP, GROUP)
    scale = (x.abs().amax(2, keepdim=True) / 6).clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn)
    y = x / scale.float()
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + torch.signbit(y).byte() * 8)
    code = code.view(-1, NOPE // 2, 2)
    packed = code[:, :, 0] | (code[:, :, 1] << 4)
    return torch.cat([packed, scale.view(torch.uint8).view(-1, NOPE // GROUP), k_pe.contiguous().view(torch.uint8)], 1)


def _values(rows):
    """Packed rows [n, 416] as values [n, 576] in 32 bits."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=rows.device)
    codes = torch.stack([rows[:, :NOPE // 2] & 15, rows[:, :NOPE // 2] >> 4], 2).view(-1, NOPE // GROUP, GROUP)
    scale = rows[:, NOPE // 2:NOPE // 2 + NOPE // GROUP].contiguous().view(torch.float8_e4m3fn).float()
    latent = (level[codes.int()] * scale[:, :, None]).view(-1, NOPE)
    return torch.cat([latent, rows[:, ROW - 2 * ROPE:].contiguous().view(torch.bfloat16).float()], 1)


def _slots_of(table, req, pos, page):
    return table[req, pos // page].long() * page + pos % page


def _attend(q, cache, slots, live):
    """q [T, H, 576], slots and live [T, G, n]: outputs [T, H, 512] and log-sum-exps [T, H]."""
    T, H, _ = q.shape
    G, n = slots.shape[1:]
    k = _values(cache[slots.clamp(min=0).view(-1)]).view(T, G, n, NOPE + ROPE)
    s = q.float().view(T, G, H // G, -1) @ k.transpose(2, 3) * SM_SCALE
    s = s.masked_fill(~live[:, :, None, :], float("-inf"))
    m = s.amax(3, keepdim=True)
    p = torch.exp(s - m.clamp(min=-3e38))
    l = p.sum(3, keepdim=True)
    out = (p @ k[..., :NOPE]) / l.clamp(min=1e-38)
    return out.to(torch.bfloat16).view(T, H, NOPE), (m + torch.log(l)).view(T, H)


def _plain(s):
    if s["op"] == "write":
        kept = s["slots"] >= 0
        rows = _quantise(s["kv_c"], s["k_pe"])
        s["cache"][s["slots"][kept]] = rows[kept]
        read = _values(s["cache"][s["slots"].clamp(min=0)])
        return (read * kept[:, None]).to(torch.bfloat16)
    if s["op"] == "gather":
        row = torch.arange(s["rows"], device="cuda")
        req = torch.searchsorted(s["cum"].long(), row, right=True) - 1
        pos = row - s["cum"].long()[req] + s["starts"].long()[req]
        return _values(s["cache"][_slots_of(s["table"], req, pos, s["page"])]).to(torch.bfloat16)
    if s["op"] == "sparse":
        live, at = s["idx"] >= 0, s["idx"].long()
        if s["page"]:
            at = _slots_of(s["table"], s["req"].long()[:, None, None], at.clamp(min=0), s["page"])
        return _attend(s["q"], s["cache"], at, live)
    pos = torch.arange(s["most"], device="cuda")[None, None, :]
    live = pos < s["lens"].long()[:, None, None]
    return _attend(s["q"], s["cache"], _slots_of(s["table"], s["req"].long()[:, None, None], pos, s["page"]), live)


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def _own(s):
    import sys
    if "vllm-fp8kv_b200" not in sys.path:
        sys.path.insert(0, "vllm-fp8kv_b200")
    from vllm_fp8kv import fp4_ds_mla as F
    if s["op"] == "write":
        F.concat_and_cache_fp4_ds_mla(s["kv_c"], s["k_pe"], s["cache"], s["slots"])
        return F.dequant_fp4_ds_mla_rows(s["cache"], s["slots"])
    if s["op"] == "gather":
        return F.gather_fp4_ds_mla(s["cache"], s["table"], s["cum"], s["rows"], block_size=s["page"], seq_starts=s["starts"])
    if s["op"] == "sparse" and s["page"]:
        return F.fp4_ds_mla_sparse_decode_paged(s["q"], s["cache"], s["req"], s["table"], s["idx"], SM_SCALE, block_size=s["page"], return_lse=True)
    if s["op"] == "sparse":
        return F.fp4_ds_mla_sparse_decode(s["q"], s["cache"], s["idx"], SM_SCALE, return_lse=True)
    return F.fp4_ds_mla_decode(s["q"], s["cache"], s["req"], s["table"], s["lens"], SM_SCALE, block_size=s["page"], return_lse=True)


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "write":
        kept = case["n"] * (1 - case["pad"])
        # latents, ropes and slots in, rows out; rows in, values out
        return {"bytes": kept * (1152 + ROW) + case["n"] * 8 + kept * ROW + case["n"] * 1152, "flops": kept * NOPE * 4}
    if op == "gather":
        rows = sum(_lens(case, case["B"]))
        return {"bytes": rows * (ROW + 1152) + rows * 4 / case["page"], "flops": rows * NOPE}
    T, H = case["T"], case["H"]
    fixed = T * H * (2 * (NOPE + ROPE) + 2 * NOPE + 4)
    if op == "sparse":
        entries = T * case["G"] * case["topk"]
        live = entries * (1 - case["mask"])
        return {"bytes": fixed + entries * 4 + live * ROW, "flops": 2 * live * (H // case["G"]) * (2 * NOPE + ROPE)}
    lens = _lens(case, T // case["next_n"])
    pairs = sum(max(0, n - b) for n in lens for b in range(case["next_n"]))
    return {"bytes": fixed + sum(lens) * ROW, "flops": 2 * pairs * H * (2 * NOPE + ROPE)}


# ---- the definitions in 64 bits -----------------------------------------------------------

def _nearest(x):
    """x (64 bits) [n, 512] as the value its 4-bit code and scale stand for."""
    g = x.view(-1, GROUP)
    big = g.abs().max(1).values / 6
    # e4m3: the nearest of its positive values, the even one of two as near
    e4m3 = torch.arange(1, 127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    up = torch.bucketize(big, e4m3).clamp(max=125)
    lo, hi = e4m3[(up - 1).clamp(min=0)], e4m3[up]
    # the code of entry i is i + 1: entry i is even where i is odd
    take_hi = (hi - big < big - lo) | ((hi - big == big - lo) & (up % 2 == 1)) | (up == 0)
    scale = torch.where(take_hi, hi, lo)[:, None]
    level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    far = (g.abs()[:, :, None] - level * scale[:, :, None]).abs()
    best = far.min(2, keepdim=True).values
    odd = torch.arange(8, device=x.device) % 2
    code = torch.where(far == best, odd, 2).argmin(2)
    return (level[code] * scale * torch.sign(g)).view(x.shape)


def _decoded(rows):
    """Packed rows as values in 64 bits."""
    b = rows[:, :256].long()
    code = torch.empty(len(rows), NOPE, dtype=torch.long, device=rows.device)
    code[:, 0::2], code[:, 1::2] = b % 16, b // 16
    m, e = (code % 2).double(), code // 2 % 4
    size = torch.where(e == 0, m / 2, (1 + m / 2) * 2.0 ** (e - 1).double())
    size = torch.where(code >= 8, -size, size)
    s = rows[:, 256:288].long()
    se, sm = s // 8 % 16, (s % 8).double() / 8
    scale = torch.where(se == 0, sm * 2.0 ** -6, (1 + sm) * 2.0 ** (se - 7).double())
    rope = rows[:, 288:].contiguous().view(torch.bfloat16).double()
    return torch.cat([size * scale.repeat_interleave(GROUP, 1), rope], 1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "write":
        out = torch.zeros(case["n"], NOPE + ROPE, dtype=torch.float64, device="cuda")
        for at in range(0, case["n"], 4096):
            part = slice(at, min(case["n"], at + 4096))
            out[part] = torch.cat([_nearest(s["kv_c"][part].double()), s["k_pe"][part].double()], 1)
        out[s["slots"] < 0] = 0
        return out
    if s["op"] == "gather":
        lens, out = _lens(case, case["B"]), []
        for b, n in enumerate(lens):
            pos = torch.arange(case["start"], case["start"] + n, device="cuda")
            out.append(_decoded(s["cache"].view(-1, case["page"], ROW)[s["table"][b].long()[pos // case["page"]], pos % case["page"]]))
        return torch.cat(out)
    T, H = case["T"], case["H"]
    G = case.get("G", 1)
    outs = torch.zeros(T, H, NOPE, dtype=torch.float64, device="cuda")
    lses = torch.full((T, H), float("-inf"), dtype=torch.float64, device="cuda")
    for t in range(T):
        for g in range(G):
            if s["op"] == "sparse":
                at = s["idx"][t, g].long()
                at = at[at >= 0]
            else:
                at = torch.arange(int(s["lens"][t]), device="cuda")
            if not len(at):
                continue
            if s["page"]:
                rows = s["cache"].view(-1, ROW)[:len(s["cache"]) // s["page"] * s["page"]].view(-1, s["page"], ROW)
                rows = rows[s["table"][int(s["req"][t])].long()[at // s["page"]], at % s["page"]]
            else:
                rows = s["cache"][at]
            k = _decoded(rows)
            part = slice(g * (H // G), (g + 1) * (H // G))
            z = s["q"][t, part].double() @ k.T * SM_SCALE
            lses[t, part] = torch.logsumexp(z, 1)
            outs[t, part] = torch.softmax(z, 1) @ k[:, :NOPE]
    return outs, lses
