"""The measured calls of the steps of a decoder layer between its quantized
products: residual addition and root-mean-square norm into an 8-bit
activation, K and V into a paged Q8_0 cache and back, and the attention of
new tokens over that cache.

Each case has a plain form (elementary torch operations in 32 bits), the
framework's own calls (`own`), and its value from the definition in 64 bits
(`exact`).

The cache is four planes, quantized per 32 values of a head as Q8_0 blocks
are (an f16 scale, 8-bit codes): K codes [pages, kv_heads, page, hd] with
scales [pages, kv_heads, page, hd / 32], V codes [pages, kv_heads, hd, page]
with scales [pages, kv_heads, hd / 32, page]. Position p of a sequence lies in
slot table[p // page] * page + p % page.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def listed():
    return [
        # one token's hidden state between two products of an 8B decode layer
        norm("norm_1x4096", 1, 4096, "f32", True, "q8k"),
        # a short batch, hidden size of the MXFP4 expert model, 16-bit stream
        norm("norm_77x2880_bf16", 77, 2880, "bf16", True, "q8_0"),
        # a prompt chunk of a 70B model
        norm("norm_2000x8192", 2000, 8192, "f32", True, "q8k"),
        # one new token of each of 8 sequences into the cache, and back
        write("write_8x8x128", 8, 8, 128, 64, "f32"),
        # a prompt's keys and values, straight from the fused q/k/v product's rows
        write("write_2000x8x128", 2000, 8, 128, 64, "f32"),
        # a prefix handed to code that wants plain values
        read("read_333x8x64", 333, 8, 64, 16, "f32"),
        # a long context read back
        read("read_32768x8x128", 32768, 8, 128, 64, "f16"),
        # the smallest decode step: one sequence of an 8B model
        attend("decode_1x500", 1, 1, 500, 32, 8, 128, 64, "f16"),
        # a decode batch of a 70B shard's heads, ragged long contexts
        attend("decode_16x8000", 16, 1, 8000, 64, 8, 128, 64, "bf16"),
        # three drafted tokens a sequence, small heads, window and sinks
        attend("draft_5x3x4000_w128", 5, 3, 4000, 64, 8, 64, 32, "bf16", window=128, sinks=True),
        # a prompt chunk of 512 over an 8B model's context
        attend("chunk_512x4096", 1, 512, 4096, 32, 8, 128, 64, "f16"),
        # two prompts' chunks of a 70B model
        attend("chunk_2x2000x7777", 2, 2000, 7777, 64, 8, 128, 64, "bf16"),
    ]


def norm(name, rows, k, dtype, residual, layout):
    return dict(name=name, op="norm", rows=rows, k=k, dtype=dtype, residual=residual, layout=layout)


def write(name, tokens, heads, hd, page, dtype):
    return dict(name=name, op="write", tokens=tokens, heads=heads, hd=hd, page=page, dtype=dtype)


def read(name, tokens, heads, hd, page, dtype):
    return dict(name=name, op="read", tokens=tokens, heads=heads, hd=hd, page=page, dtype=dtype)


def attend(name, seqs, new, context, heads, kv_heads, hd, page, dtype, window=0, sinks=False):
    """`new` and `context` are the longest sequence's; the others are shorter."""
    return dict(name=name, op="attend", seqs=seqs, new=new, context=context, heads=heads, kv_heads=kv_heads, hd=hd,
                page=page, dtype=dtype, window=window, sinks=sinks)


def spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "write", "read", "attend", "attend", "attend"])
    if op == "norm":
        layout = rng.choice(["q8k", "q8_0"])
        unit = 256 if layout == "q8k" else 32
        c = norm("", spread(rng, 1, 2000), unit * spread(rng, 256 // unit, 8192 // unit), rng.choice(list(DTYPES)),
                 rng.random() < 0.7, layout)
    elif op == "write":
        c = write("", spread(rng, 1, 2000), rng.choice([1, 2, 4, 8]), rng.choice([64, 96, 128, 256]),
                  rng.choice([16, 32, 64, 128]), rng.choice(list(DTYPES)))
    elif op == "read":
        c = read("", spread(rng, 16, 32768), rng.choice([1, 2, 4, 8]), rng.choice([64, 96, 128]),
                 rng.choice([16, 32, 64, 128]), rng.choice(list(DTYPES)))
    else:
        new = rng.choice([1, spread(rng, 2, 8), spread(rng, 9, 2000)])
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
        hd = rng.choice([64, 96, 128, 256] if kv_heads * group <= 32 else [64, 96, 128])
        context = new + spread(rng, 1, 6000)
        seqs = max(1, min(spread(rng, 1, 16), 4000 // new))
        c = attend("", seqs, new, context, kv_heads * group, kv_heads, hd, rng.choice([16, 32, 64, 128]),
                   rng.choice(["f16", "bf16"]), window=rng.choice([0, 0, 128, 1000]), sinks=rng.random() < 0.3)
    del c["name"]
    return c


def lengths(c):
    """New tokens and cached tokens (the new ones among them) of each sequence: the first has the most, the rest fall off."""
    n = c["seqs"]
    new = [max(1, c["new"] * (3 * n - 2 * b) // (3 * n)) for b in range(n)]
    return new, [max(new[b], c["context"] * (2 * n - b) // (2 * n)) for b in range(n)]


def outlying(g, rows, k, scale=20.0):
    """Values as a residual stream has them: normal, a few channels far larger."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    big = torch.randperm(k, generator=g, device="cuda")[: max(1, k // 500)]
    x[:, big] *= scale
    return x


def empty_planes(pages, heads, page, hd):
    return [torch.zeros(s, dtype=d, device="cuda") for s, d in (
        ((pages, heads, page, hd), torch.int8), ((pages, heads, page, hd // 32), torch.float16),
        ((pages, heads, hd, page), torch.int8), ((pages, heads, hd // 32, page), torch.float16))]


def filled_planes(g, pages, heads, page, hd):
    """Planes that hold keys and values of unit size: codes that reach 127 once in a block or so, scales to match."""
    planes = empty_planes(pages, heads, page, hd)
    for i in (0, 2):
        planes[i].copy_((torch.randn(planes[i].shape, generator=g, device="cuda") * 50).round().clamp(-127, 127))
        planes[i + 1].copy_(0.016 + 0.008 * torch.rand(planes[i + 1].shape, generator=g, device="cuda"))
    return planes


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "norm":
        t = DTYPES[case["dtype"]]
        s["x"] = outlying(g, case["rows"], case["k"]).to(t)
        s["r"] = torch.randn(case["rows"], case["k"], generator=g, device="cuda").to(t) if case["residual"] else None
        s["w"] = 1.0 + 0.2 * torch.randn(case["k"], generator=g, device="cuda")
        return s
    page, hd = case["page"], case["hd"]
    if case["op"] in ("write", "read"):
        n, heads = case["tokens"], case["heads"]
        pages = -(-n // page) + 3
        s["slots"] = (torch.randperm(pages, generator=g, device="cuda")[:, None] * page
                      + torch.arange(page, device="cuda")).reshape(-1)[:n].contiguous()
        if case["op"] == "write":
            # k and v are slices of the rows that one fused product wrote
            qkv = outlying(g, n, 6 * heads * hd, 5.0).to(DTYPES[case["dtype"]])
            s["k"] = qkv[:, 4 * heads * hd: 5 * heads * hd].view(n, heads, hd)
            s["v"] = qkv[:, 5 * heads * hd:].view(n, heads, hd)
            s["planes"] = empty_planes(pages, heads, page, hd)
        else:
            s["planes"] = filled_planes(g, pages, heads, page, hd)
        return s
    new, kv = lengths(case)
    per_seq = -(-case["context"] // page)
    pages = case["seqs"] * per_seq + 1
    s["planes"] = filled_planes(g, pages, case["kv_heads"], page, hd)
    s["tables"] = torch.randperm(pages, generator=g, device="cuda")[: case["seqs"] * per_seq].view(
        case["seqs"], per_seq).to(torch.int32)
    s["q_starts"] = torch.tensor([sum(new[:b]) for b in range(case["seqs"] + 1)], dtype=torch.int32, device="cuda")
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["q"] = (1.5 * torch.randn(sum(new), case["heads"], hd, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
    s["sinks"] = torch.randn(case["heads"], generator=g, device="cuda") if case["sinks"] else None
    s["scale"] = hd ** -0.5
    return s


def run(state):
    return {"norm": run_norm, "write": run_write, "read": run_read, "attend": run_attend}[state["op"]](state)


def run_norm(s):
    """The stream after the addition, and the values that the 8-bit activation stands for."""
    if own:
        from swarmllm_amd import GgmlDType, rms_norm_act

        out = rms_norm_act(s["x"], s["w"], EPS, residual=s["r"],
                           dtype=GgmlDType.Q4K if s["layout"] == "q8k" else GgmlDType.Q8_0)
        return [out.h, out.act.dequantize_f16()]
    h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    f = h.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * s["w"]
    if s["layout"] == "q8k":  # the value of largest magnitude (the first of several) is coded -127
        b = y.view(s["rows"], -1, 256)
        mag = b.abs()
        top = mag.amax(-1, keepdim=True)
        at = torch.where(mag == top, torch.arange(256, device=y.device), 256).amin(-1, keepdim=True)
        inv = -127.0 / b.gather(-1, at)
        codes = half_away(b * inv).clamp(max=127)
        v = codes / inv
    else:
        b = y.view(s["rows"], -1, 32)
        d = b.abs().amax(-1, keepdim=True) / 127.0
        v = half_away(b * (1.0 / d)) * d.half().float()
    return [h, v.view(s["rows"], -1).half()]


def half_away(t):
    """To the nearest whole number, halves away from zero."""
    whole = t.trunc()
    return whole + ((t - whole).abs() >= 0.5) * t.sign()


def q8_0(x):
    """Codes and scales of [..., hd] values per 32 of the last axis."""
    b = x.float().view(*x.shape[:-1], -1, 32)
    d = b.abs().amax(-1, keepdim=True) / 127.0
    codes = half_away(b * torch.where(d == 0, 0.0, 1.0 / d)).clamp(-127, 127)
    return codes.to(torch.int8).view(x.shape), d.squeeze(-1).half()


def run_write(s):
    """Keys and values quantized into the cache, and what the cache then holds of them."""
    if own:
        from swarmllm_amd import KvCache

        kv = KvCache(*s["planes"])
        kv.write(s["k"], s["v"], s["slots"])
        return list(kv.read(s["slots"], torch.float16))
    kc, ks, vc, vs = s["planes"]
    p, o = s["slots"] // s["page"], s["slots"] % s["page"]
    kc[p, :, o], ks[p, :, o] = q8_0(s["k"])
    vc[p, :, :, o], vs[p, :, :, o] = q8_0(s["v"])
    return plain_read(s, torch.float16)


def plain_read(s, dtype):
    kc, ks, vc, vs = s["planes"]
    p, o = s["slots"] // s["page"], s["slots"] % s["page"]
    return [(c.float().view(*c.shape[:-1], -1, 32) * d.float()[..., None]).view(c.shape).to(dtype)
            for c, d in ((kc[p, :, o], ks[p, :, o]), (vc[p, :, :, o], vs[p, :, :, o]))]


def run_read(s):
    if own:
        from swarmllm_amd import KvCache

        return list(KvCache(*s["planes"]).read(s["slots"], DTYPES[s["dtype"]]))
    return plain_read(s, DTYPES[s["dtype"]])


def run_attend(s):
    if own:
        from swarmllm_amd import KvCache

        return KvCache(*s["planes"]).attend(s["q"], s["q_starts"], s["kv_lens"], s["tables"], max_q=s["new"],
                                            max_kv=s["context"], scale=s["scale"], window=s["window"],
                                            sinks=s["sinks"])
    kc, ks, vc, vs = s["planes"]
    b, h, hk, hd = s["seqs"], s["heads"], s["kv_heads"], s["hd"]
    group, t = h // hk, s["new"]
    pages = s["tables"].long()
    k = kc[pages].float().view(*kc[pages].shape[:-1], -1, 32) * ks[pages].float()[..., None]
    k = k.view(b, -1, hk, s["page"], hd).transpose(1, 2).reshape(b, hk, -1, hd)
    v = vc[pages].float().view(b, -1, hk, hd // 32, 32, s["page"]) * vs[pages].float()[..., None, :]
    v = v.view(b, -1, hk, hd, s["page"]).permute(0, 2, 1, 4, 3).reshape(b, hk, -1, hd)
    # the new tokens of each sequence side by side, behind the shorter ones whatever comes next
    start, count = s["q_starts"][:-1, None].long(), s["q_starts"].diff()[:, None].long()
    i = torch.arange(t, device=k.device)
    q = s["q"][(start + i).clamp(max=s["q"].shape[0] - 1)].float().view(b, t, hk, group, hd).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(b, hk, group * t, hd), k.transpose(2, 3).contiguous()).view(b, hk, group, t, -1)
    score = score * s["scale"]
    pos = (s["kv_lens"][:, None] - count + i)[:, :, None]
    j = torch.arange(k.shape[2], device=k.device)
    seen = (j <= pos) & (j > pos - s["window"]) if s["window"] else j <= pos
    score = torch.where(seen[:, None, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(hk, group, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    o = torch.matmul(p.view(b, hk, group * t, -1), v).view(b, hk, group, t, hd) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(b, t, h, hd)
    n = torch.arange(s["q"].shape[0], device=k.device)
    of = torch.searchsorted(s["q_starts"][1:].long(), n, right=True)
    return o[of, n - start[of, 0]].to(s["q"].dtype)


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["k"]
        # in: x, the residual, the weight; out: the stream where it was added to, and the activation's 8-bit values
        streams = 3 if case["residual"] else 1
        scales = n // 256 * 4 if case["layout"] == "q8k" else n // 32 * 4
        return {"bytes": streams * n * SIZES[case["dtype"]] + 4 * case["k"] + n + scales, "flops": 7 * n}
    if case["op"] in ("write", "read"):
        n = 2 * case["tokens"] * case["heads"] * case["hd"]
        held = n + n // 16
        if case["op"] == "read":
            return {"bytes": held + SIZES[case["dtype"]] * n + 8 * case["tokens"], "flops": n}
        return {"bytes": n * SIZES[case["dtype"]] + held + 2 * n + 8 * case["tokens"], "flops": 4 * n}
    new, kv = lengths(case)
    hd, w = case["hd"], case["window"]
    pairs = tokens = 0
    for t, n in zip(new, kv):
        for i in range(t):
            pairs += min(n - t + i + 1, w) if w else n - t + i + 1
        tokens += min(n, w + t - 1) if w else n
    io = 2 * sum(new) * case["heads"] * hd * SIZES[case["dtype"]]
    return {"bytes": io + 2 * tokens * case["kv_heads"] * (hd + hd // 16), "flops": 4 * pairs * case["heads"] * hd}


def exact(case, seed):
    """The same outputs in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = (h + s["r"].double()).to(s["x"].dtype).double()
        y = h / ((h ** 2).sum(1, keepdim=True) / case["k"] + EPS).sqrt() * s["w"].double()
        size = 256 if case["layout"] == "q8k" else 32
        blocks = y.split(size, dim=1)
        out = []
        for b in blocks:
            if size == 256:
                d = b.gather(1, b.abs().argmax(1, keepdim=True)) / -127.0
                out.append((b / d).round().clamp(-128, 127) * d)
            else:
                d = b.abs().max(1, keepdim=True).values / 127.0
                out.append((b / d).round() * d.half().double())
        return [h, torch.cat(out, 1)]
    page = case["page"]
    if case["op"] in ("write", "read"):
        out = []
        for i, name in enumerate(("k", "v")):
            if case["op"] == "write":
                x = s[name].double().reshape(-1, 32)
                d = x.abs().max(1, keepdim=True).values / 127.0
                out.append(((x / d).round() * d.half().double()).view(s[name].shape))
            else:
                out.append(values64(s["planes"], i)[s["slots"]])
        return out
    new, kv = lengths(case)
    k, v = (values64(s["planes"], i) for i in (0, 1))
    group = case["heads"] // case["kv_heads"]
    outs, at = [], 0
    for b in range(case["seqs"]):
        j = torch.arange(kv[b], device="cuda")
        slots = s["tables"][b].long()[j // page] * page + j % page
        q = s["q"][at:at + new[b]].double()
        pos = torch.arange(kv[b] - new[b], kv[b], device="cuda")[:, None]
        hidden = j > pos
        if case["window"]:
            hidden = hidden | (j <= pos - case["window"])
        heads = []
        for h in range(case["heads"]):
            x = q[:, h] @ k[slots, h // group].T * s["scale"]
            x = x.masked_fill(hidden, float("-inf"))
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double().expand(new[b], 1)], 1)
            heads.append(torch.softmax(x, 1)[:, :kv[b]] @ v[slots, h // group])
        outs.append(torch.stack(heads, 1))
        at += new[b]
    return torch.cat(outs)


def values64(planes, i):
    """Every slot's keys (i = 0) or values (1) [slots, heads, hd] in 64 bits."""
    c, d = planes[2 * i].double(), planes[2 * i + 1].double()
    if i:
        c, d = c.transpose(2, 3), d.transpose(2, 3)
    c = c.reshape(*c.shape[:-1], -1, 32) * d[..., None]
    return c.flatten(-2).transpose(1, 2).flatten(0, 1)
