"""The measured calls of what a batch of many requests needs around the
quantized products: its page tables and rows (PageTables.step), its low-rank
adapters beside a shared projection (Adapters.add, add_shared), and its next
tokens from the output head's logits (sample).

Each case has a plain form (elementary torch operations, in 32 bits, sums and
weights next to a border in 64), the framework's own calls (`own`), and its
value from the definition in 64 bits (`exact`).

A step of the page tables, for sequences b = 0, 1, ... in order: the length
len[b] is cut to keep[b] and the pages past it return to the stack of free
pages; the sequence then takes pages for new[b] tokens off the stack's end. The
pages returned by one step are the first that it takes, in the order of
sequences and pages. Rows of the batch are numbered sequence after sequence. A
sequence past the pages left, its table or the batch's rows is not extended;
its rows have slot and position -1.

Sampling: weights w = exp((x - max x) / temperature); of the values ordered by
x (equal ones by index) the first top_k stay, of those the shortest run whose
weight reaches top_p of theirs, of those the ones of weight min_p at least. The
token is the first, by index, whose running sum passes u times the total.

An adapter: y[r] + scale[i] * (x[r] A[i]^T) B[i]^T with i the row's adapter.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
GREEDY, NO_K = 0.0, 0


def listed():
    return [
        # eight chats decoded together, one token each
        step("step_8x1", 8, 1, 4096, 64, 0, "steady"),
        # five drafted tokens a sequence, some of the last five cut
        step("step_64x5_drafts", 64, 5, 8000, 64, 5, "steady"),
        # a batch refilled: finished requests leave their pages to prompts, beside the ones that go on
        step("step_48_prompts", 48, 2000, 4096, 32, 1, "refill"),
        # a full pool: many short requests, the last ones find no pages
        step("step_700_full", 700, 400, 300, 16, 3, "full"),
        # a chat's next token, 128K vocabulary
        sample("sample_1x128256", 1, 128256, "f32", "chat"),
        # a batch with each request's own settings, an odd vocabulary size, bf16 logits
        sample("sample_21x50257_bf16", 21, 50257, "bf16", "mixed"),
        # a decode batch, each request its own settings
        sample("sample_64x128256", 64, 128256, "f32", "mixed"),
        # rollouts drawn from the whole distribution
        sample("sample_512x128256", 512, 128256, "f32", "whole"),
        # one request's adapter at the attention output of an 8B model
        lora("lora_o_1row", 1, 4096, "4096", 16, 4, "f32", "bf16"),
        # a decode batch, each row its own adapter, beside the q, k and v products
        lora("lora_qkv_21rows", 21, 4096, "4096,1024,1024", 16, 24, "f32", "bf16"),
        # a prompt chunk of four requests beside gate and up, the norm's values in bf16
        lora("lora_gate_up_512rows", 512, 4096, "14336,14336", 32, 4, "bf16", "bf16"),
        # long prompts beside the down product of a 70B model
        lora("lora_down_2000rows", 2000, 28672, "8192", 64, 3, "f32", "f16"),
    ]


def step(name, seqs, new, context, page, cut, kind):
    """`new`, `context` and `cut` are the most of a sequence; a refill's prompts begin at no context."""
    return dict(name=name, op="step", seqs=seqs, new=new, context=context, page=page, cut=cut, kind=kind)


def sample(name, rows, vocab, dtype, settings):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, dtype=dtype, settings=settings)


def lora(name, rows, k, ns, rank, slots, x, w):
    """Adapters beside the products of one activation with output widths `ns`."""
    return dict(name=name, op="lora", rows=rows, k=k, ns=ns, rank=rank, slots=slots, x=x, w=w)


def spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["step", "sample", "sample", "lora", "lora"])
    if op == "step":
        seqs = spread(rng, 1, 1000)
        c = step("", seqs, spread(rng, 1, max(2, min(2000, 80000 // seqs))), spread(rng, 100, 8000),
                 rng.choice([16, 32, 64, 128]), rng.choice([0, 1, 5]), rng.choice(["steady", "refill", "full"]))
    elif op == "sample":
        vocab = spread(rng, 1000, 200000)
        c = sample("", spread(rng, 1, min(512, 60000000 // vocab)), vocab, rng.choice(list(DTYPES)),
                   rng.choice(["chat", "mixed", "mixed", "whole"]))
    else:
        k = 32 * spread(rng, 16, 512)
        ns = [spread(rng, 128, 16384) for _ in range(rng.choice([1, 1, 2, 3]))]
        rank = rng.choice([8, 16, 16, 24, 32, 64])
        c = lora("", spread(rng, 1, min(2000, 50000000 // (k + sum(ns)))), k, ",".join(map(str, ns)), rank,
                 spread(rng, 1, max(1, min(32, 30000000 // (rank * (k + sum(ns)))))), rng.choice(["f32", "f32", "bf16", "f16"]), rng.choice(["bf16", "f16", "f32"]))
    del c["name"]
    return c


def lengths(c):
    """Of each sequence: tokens held, kept and new."""
    n, held, keep, new = c["seqs"], [], [], []
    for b in range(n):
        context = max(c["cut"], c["context"] * (2 * n - b) // (2 * n) - 37 * b % max(1, c["context"] // 2))
        fresh = c["kind"] == "refill" and b % 3 == 0 or c["kind"] == "full" and b % 2 == 0
        cut = c["cut"] - b % 3 if c["cut"] > 2 else c["cut"]
        held.append(context)
        keep.append(0 if fresh else max(0, context - cut))
        more = max(1, c["new"] * (3 * n - 2 * b) // (3 * n))
        new.append(more if fresh or c["kind"] == "steady" else 1 if c["kind"] == "refill" else b % 4)
    return held, keep, new


def sizes(c):
    """Of a step's case: table rows, pages of the pool and rows of the batch."""
    held, keep, new = lengths(c)
    page = c["page"]
    row = max(-(-max(h, k + t) // page) for h, k, t in zip(held, keep, new)) + 1
    after = sum(-(-(k + t) // page) for k, t in zip(keep, new))
    before = sum(-(-h // page) for h in held)
    pool = max(before, after + 7 if c["kind"] != "full" else 9 * after // 10)
    return row, pool, sum(new)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "step":
        held, keep, new = lengths(case)
        row, pool, s["tokens"] = sizes(case)
        order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        lens = torch.tensor(held, device="cuda")
        count = (lens + case["page"] - 1) // case["page"]
        j = torch.arange(row, device="cuda")
        first = (count.cumsum(0) - count)[:, None]
        used = int(count.sum())
        s["tables"] = torch.where(j < count[:, None], order[(first + j).clamp(max=pool - 1)], -1).to(torch.int32)
        s["lens"] = lens.to(torch.int32)
        s["free"] = torch.full((pool,), -1, dtype=torch.int32, device="cuda")
        s["free"][:pool - used] = order[used:]
        s["free_count"] = torch.full((1,), pool - used, dtype=torch.int32, device="cuda")
        s["keep"] = torch.tensor(keep, dtype=torch.int32, device="cuda")
        s["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        if own:
            from swarmllm_amd import PageTables

            s["pages"] = PageTables(s["tables"], s["lens"], s["free"], s["free_count"], case["page"])
        return s
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # most of a vocabulary well below a few dozen candidates, as a language model's head gives it
        x = 2.2 * torch.randn(rows, vocab, generator=g, device="cuda")
        few = torch.randint(vocab, (rows, 50), generator=g, device="cuda")
        x.scatter_add_(1, few, 7.0 + 3.0 * torch.randn(rows, 50, generator=g, device="cuda"))
        r = torch.arange(rows, device="cuda")
        if case["settings"] == "mixed":  # every seventh request is held to a grammar: most tokens masked
            masked = (r % 7 == 3)[:, None] & (torch.rand(rows, vocab, generator=g, device="cuda") < 0.99)
            x.masked_fill_(masked, float("-inf"))
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        jitter = torch.rand(rows, generator=g, device="cuda")
        s["temperature"] = s["top_k"] = s["top_p"] = s["min_p"] = None
        if case["settings"] == "chat":
            s["temperature"] = 0.6 + 0.2 * jitter
            s["top_k"] = torch.full((rows,), 40, dtype=torch.int32, device="cuda")
            s["top_p"] = torch.full((rows,), 0.95, device="cuda")
        elif case["settings"] == "mixed":
            s["temperature"] = torch.where(r % 5 == 0, GREEDY, 0.5 + jitter)
            s["top_k"] = torch.where(r % 3 == 1, 20 + 100 * (r % 4), NO_K).to(torch.int32)
            s["top_p"] = torch.where(r % 4 < 2, 0.8 + 0.19 * jitter, 1.0)
            s["min_p"] = torch.where(r % 6 == 5, 0.05, 0.0)
        return s
    rows, k, rank, slots, t = case["rows"], case["k"], case["rank"], case["slots"], DTYPES[case["w"]]
    ns = widths(case)
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 500)]] *= 20.0
    s["x"] = x.to(DTYPES[case["x"]])
    s["y"] = [torch.randn(rows, n, generator=g, device="cuda") for n in ns]
    s["out"] = [torch.empty_like(y) for y in s["y"]]
    s["a"] = [(torch.randn(slots, rank, k, generator=g, device="cuda") / k ** 0.5).to(t) for _ in ns]
    s["b"] = [(0.05 * torch.randn(slots, n, rank, generator=g, device="cuda")).to(t) for n in ns]
    s["scales"] = [1.0 + torch.rand(slots, generator=g, device="cuda") for _ in ns]
    # a decode batch has a request a row, a prompt's rows lie together; every ninth request has no adapter
    request = torch.arange(rows, device="cuda") // max(1, rows // 60)
    of = torch.randint(slots, (rows,), generator=g, device="cuda")
    s["ids"] = torch.where(request % 9 == 8, -1, of[request]).to(torch.int32)
    if own:
        from swarmllm_amd import Adapters

        s["adapters"] = [Adapters(*abs) for abs in zip(s["a"], s["b"], s["scales"])]
    return s


def widths(c):
    return [int(n) for n in c["ns"].split(",")]


def run(state):
    return {"step": run_step, "sample": run_sample, "lora": run_lora}[state["op"]](state)


def run_step(s):
    """The batch's rows, and the tables, lengths and free pages afterwards. (A pass cuts what the one before it added:
    every pass does the same.)"""
    if own:
        rows = s["pages"].step(s["new"], s["tokens"], keep=s["keep"])
        return [rows.q_starts, rows.taken, rows.slots, rows.positions, rows.seq, s["tables"], s["lens"], s["free_count"]]
    page, tables, lens, free, count = s["page"], s["tables"], s["lens"], s["free"], s["free_count"]
    seqs, row = tables.shape
    tokens, device = s["tokens"], tables.device
    keep, new = torch.minimum(s["keep"], lens).long(), s["new"].long()
    held, kept = (lens.long() + page - 1) // page, (keep + page - 1) // page
    j = torch.arange(row, device=device)
    # the pages past what is kept, in order, on top of the stack: the first of them its end
    cut = (j >= kept[:, None]) & (j < held[:, None])
    n = cut.sum()
    at = torch.where(cut, count + n - cut.flatten().cumsum(0).view(seqs, row), free.numel())
    free = torch.cat([free, free.new_zeros(1)]).scatter_(0, at.flatten(), tables.flatten())
    total = count + n
    end = new.cumsum(0)
    fits = (end <= tokens) & (keep + new <= row * page)
    need = torch.where(fits, (keep + new + page - 1) // page - kept, 0)
    last = need.cumsum(0)
    taken = fits & ((need == 0) | (last <= total))
    take = (j >= kept[:, None]) & (j < (kept + need)[:, None]) & taken[:, None]
    which = (total - 1 - (last - need)[:, None] - (j - kept[:, None])).clamp(0, free.numel() - 1)
    after = torch.where(take, free[which], torch.where(j < kept[:, None], tables, -1))
    popped = torch.where(last <= total, last, 0).amax()
    q_starts = torch.cat([end.new_zeros(1), end]).clamp(max=tokens)
    t = torch.arange(tokens, device=device)
    seq = torch.searchsorted(q_starts[1:], t, right=True)
    seq = torch.where(t < q_starts[-1], seq, -1)
    of = seq.clamp(min=0)
    pos = keep[of] + t - q_starts[of]
    there = (seq >= 0) & taken[of]
    slots = torch.where(there, after[of, (pos // page).clamp(max=row - 1)].long() * page + pos % page, -1)
    s["tables"].copy_(after)
    s["lens"].copy_(keep + torch.where(taken, new, 0))
    s["free"].copy_(free[:-1])
    s["free_count"].copy_(total - popped)
    return [q_starts.int(), torch.where(taken, new, 0).int(), slots, torch.where(there, pos, -1).int(), seq.int(),
            s["tables"], s["lens"], s["free_count"]]


def run_sample(s):
    """Each row's token, and the chance that it was drawn with."""
    if own:
        import swarmllm_amd as sa

        out = sa.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                        min_p=s["min_p"])
        return [out.ids, out.probs]
    x = s["logits"].float()
    rows, vocab = x.shape
    top = x.amax(1, keepdim=True)
    t = s["temperature"][:, None].double() if s["temperature"] is not None else 1.0
    greedy = t == GREEDY if s["temperature"] is not None else torch.zeros(rows, 1, dtype=torch.bool, device=x.device)
    w = torch.exp((x.double() - top) / torch.where(greedy, 1.0, t) if s["temperature"] is not None else x.double() - top)
    if s["top_k"] is not None or s["top_p"] is not None:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        if s["top_k"] is not None:
            k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
            ws = torch.where(torch.arange(vocab, device=x.device) < k, ws, 0.0)
        if s["top_p"] is not None:
            p = s["top_p"][:, None].double()
            sums = ws.cumsum(1)
            ws = torch.where((sums - ws < p * sums[:, -1:]) | (p >= 1.0), ws, 0.0)
        w = torch.zeros_like(w).scatter_(1, order, ws)
    if s["min_p"] is not None:
        w = torch.where(w >= s["min_p"][:, None].double(), w, 0.0)
    sums = w.cumsum(1)
    total = sums[:, -1:]
    ids = torch.searchsorted(sums, s["u"][:, None].double() * total, right=True).clamp(max=vocab - 1)
    i = torch.arange(vocab, device=x.device)
    first = torch.where(x == top, i, vocab).amin(1, keepdim=True)
    ids = torch.where(greedy, first, ids)
    return [ids[:, 0].int(), torch.where(greedy, 1.0, w.gather(1, ids) / total)[:, 0].float()]


def run_lora(s):
    """The products with the adapters' parts added."""
    if own:
        if len(s["y"]) == 1:
            return s["adapters"][0].add(s["y"][0], s["x"], s["ids"], out=s["out"][0])
        return type(s["adapters"][0]).add_shared(s["y"], s["x"], s["adapters"], s["ids"], outs=s["out"])
    x, outs = s["x"].float(), []
    # every adapter's part of every row, those that are not the row's own left out
    mine = s["ids"][:, None] == torch.arange(s["slots"], device=x.device)
    for y, a, b, scales in zip(s["y"], s["a"], s["b"], s["scales"]):
        t = (x @ a.float().flatten(0, 1).T).view(s["rows"], s["slots"], s["rank"])
        t = torch.where(mine[..., None], t * scales[:, None], 0.0)
        outs.append(y + t.flatten(1) @ b.float().transpose(1, 2).reshape(s["slots"] * s["rank"], -1))
    return outs if len(outs) > 1 else outs[0]


def work(case):
    if case["op"] == "step":
        held, keep, new = lengths(case)
        row, pool, tokens = sizes(case)
        page = case["page"]
        moved = sum(abs(-(-h // page) - -(-k // page)) + abs(-(-(k + t) // page) - -(-k // page))
                    for h, k, t in zip(held, keep, new))
        # lengths, counts and starts of the sequences, pages that change hands, rows of the batch
        return {"bytes": 24 * case["seqs"] + 8 * moved + 16 * tokens, "flops": 4 * tokens}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZES[case["dtype"]] + 28 * case["rows"], "flops": 4 * n}
    rows, k, rank, ns = case["rows"], case["k"], case["rank"], widths(case)
    used = min(case["slots"], rows)
    b = rows * k * SIZES[case["x"]] + 4 * rows
    for n in ns:
        b += 8 * rows * n + used * rank * (k + n) * SIZES[case["w"]]
    return {"bytes": b, "flops": sum(2 * rows * rank * (k + n) for n in ns)}


def exact(case, seed):
    """The same outputs from the definitions: whole numbers counted one by one, the others in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "step":
        return exact_step(s)
    if case["op"] == "sample":
        return exact_sample(s)
    outs = []
    for y, a, b, scales in zip(s["y"], s["a"], s["b"], s["scales"]):
        out = y.double()
        for i in range(case["slots"]):
            rows = torch.nonzero(s["ids"] == i)[:, 0]
            part = torch.mm(torch.mm(s["x"][rows].double(), a[i].double().t()), b[i].double().t())
            out[rows] += scales[i].double() * part
        outs.append(out)
    return outs if len(outs) > 1 else outs[0]


def exact_step(s):
    page, tokens = s["page"], s["tokens"]
    tables, lens, keep, new = (s[n].tolist() for n in ("tables", "lens", "keep", "new"))
    row, stack = len(tables[0]), s["free"].tolist()[:int(s["free_count"])]
    back = []
    for b, table in enumerate(tables):
        lens[b], held = min(lens[b], keep[b]), -(-lens[b] // page)
        for j in range(-(-lens[b] // page), held):
            back.append(table[j])
            table[j] = -1
    stack += back[::-1]
    starts, taken, slots, positions, seq = [0], [], [], [], []
    short = False
    for b, table in enumerate(tables):
        n = new[b]
        fits = starts[-1] + n <= tokens and lens[b] + n <= row * page
        have, want = -(-lens[b] // page), -(-(lens[b] + n) // page) if fits else 0
        if fits and want > have:
            short = short or want - have > len(stack)
            fits = not short
        if fits:
            for j in range(have, want):
                table[j] = stack.pop()
        for p in range(lens[b], lens[b] + n):
            if len(slots) < tokens:
                slots.append(table[p // page] * page + p % page if fits else -1)
                positions.append(p if fits else -1)
                seq.append(b)
        starts.append(len(slots))
        taken.append(n if fits else 0)
        lens[b] += taken[-1]
    for out in (slots, positions, seq):
        out += [-1] * (tokens - len(out))
    out = [starts, taken, slots, positions, seq, tables, lens, [len(stack)]]
    return [torch.tensor(v, dtype=torch.int64 if i == 2 else torch.int32, device="cuda") for i, v in enumerate(out)]


def exact_sample(s):
    ids, probs = [], []
    of = {n: s[n].tolist() if s[n] is not None else [off] * s["rows"]
          for n, off in (("temperature", 1.0), ("top_k", NO_K), ("top_p", 1.0), ("min_p", 0.0))}
    for r, u in enumerate(s["u"].tolist()):
        x = s["logits"][r].double()
        if of["temperature"][r] == GREEDY:
            ids.append(torch.argmax((x == x.max()).int()))
            probs.append(x.new_ones(()))
            continue
        w = torch.softmax(x / of["temperature"][r], 0)
        k = of["top_k"][r] or len(x)
        values, order = torch.sort(-x, stable=True)
        chosen = order[:k]
        chosen = chosen[w[chosen] > 0]
        if of["top_p"][r] < 1.0:
            goal = of["top_p"][r] * w[chosen].sum()
            chosen = chosen[:int((w[chosen].cumsum(0) < goal).sum()) + 1]
        chosen = chosen[w[chosen] >= of["min_p"][r] * w.max()].sort().values
        sums = w[chosen].cumsum(0)
        i = chosen[(sums <= u * sums[-1]).sum().clamp(max=len(chosen) - 1)]
        ids.append(i)
        probs.append(w[i] / sums[-1])
    return [torch.stack(ids).int(), torch.stack(probs)]
