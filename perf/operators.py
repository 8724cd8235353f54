"""Operators over a paged K/V cache that many requests share, as measurable cases.

A serving step takes a batch of requests, each with tokens in the cache and some new ones: pages and slots are
found for the new tokens (`page_slots`), their keys and values are rotated and stored (`rope_append`), and their
queries attend to everything that their request has in the cache (`paged_attention`). `run` makes the calls that a
user makes where `own` is true; otherwise it computes the same with elementary torch operations. `exact` restates
the operators in 64 bits.
"""
import itertools
import math
import random

import torch

own = False
DEV = "cuda"
TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F64 = torch.float64


# ------------------------------------------------------------------ the cases
def listed():
    flagship = dict(heads=24, kv_heads=4, dim=256)  # the benchmark's hybrid model
    return [
        # one token for each of a few sessions: what every decode step of a small server begins with
        dict(name="slots-decode", kind="slots", requests=8, chunks=0, chunk=1, context=3000, page=16, pad=0, shape=1),
        # a large server's step: most requests decode, some bring a piece of their prompt; room for a fixed number of tokens
        dict(name="slots-batch", kind="slots", requests=256, chunks=60, chunk=700, context=20000, page=16, pad=500, shape=2),
        # one decode step of sixteen sessions, projections in 32 bits, a quarter of each head rotated
        dict(name="append-decode", kind="append", tokens=16, **flagship, rot=64, axes=1, pairing="half", source="f32", cache="bf16", norm=True, page=16),
        # a portion of a prompt, 16-bit projections, whole heads rotated
        dict(name="append-prompt", kind="append", tokens=4099, heads=16, kv_heads=4, dim=128, rot=128, axes=1, pairing="half", source="bf16",
             cache="bf16", norm=False, page=128),
        # the patches of some images or of a video among text: time, height and width
        dict(name="append-image", kind="append", tokens=2475, heads=24, kv_heads=4, dim=256, rot=64, axes=3, pairing="half", source="bf16",
             cache="bf16", norm=True, page=16),
        # one token of one short session: latency
        dict(name="attention-small", kind="attention", requests=1, chunks=0, chunk=1, context=45, heads=8, kv_heads=2, dim=128, cache="bf16",
             page=16, window=0, sinks=False, shape=3),
        # one decode step of 48 sessions of very different lengths
        dict(name="attention-decode", kind="attention", requests=48, chunks=0, chunk=1, context=12000, **flagship, cache="bf16", page=16,
             window=0, sinks=False, shape=4),
        # a verify pass of one long session: three drafts and the current token
        dict(name="attention-verify", kind="attention", requests=1, chunks=1, chunk=4, context=32768, **flagship, cache="bf16", page=16,
             window=0, sinks=False, shape=5),
        # the next portion of a long prompt
        dict(name="attention-chunk", kind="attention", requests=1, chunks=1, chunk=2000, context=14000, **flagship, cache="bf16", page=16,
             window=0, sinks=False, shape=6),
        # several whole prompts, sliding windows and sinks
        dict(name="attention-prompts", kind="attention", requests=3, chunks=3, chunk=4000, context=0, heads=16, kv_heads=4, dim=128,
             cache="bf16", page=128, window=1024, sinks=True, shape=7),
        # decode steps and pieces of prompts in one batch
        dict(name="attention-mixed", kind="attention", requests=26, chunks=2, chunk=700, context=6000, heads=32, kv_heads=8, dim=128,
             cache="f16", page=64, window=0, sinks=False, shape=8),
        # a whole step: pages and slots, then in each of four layers append and attention
        dict(name="step", kind="step", requests=12, chunks=2, chunk=200, context=5000, **flagship, rot=64, axes=1, pairing="half", source="f32",
             cache="bf16", norm=True, page=16, pad=0, window=0, sinks=False, layers=4, shape=9),
    ]


def log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["slots", "append", "append", "attention", "attention", "attention", "attention", "step"])
    c = dict(kind=kind, shape=rng.randrange(1 << 30))
    if kind == "slots":
        n = log_int(rng, 1, 700)
        return dict(c, requests=n, chunks=rng.choice([0, n // 4, n]), chunk=log_int(rng, 2, 1200 if n < 100 else 150),
                    context=log_int(rng, 1, 30000), page=rng.choice([16, 16, 32, 48, 64, 128]), pad=rng.choice([0, 0, 37]))
    heads, kv_heads = rng.choice([(8, 2), (24, 4), (16, 4), (16, 16), (32, 8), (5, 1), (14, 2), (32, 2)])
    dim = rng.choice([64, 128, 128, 256])
    c.update(heads=heads, kv_heads=kv_heads, dim=dim, cache=rng.choice(["bf16", "bf16", "f16"]), page=rng.choice([16, 16, 32, 48, 64, 128]))
    if kind in ("append", "step"):
        c.update(rot=rng.choice([dim, dim // 2, dim // 4]), axes=rng.choice([1, 1, 2, 3]) if kind == "append" else 1,
                 pairing=rng.choice(["half", "half", "adjacent"]), source=rng.choice(["f32", "bf16", "f16"]), norm=rng.random() < 0.6)
    if kind == "append":
        return dict(c, tokens=log_int(rng, 1, 4500))
    c.update(window=rng.choice([0, 0, 0, 100, 1024]), sinks=rng.random() < 0.3)
    if kind == "step":
        n = log_int(rng, 1, 24)
        return dict(c, requests=n, chunks=rng.choice([0, n // 4, min(n, 3)]), chunk=log_int(rng, 2, 300), context=log_int(rng, 1, 6000),
                    pad=rng.choice([0, 0, 19]), layers=rng.randint(1, 4))
    form = rng.choice(["decode", "decode", "verify", "prompt", "portion", "mixed"])
    most = 48 * 12000 * 4 * 256 // (kv_heads * dim)  # tokens in the cache: no more bytes than the largest listed case has
    if form == "decode":
        n = log_int(rng, 1, 64)
        return dict(c, requests=n, chunks=0, chunk=1, context=log_int(rng, 1, min(100000 if n < 4 else 8000, most // n)))
    if form == "verify":
        n = log_int(rng, 1, 16)
        return dict(c, requests=n, chunks=n, chunk=rng.randint(2, 16), context=log_int(rng, 20, min(60000 if n < 4 else 8000, most // n)))
    if form == "prompt":
        return dict(c, requests=rng.randint(1, 4), chunks=4, chunk=log_int(rng, 17, 3000), context=0)
    if form == "portion":
        return dict(c, requests=1, chunks=1, chunk=log_int(rng, 17, 1500), context=log_int(rng, 100, 12000))
    n = rng.randint(4, 32)
    return dict(c, requests=n, chunks=rng.randint(1, 3), chunk=log_int(rng, 20, 700), context=log_int(rng, 100, 5000))


def batch(c):
    """[(tokens in the cache before, new tokens)] of every request. The longest context and chunk are there as named."""
    rng = random.Random(c["shape"])
    n, chunks = c["requests"], min(c["chunks"], c["requests"])
    rest = 0 if c["context"] == 0 else 1
    lens = [(log_int(rng, max(1, c["context"] // 20), c["context"]) if rest else 0, log_int(rng, max(1, c["chunk"] // 4), c["chunk"]) if i < chunks else 1)
            for i in range(n)]
    lens[0] = (c["context"], c["chunk"] if chunks else 1)
    rng.shuffle(lens)
    return lens


def pages_of(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------ inputs, made on the GPU from the seed alone
class Rng:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(1000003 * seed + 17)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEV, generator=self.g) * std + mean).to(dtype)

    def permutation(self, n):
        return torch.randperm(n, device=DEV, generator=self.g).to(torch.int32)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def paged_inputs(c, r, lens):
    """The page manager's state: which pages the requests hold, and the stack of free ones (its top is taken first)."""
    n, page = len(lens), c["page"]
    held = [pages_of(a, page) for a, _ in lens]
    wanted = [pages_of(a + b, page) for a, b in lens]
    n_pages = sum(wanted) + 7
    pages = r.permutation(n_pages)
    rows = r.permutation(n + 3)[:n].contiguous()  # a server's rows outlive single requests: they come in any order
    table = torch.full((n + 3, max(wanted) + 2), -1, dtype=torch.int32, device=DEV)
    first = i32([sum(held[:i]) for i in range(n)])
    at = torch.arange(table.shape[1], device=DEV, dtype=torch.int32)
    mine = at[None, :] < i32(held)[:, None]
    table[rows.long()] = torch.where(mine, pages[(first[:, None] + at[None, :]).clamp(max=n_pages - 1).long()], -1)
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[:n_pages - sum(held)] = pages[sum(held):]
    return dict(n_pages=n_pages, rows=rows, table=table, free=free, free_count=i32([n_pages - sum(held)]), kv_lens=i32([a for a, _ in lens]),
                new=i32([b for _, b in lens]), tokens=sum(b for _, b in lens) + c.get("pad", 0),
                free_after=torch.zeros(1, dtype=torch.int32, device=DEV), kv_after=torch.zeros(n, dtype=torch.int32, device=DEV),
                offsets=torch.zeros(n + 1, dtype=torch.int32, device=DEV), status=torch.zeros(2, dtype=torch.int32, device=DEV))


def token_outputs(s):
    for name in ("slots", "positions", "requests"):
        s[name] = torch.zeros(s["tokens"], dtype=torch.int32, device=DEV)


def rope_inputs(c, r, tokens):
    """Projections of one layer: rows [queries | keys | values]; with a norm also its weights, stored around zero."""
    H, K, D = c["heads"], c["kv_heads"], c["dim"]
    s = dict(qkv=r.normal(tokens, H + 2 * K, D, std=1.5, dtype=TYPE[c["source"]]), q=torch.zeros(tokens, H, D, dtype=TYPE[c["cache"]], device=DEV))
    if c["norm"]:
        s.update(q_norm=r.normal(D, std=0.2), k_norm=r.normal(D, std=0.2))
    return s


def axis_of_pairs(c):
    """Which position turns each pair of a head: a quarter time, the rest height and width (one axis: all alike)."""
    pairs = c["rot"] // 2
    if c["axes"] == 1:
        return [0] * pairs
    first = pairs // 4 if c["axes"] == 3 else pairs // 2
    return [0] * first + [1 + (i * (c["axes"] - 1)) // (pairs - first) for i in range(pairs - first)]


def prepare(case, seed):
    r, kind = Rng(seed), case["kind"]
    s = dict(case=case)
    if kind == "append":
        T, P = case["tokens"], case["page"]
        s.update(rope_inputs(case, r, T))
        n_pages = pages_of(T, P) + 5
        s["k_cache"], s["v_cache"] = (r.normal(n_pages, P, case["kv_heads"], case["dim"], dtype=TYPE[case["cache"]]) for _ in range(2))
        s["slots"] = (r.permutation(n_pages)[:pages_of(T, P), None] * P + torch.arange(P, device=DEV, dtype=torch.int32)).reshape(-1)[:T].contiguous()
        start = torch.randint(0, 200000, (1,), device=DEV, generator=r.g, dtype=torch.int32)
        at = torch.arange(T, device=DEV, dtype=torch.int32)
        side = max(1, math.isqrt(T // 2))  # images of side x side patches, one after the other
        s["positions"] = (start + torch.stack([at] if case["axes"] == 1 else [at // (side * side), at // side % side, at % side][:case["axes"]])).contiguous()
        s["layers"] = [s]
    else:
        lens = batch(case)
        s.update(paged_inputs(case, r, lens))
        s["lens"] = lens
        token_outputs(s)
        if kind == "attention":
            H, K, D, t = case["heads"], case["kv_heads"], case["dim"], TYPE[case["cache"]]
            plain_slots(s)  # the step's own plan: what stands before attention
            s["table"], s["kv_lens"] = s["table_after"], s["kv_after"]
            s["q"] = r.normal(s["tokens"], H, D, std=2.0, dtype=t)
            s["k_cache"], s["v_cache"] = (r.normal(s["n_pages"], case["page"], K, D, dtype=t) for _ in range(2))
            s["out"] = torch.zeros(s["tokens"], H, D, dtype=t, device=DEV)
            s["layers"] = [s]
        elif kind == "step":
            s["layers"] = []
            for _ in range(case["layers"]):
                l = rope_inputs(case, r, s["tokens"])
                l["k_cache"], l["v_cache"] = (r.normal(s["n_pages"], case["page"], case["kv_heads"], case["dim"], dtype=TYPE[case["cache"]])
                                              for _ in range(2))
                l["out"] = torch.zeros_like(l["q"])
                s["layers"].append(l)
        else:
            s["layers"] = []
        for l in s["layers"]:
            l["sinks"] = r.normal(case["heads"]) if case.get("sinks") else None
    s["table_after"] = s["table"].clone() if "table" in s else None
    if own:
        own_operations(s)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ the framework's calls
def own_operations(s):
    """The operations that a program keeps: addresses and sizes; lengths, tables and slots stay on the device."""
    import ctox_llm_b200 as ctox
    c, N = s["case"], ctox.native
    code = {"bf16": N.BF16, "f16": N.F16, "f32": N.F32}
    # torch's default stream has no address; 1 names it
    s["be"] = be = ctox.B200Backend(torch.cuda.current_device(), stream=torch.cuda.current_stream().cuda_stream or 1)
    if "table" in s and c["kind"] != "attention":
        s["slots_op"] = ctox.PageSlots(
            n_requests=len(s["lens"]), page_tokens=c["page"], n_pages=s["n_pages"], table_rows=s["table"].shape[0], max_pages=s["table"].shape[1],
            n_tokens=s["tokens"], new_tokens=s["new"].data_ptr(), rows=s["rows"].data_ptr(), kv_lens_in=s["kv_lens"].data_ptr(),
            kv_lens_out=s["kv_after"].data_ptr(), block_table=s["table_after"].data_ptr(), table_stride=s["table"].stride(0),
            free_pages=s["free"].data_ptr(), free_count_in=s["free_count"].data_ptr(), free_count_out=s["free_after"].data_ptr(),
            query_offsets=s["offsets"].data_ptr(), slots=s["slots"].data_ptr(), positions=s["positions"].data_ptr(),
            requests=s["requests"].data_ptr(), status=s["status"].data_ptr())
    for l in s["layers"]:
        k = l["k_cache"]
        kv = ctox.PagedKV(k=k.data_ptr(), v=l["v_cache"].data_ptr(), dtype=code[c["cache"]], page_tokens=c["page"], n_pages=k.shape[0],
                          page_stride=k.stride(0), token_stride=k.stride(1), head_stride=k.stride(2))
        q = l["q"]
        if c["kind"] != "attention":
            x, H, K = l["qkv"], c["heads"], c["kv_heads"]
            at = [x.data_ptr() + i * x.stride(1) * x.element_size() for i in (0, H, H + K)]
            l["append_op"] = ctox.RopeAppend(
                tokens=x.shape[0], heads=H, kv_heads=K, dim=c["dim"], rot_dim=c["rot"], axes=c["axes"],
                pairing=N.ROPE_HALF if c["pairing"] == "half" else N.ROPE_ADJACENT, rope_base=10000.0, axis=bytes(axis_of_pairs(c)),
                positions=s["positions"].data_ptr(), position_stride=s["positions"].stride(0) if c["axes"] > 1 else 0,
                source_dtype=code[c["source"]], q=at[0], k=at[1], v=at[2], q_token_stride=x.stride(0), q_head_stride=x.stride(1),
                k_token_stride=x.stride(0), k_head_stride=x.stride(1), v_token_stride=x.stride(0), v_head_stride=x.stride(1),
                q_norm=l["q_norm"].data_ptr() if c["norm"] else None, k_norm=l["k_norm"].data_ptr() if c["norm"] else None, norm_offset=1.0,
                norm_eps=1e-6, q_out=q.data_ptr(), q_out_token_stride=q.stride(0), q_out_head_stride=q.stride(1), slots=s["slots"].data_ptr(), kv=kv)
        if c["kind"] != "append":
            op = l["attention_op"] = ctox.PagedAttention(
                n_requests=len(s["lens"]), n_tokens=s["tokens"], max_new_tokens=max(b for _, b in s["lens"]),
                max_kv_tokens=max(a + b for a, b in s["lens"]), heads=c["heads"], dim=c["dim"], kv_heads=c["kv_heads"], causal=1,
                window=c["window"], scale=c["dim"] ** -0.5, query_offsets=s["offsets"].data_ptr(),
                kv_lens=(s["kv_lens"] if c["kind"] == "attention" else s["kv_after"]).data_ptr(), rows=s["rows"].data_ptr(),
                block_table=(s["table"] if c["kind"] == "attention" else s["table_after"]).data_ptr(), table_rows=s["table"].shape[0],
                max_pages=s["table"].shape[1], table_stride=s["table"].stride(0), sinks=l["sinks"].data_ptr() if c["sinks"] else None,
                q=q.data_ptr(), q_token_stride=q.stride(0), q_head_stride=q.stride(1), out=l["out"].data_ptr(),
                out_token_stride=l["out"].stride(0), out_head_stride=l["out"].stride(1), kv=kv)
            if "workspace" not in s:  # the layers of a step take turns with one
                s["workspace"] = torch.empty(be.paged_attention_workspace(op), dtype=torch.uint8, device=DEV)
            op.workspace, op.workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()


def run(s):
    kind = s["case"]["kind"]
    if own:
        be = s["be"]
        if kind in ("slots", "step"):
            be.page_slots(s["slots_op"])
        for l in s["layers"]:
            if kind != "attention":
                be.rope_append(l["append_op"])
            if kind != "append":
                be.paged_attention(l["attention_op"])
    else:
        if kind in ("slots", "step"):
            plain_slots(s)
        if kind == "append":
            plain_append(s, s)
        elif kind == "attention":
            plain_attention(s, s, s["table"], s["kv_lens"])
        else:
            for l in s["layers"]:
                plain_append(s, l)
                plain_attention(s, l, s["table_after"], s["kv_after"])
    out = {}
    if kind in ("slots", "step"):
        out.update((k, s[k]) for k in ("table_after", "free_after", "kv_after", "offsets", "slots", "positions", "requests", "status"))
    if kind in ("append", "step"):
        out.update(layers=[(l["q"], l["k_cache"], l["v_cache"]) for l in s["layers"]])
    if kind in ("attention", "step"):
        out.update(out=[l["out"] for l in s["layers"]])
    return out


# ------------------------------------------------------------------ the plain forms
def plain_slots(s):
    P, n = s["case"]["page"], s["new"].numel()
    old, new = s["kv_lens"].long(), s["new"].long()
    after = old + new
    held, wanted = (old + P - 1) // P, (after + P - 1) // P
    taken = torch.cumsum(wanted - held, 0)
    before = taken - (wanted - held)
    count = s["free_count"].long()
    fine = ((taken[-1] <= count[0]) & (wanted <= s["table"].shape[1]).all()).long()
    rows = s["rows"].long()
    at = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    fresh = (at >= held[:, None]) & (at < wanted[:, None]) & (fine == 1)
    page = s["free"][(count - 1 - (before - held)[:, None] - at).clamp(0, s["free"].numel() - 1)]
    s["table_after"] = s["table"].index_copy(0, rows, torch.where(fresh, page, s["table"][rows]))
    ends = torch.cumsum(new * fine, 0)
    t = torch.arange(s["tokens"], device=DEV)
    req = torch.searchsorted(ends, t, right=True)
    real = req < n
    req_ = req.clamp(max=n - 1)
    place = old[req_] + t - (ends - new)[req_]
    page = s["table_after"][rows[req_], (place // P).clamp(0, s["table"].shape[1] - 1)].long()
    s["slots"] = torch.where(real, page * P + place % P, -1).int()
    s["positions"] = torch.where(real, place, 0).int()
    s["requests"] = torch.where(real, req, -1).int()
    s["offsets"] = torch.cat([torch.zeros_like(ends[:1]), ends]).int()
    s["kv_after"] = (old + new * fine).int()
    s["free_after"] = (count - taken[-1] * fine).int()
    s["status"] = torch.stack([taken[-1] * fine, 1 - fine]).int()


def turned(x, cos, sin, pairing):
    """The rotated dimensions x [tokens, heads, rot]; cos and sin [tokens, 1, rot / 2]."""
    a, b = x.chunk(2, -1) if pairing == "half" else (x[..., 0::2], x[..., 1::2])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.cat([u, w], -1) if pairing == "half" else torch.stack([u, w], -1).flatten(-2)


def angles(s):
    c = s["case"]
    freq = 10000.0 ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=F64) / c["rot"])
    positions = s["positions"].reshape(-1, s["positions"].shape[-1])
    a = positions[i32(axis_of_pairs(c)).long()].to(F64).t() * freq
    return a.cos()[:, None], a.sin()[:, None]


def plain_append(s, l):
    c = s["case"]
    H, K, R = c["heads"], c["kv_heads"], c["rot"]
    cos, sin = (a.float() for a in angles(s))
    q, k, v = l["qkv"].float().split([H, K, K], 1)
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * (1.0 + l["q_norm"])
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * (1.0 + l["k_norm"])
    q = torch.cat([turned(q[..., :R], cos, sin, c["pairing"]), q[..., R:]], -1)
    k = torch.cat([turned(k[..., :R], cos, sin, c["pairing"]), k[..., R:]], -1)
    l["q"].copy_(q)
    real = s["slots"] >= 0
    if c.get("pad"):
        k, v, slots = k[real], v[real], s["slots"][real].long()
    else:
        slots = s["slots"].long()
    t = TYPE[c["cache"]]
    l["k_cache"].view(-1, K, c["dim"]).index_copy_(0, slots, k.to(t))
    l["v_cache"].view(-1, K, c["dim"]).index_copy_(0, slots, v.to(t))


def attend(q, k, v, lens, new, c, sinks):
    """q [batch, m, heads, dim], k and v [batch, length, kv_heads, dim]; request b has `lens[b]` tokens in the cache, the last new[b] of
    them those of its first new[b] rows of q."""
    B, m, H, D = q.shape
    L, K = k.shape[1:3]
    s = (q.float() * D ** -0.5).view(B, m, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(B, K, -1, D) @ k.float().permute(0, 2, 3, 1)
    s = s.view(B, K, H // K, m, L)
    last = (lens - new)[:, None] + torch.arange(m, device=DEV)
    key = torch.arange(L, device=DEV)
    seen = key <= last[..., None]
    if c["window"]:
        seen &= key > last[..., None] - c["window"]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + (sinks.view(1, K, H // K, 1, 1) - top).exp()
    o = (p.view(B, K, -1, L) @ v.float().permute(0, 2, 1, 3)).view(B, K, H // K, m, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, m, H, D)


def plain_attention(s, l, table, kv_lens):
    c, lens = s["case"], s["lens"]
    n, P, m = len(lens), c["page"], max(b for _, b in lens)
    rows, K, D = s["rows"].long(), c["kv_heads"], c["dim"]
    kv = kv_lens.long()

    def of(i, j, q, length):  # requests i to j, of `length` tokens at most, as one batch
        pages = table[rows[i:j], :pages_of(length, P)].clamp(min=0).long()
        k, v = (l[x][pages].reshape(j - i, -1, K, D) for x in ("k_cache", "v_cache"))
        return attend(q, k, v, kv[i:j], s["new"][i:j].long(), c, l["sinks"])

    ends = list(itertools.accumulate((b for _, b in lens), initial=0))
    if ends[-1] == n * m:  # every request has as many rows
        o = of(0, n, l["q"][:n * m].view(n, m, c["heads"], D), max(a + b for a, b in lens)).flatten(0, 1)
    else:
        o = torch.cat([of(i, i + 1, l["q"][None, ends[i]:ends[i + 1]], sum(lens[i]))[0] for i in range(n)])
    l["out"][:ends[-1]] = o


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, kind = case, case["kind"]
    lens = batch(c) if kind != "append" else []
    T = c["tokens"] if kind == "append" else sum(b for _, b in lens)
    size = {"f32": 4, "bf16": 2, "f16": 2}
    total, flops = 0.0, 0.0
    if kind in ("slots", "step"):
        fresh = sum(pages_of(a + b, c["page"]) - pages_of(a, c["page"]) for a, b in lens)
        # lengths, rows and offsets of the requests, pages from the stack into the table, the page that each request writes on into, three words a token
        total += 4.0 * (6 * len(lens) + 2 * fresh + 3 * (T + c["pad"]))
        flops += 4.0 * (T + len(lens))
    L = c.get("layers", 1)
    if kind in ("append", "step"):
        H, K, D = c["heads"], c["kv_heads"], c["dim"]
        total += L * T * ((H + 2 * K) * D * (size[c["source"]] + size[c["cache"]]) + 4.0 * (c["axes"] + 1))
        flops += L * T * (H + K) * (3.0 * c["rot"] + (4.0 * D if c["norm"] else 0))
    if kind in ("attention", "step"):
        H, K, D, W = c["heads"], c["kv_heads"], c["dim"], c["window"]
        pairs = sum(sum(min(a + i + 1, W) if W else a + i + 1 for i in range(b)) for a, b in lens)
        keys = sum(min(a + b, W + b - 1) if W else a + b for a, b in lens)
        total += L * (2.0 * T * H * D * size[c["cache"]] + 2.0 * keys * K * D * size[c["cache"]] + 4.0 * keys / c["page"])
        flops += L * 4.0 * pairs * H * D
    return dict(bytes=total, flops=flops)


# ------------------------------------------------------------------ the same from the definitions, in 64 bits
def exact_slots(s):
    """In order, request by request and token by token, on the host."""
    P, lens = s["case"]["page"], s["lens"]
    rows, table = s["rows"].tolist(), s["table"].cpu().clone()
    free, top = s["free"].tolist(), int(s["free_count"])
    start, slots, positions, requests, offsets = top, [], [], [], [0]
    for i, (a, b) in enumerate(lens):
        for t in range(a, a + b):
            if t % P == 0:
                top -= 1
                table[rows[i], t // P] = free[top]
            slots.append(int(table[rows[i], t // P]) * P + t % P)
            positions.append(t)
            requests.append(i)
        offsets.append(offsets[-1] + b)
    pad = s["tokens"] - len(slots)
    return dict(table_after=table.to(DEV), free_after=i32([top]), kv_after=i32([a + b for a, b in lens]), offsets=i32(offsets),
                slots=i32(slots + [-1] * pad), positions=i32(positions + [0] * pad), requests=i32(requests + [-1] * pad),
                status=i32([start - top, 0]))


def exact_rope(x, weight, s):
    """x [tokens, heads, dim] in 64 bits, normed and turned as complex numbers."""
    c = s["case"]
    R = c["rot"]
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * (1.0 + weight.to(F64))
    positions = s["positions"].reshape(-1, s["positions"].shape[-1]).to(F64)
    turn = torch.stack([torch.polar(torch.ones_like(positions[a]), positions[a] * 10000.0 ** (-2.0 * i / R)) for i, a in enumerate(axis_of_pairs(c))], -1)[:, None]
    if c["pairing"] == "half":
        z = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * turn
        return torch.cat([z.real, z.imag, x[..., R:]], -1)
    z = torch.complex(x[..., 0:R:2].contiguous(), x[..., 1:R:2].contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), x[..., R:]], -1)


def exact_append(s, l):
    """(queries, keys, values, key cache, value cache); the caches hold what is stored there, rounded to their type."""
    c, t = s["case"], TYPE[s["case"]["cache"]]
    H, K = c["heads"], c["kv_heads"]
    x = l["qkv"].to(F64)
    q = exact_rope(x[:, :H], l.get("q_norm"), s)
    k = exact_rope(x[:, H:H + K], l.get("k_norm"), s)
    caches = []
    for cache, new in ((l["k_cache"], k), (l["v_cache"], x[:, H + K:])):
        flat = cache.to(F64).view(-1, K, c["dim"]).clone()
        real = s["slots"] >= 0
        flat[s["slots"][real].long()] = new[real].to(t).to(F64)
        caches.append(flat.view(cache.shape))
    return q, caches[0], caches[1]


def exact_attention(s, q, k_cache, v_cache, table, sinks):
    c, start, out = s["case"], 0, []
    H, K, D, P, W = c["heads"], c["kv_heads"], c["dim"], c["page"], c["window"]
    for i, (a, b) in enumerate(s["lens"]):
        n = a + b
        pages = table[s["rows"][i].long()][:pages_of(n, P)].long()
        k, v = (x[pages].flatten(0, 1)[:n].to(F64) for x in (k_cache, v_cache))
        i0, keys = torch.arange(a, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        hidden = (keys > i0) | ((i0 - keys >= W) if W else False)
        heads = []
        for h in range(H):
            w = (q[start:start + b, h].to(F64) @ k[:, h // (H // K)].t() / math.sqrt(D)).masked_fill(hidden, -math.inf)
            z = torch.logsumexp(w, -1, keepdim=True)
            if sinks is not None:
                z = torch.logaddexp(z, sinks[h].to(F64))
            heads.append((w - z).exp() @ v[:, h // (H // K)])
        out.append(torch.stack(heads, 1))
        start += b
    if s["tokens"] > start:
        out.append(torch.zeros(s["tokens"] - start, H, D, dtype=F64, device=DEV))
    return torch.cat(out)


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    kind, t = case["kind"], TYPE.get(case.get("cache"))
    if kind == "attention":
        return dict(out=[exact_attention(s, s["q"], s["k_cache"], s["v_cache"], s["table"], s["sinks"])])
    out = {}
    if kind in ("slots", "step"):
        out = exact_slots(s)
        if kind == "slots":
            return out
        s.update(out)
    layers = [exact_append(s, l) for l in s["layers"]]
    if kind == "step":
        out["out"] = [exact_attention(s, q.to(t), k.to(t), v.to(t), out["table_after"], l["sinks"]) for (q, k, v), l in zip(layers, s["layers"])]
    return dict(out, layers=layers)
