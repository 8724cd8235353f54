"""A plain 64-bit model of a batch over a paged K/V cache, and the operations on it."""
import math

import torch

import ctox_llm_b200 as ctox

N = ctox.native
DTYPE = {"bf16": (torch.bfloat16, N.BF16), "f16": (torch.float16, N.F16), "f32": (torch.float32, N.F32)}


def near(got, want, tolerance):
    """Whether all of got is within the tolerance; prints by how much not."""
    off = ((got.double() - want).abs() / tolerance.clamp(min=1e-300)).nan_to_num(nan=float("inf"))
    worst = off.max().item() if off.numel() else 0.0
    if worst > 1:
        at = off.argmax().item()
        print(f"{worst:.4g} times the tolerance at {at} of {tuple(off.shape)}: {got.reshape(-1)[at].item()} for {want.reshape(-1)[at].item()}, "
              f"{(off > 1).sum().item()} values")
    return worst <= 1


class Cache:
    """Pages of keys and values for requests of `lens` tokens, permuted; everything outside the requests' tokens is NaN.
    layout: "nhd" [page][token][head][dim], "hnd" [page][head][token][dim], "both" [page][token][head][key | value]."""

    def __init__(self, lens, kv_heads, dim, page, dtype, layout="nhd", seed=0, extra_pages=3, spare_rows=2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.page, self.kv_heads, self.dim, self.dtype = list(lens), page, kv_heads, dim, dtype
        t = DTYPE[dtype][0]
        held = [-(-n // page) for n in lens]
        self.n_pages = sum(held) + extra_pages
        shape = {"nhd": (self.n_pages, page, kv_heads, dim), "hnd": (self.n_pages, kv_heads, page, dim),
                 "both": (self.n_pages, page, kv_heads, 2 * dim)}[layout]
        if layout == "both":
            self.store = torch.full(shape, float("nan"), dtype=t, device="cuda")
            k, v = self.store[..., :dim], self.store[..., dim:]
        else:
            k, v = (torch.full(shape, float("nan"), dtype=t, device="cuda") for _ in range(2))
            if layout == "hnd":
                k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.k, self.v = k, v  # [page][token][head][dim], strided
        order = torch.randperm(self.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        n_rows = len(lens) + spare_rows
        self.rows_list = torch.randperm(n_rows, generator=torch.Generator().manual_seed(seed + 1)).tolist()[:len(lens)]
        self.table = torch.full((n_rows, max(held, default=0) + 2), -1, dtype=torch.int32)
        self.pages, at = [], 0
        for r, n in zip(self.rows_list, held):
            self.pages.append(order[at:at + n])
            self.table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.free = order[at:]
        self.table, self.rows = self.table.cuda(), torch.tensor(self.rows_list, dtype=torch.int32, device="cuda")
        self.key, self.value = [], []
        for i, n in enumerate(lens):
            a, b = (torch.randn(n, kv_heads, dim, generator=g, device="cuda").to(t) for _ in range(2))
            self.key.append(a)
            self.value.append(b)
            for j, p in enumerate(self.pages[i]):
                part = slice(j * page, min((j + 1) * page, n))
                self.k[p, :part.stop - part.start] = a[part]
                self.v[p, :part.stop - part.start] = b[part]

    def op(self):
        s = self.k.stride()
        return ctox.PagedKV(k=self.k.data_ptr(), v=self.v.data_ptr(), dtype=DTYPE[self.dtype][1], page_tokens=self.page, n_pages=self.n_pages,
                            page_stride=s[0], token_stride=s[1], head_stride=s[2])


def attention_op(be, cache, q, out, new, causal=1, window=0, scale=None, sinks=None, **more):
    """The operation and the tensors that it points to."""
    heads, dim = q.shape[1:]
    offsets = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    kv_lens = torch.tensor(cache.lens, dtype=torch.int32, device="cuda")
    fields = dict(n_requests=len(new), n_tokens=q.shape[0], max_new_tokens=max(new), max_kv_tokens=max(cache.lens), heads=heads,
                  kv_heads=cache.kv_heads, dim=dim, causal=causal, window=window, scale=scale or dim ** -0.5, query_offsets=offsets.data_ptr(),
                  kv_lens=kv_lens.data_ptr(), rows=cache.rows.data_ptr(), block_table=cache.table.data_ptr(), table_rows=cache.table.shape[0],
                  max_pages=cache.table.shape[1], table_stride=cache.table.stride(0), sinks=None if sinks is None else sinks.data_ptr(),
                  q=q.data_ptr(), q_token_stride=q.stride(0), q_head_stride=q.stride(1), out=out.data_ptr(),
                  out_token_stride=out.stride(0), out_head_stride=out.stride(1), kv=cache.op())
    fields.update(more)
    op = ctox.PagedAttention(**fields)
    workspace = torch.full((be.paged_attention_workspace(op),), 255, dtype=torch.uint8, device="cuda")
    if "workspace" not in more:
        op.workspace, op.workspace_bytes = workspace.data_ptr(), workspace.numel()
    return op, (offsets, kv_lens, workspace, sinks)


def attention64(cache, q, new, causal=True, window=0, scale=None, sinks=None):
    """[sum(new), heads, dim] in 64 bits, and the same with absolute values: sum of w |v| / sum of w."""
    heads, dim = q.shape[1:]
    group = heads // cache.kv_heads
    out, size, start = [], [], 0
    for i, m in enumerate(new):
        L = cache.lens[i]
        k, v = (x[i].double().repeat_interleave(group, 1).transpose(0, 1) for x in (cache.key, cache.value))
        s = q[start:start + m].double().transpose(0, 1) @ k.transpose(1, 2) * (scale or dim ** -0.5)
        if causal:
            last = L - m + torch.arange(m, device=q.device)[:, None]
            t = torch.arange(L, device=q.device)[None]
            s = s.masked_fill((t > last) | ((t <= last - window) if window else torch.zeros_like(t, dtype=torch.bool)), -math.inf)
        if L:
            top = s.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            w = (s - top).exp()
            total = w.sum(-1, keepdim=True)
            if sinks is not None:
                total = total + (sinks.double()[:, None, None] - top).exp()
            w = torch.where(w.sum(-1, keepdim=True) > 0, w / total, 0.0)
            out.append((w @ v).transpose(0, 1))
            size.append((w @ v.abs()).transpose(0, 1))
        else:
            out.append(torch.zeros(m, heads, dim, dtype=torch.float64, device=q.device))
            size.append(out[-1])
        start += m
    return torch.cat(out), torch.cat(size)


def attention_tolerance(dtype, want, size, longest):
    """How far a kernel's output may be. Weights w rounded to the type: half a step of each, so half * sum w |v| (`size`); the
    output's own rounding. Scores in 32 bits: a product of up to 256 terms added in at most 32 steps, each off by 2^-23 of the sum
    of absolute values, which is below 64 here (|q| |k| / sqrt(dim)): 2^-12, and a weight is off by twice that, its own and
    the denominator's. In f16 weights below 2^-14 of the largest are off by up to 2^-25, values of up to 6 times as many keys, and
    so is an output below 2^-14."""
    half = torch.finfo(DTYPE[dtype][0]).eps / 2
    small = 2.0 ** -25 * (1 + 6 * longest) if dtype == "f16" else 0.0
    return half * size + half * (1 + half) * want.abs() + 2.0 ** -11 * size + small
