"""The operators of serving from a paged cache on the caller's own memory, as cases to
time: appending tokens (norm, rotation, f32 rows or 8-bit blocks), attention of
packed prompts, and attention of new tokens over the 8-bit cache.

Head shapes, windows and rotation bases are those of spkv.SHAPES (`small` those of the
smoke test); the cache is the library's: pages of 64 positions.  `run` computes the
operators in elementary torch operations, or, where `own` is true, calls the library
on the same memory.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

PAGE, BLOCK = 64, 16
# q heads, kv heads, head dim, sliding window of the window layers
SHAPES = {
    "small": (4, 2, 64, 0),
    "qwen3-0.6b": (16, 8, 128, 0),
    "qwen3-8b": (32, 8, 128, 0),
    "gemma3-12b": (16, 8, 256, 1024),
}
ROPE_BASE, EPS = 1e6, 1e-6
RING_SPARE = 128                 # positions a ring keeps behind its window
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of a short chat: nothing but latency
        dict(name="append 0.6b 1 at 100", op="append", shape="qwen3-0.6b", type="f32", rows="block8", norm=True, kout=False, seqs=1, lo=100, hi=100, nlo=1, nhi=1),
        # a server's step: one token of each session
        dict(name="append 8b 64 sessions", op="append", shape="qwen3-8b", type="bf16", rows="block8", norm=True, kout=False, seqs=64, lo=256, hi=2048, nlo=1, nhi=1),
        # a packed batch of prompts into the f32 cache that tree attention reads
        dict(name="append 12b 5 prompts f32", op="append", shape="gemma3-12b", type="f32", rows="f32", norm=True, kout=True, seqs=5, lo=0, hi=0, nlo=33, nhi=777),
        # a long prompt into the 8-bit cache
        dict(name="append 8b 4096 tokens", op="append", shape="qwen3-8b", type="bf16", rows="block8", norm=True, kout=True, seqs=1, lo=0, hi=0, nlo=4096, nhi=4096),
        # a prompt of a few words
        dict(name="prompt 0.6b 7 tokens", op="prompt", shape="qwen3-0.6b", type="f32", window=0, seqs=1, nlo=7, nhi=7),
        # a server's packed batch of prompts of different lengths
        dict(name="prompt 8b 9 packed", op="prompt", shape="qwen3-8b", type="bf16", window=0, seqs=9, nlo=64, nhi=1000),
        # a window layer's long prompt in f32
        dict(name="prompt 12b window 2047", op="prompt", shape="gemma3-12b", type="f32", window=1024, seqs=1, nlo=2047, nhi=2047),
        # the longest prompt, every position before it seen
        dict(name="prompt 8b 8192", op="prompt", shape="qwen3-8b", type="bf16", window=0, seqs=1, nlo=8192, nhi=8192),
        # one token of a short chat
        dict(name="cache 0.6b 1 at 100", op="cache", shape="qwen3-0.6b", type="f32", window=0, seqs=1, lo=100, hi=100, nlo=1, nhi=1),
        # a server's step over ragged sessions
        dict(name="cache 8b 64 sessions", op="cache", shape="qwen3-8b", type="bf16", window=0, seqs=64, lo=256, hi=4096, nlo=1, nhi=1),
        # one token at the headline context
        dict(name="cache 12b 1 at 32k", op="cache", shape="gemma3-12b", type="f32", window=0, seqs=1, lo=32703, hi=32703, nlo=1, nhi=1),
        # pieces of prompts behind what is cached, in a window layer's ring
        dict(name="cache 12b window 4 x 48", op="cache", shape="gemma3-12b", type="f32", window=1024, seqs=4, lo=2000, hi=6001, nlo=17, nhi=48),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, shape, typ = rng.choice(["append", "prompt", "cache"]), rng.choice(sorted(SHAPES)), rng.choice(sorted(TYPES))
    W = SHAPES[shape][3]
    if op == "prompt":
        seqs = rng.choice([1, 1, _log_int(rng, 2, 16)])
        nhi = _log_int(rng, 2, 4096 if seqs == 1 else 1000)
        nlo = nhi if seqs == 1 else _log_int(rng, 1, nhi)
        return dict(op=op, shape=shape, type=typ, window=W if rng.random() < 0.5 else 0, seqs=seqs, nlo=nlo, nhi=nhi)
    if op == "cache":
        seqs = rng.choice([1, 1, _log_int(rng, 2, 48)])
        lo = _log_int(rng, 1, 32000 if seqs == 1 else 2000)
        nhi = rng.choice([1, 1, _log_int(rng, 2, 48)])
        if seqs * nhi > 256:
            nhi = 256 // seqs
        return dict(op=op, shape=shape, type=typ, window=W if rng.random() < 0.5 else 0, seqs=seqs, lo=lo,
                    hi=lo + (0 if seqs == 1 else _log_int(rng, 1, 2000)), nlo=rng.randint(1, nhi), nhi=nhi)
    rows, norm, kout = rng.choice(["block8", "block8", "f32"]), rng.random() < 0.7, rng.random() < 0.5
    seqs = rng.choice([1, _log_int(rng, 2, 64)])
    nhi = rng.choice([1, _log_int(rng, 2, 4000 // seqs)])
    lo = rng.choice([0, _log_int(rng, 1, 2000)])
    return dict(op=op, shape=shape, type=typ, rows=rows, norm=norm, kout=kout, seqs=seqs, lo=lo, hi=lo + rng.randint(0, 63), nlo=rng.randint(1, nhi), nhi=nhi)


# ---------------------------------------------------------------- inputs
def _sizes(what, lo, hi, n):
    """n sizes of [lo, hi], the case's own: outputs have one shape whatever the seed."""
    return np.random.default_rng([what, lo, hi, n]).integers(lo, hi + 1, n)


def _page_bytes(rows, NKV, HD):
    """8-bit pages: K codes [kv head][64][HD], V codes [kv head][HD][64], scales [K, V][kv head][block] f32."""
    return 2 * NKV * PAGE * HD * 4 if rows == "f32" else 2 * NKV * PAGE * HD + 2 * NKV * (PAGE // BLOCK) * 4


def _v_byte(pos):
    """The byte of a position in a column of a page's V codes: position 16 u + 4 g + i at 16 g + 4 u + i."""
    return (pos // 4 % 4) * 16 + (pos // 16 % 4) * 4 + pos % 4


def _views(pool, rows, NKV, HD):
    """The pool's parts as tensors: K, V rows, or K codes, V codes and scales."""
    n = pool.shape[0]
    if rows == "f32":
        return dict(rows=pool.view(torch.float32).view(n, 2, NKV, PAGE, HD))
    c = NKV * PAGE * HD
    return dict(k=pool[:, :c].view(torch.int8).view(n, NKV, PAGE, HD), v=pool[:, c:2 * c].view(torch.int8).view(n, NKV, HD, PAGE),
                scales=pool.view(torch.float32)[:, c // 2:].view(n, 2, NKV, PAGE // BLOCK))


def prepare(case, seed):
    g = np.random.default_rng([seed & 0x7FFFFFFF, 9])
    gen = torch.Generator(DEV).manual_seed(seed)
    NH, NKV, HD, _ = SHAPES[case["shape"]]
    dt = TYPES[case["type"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def put(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)

    S = case["seqs"]
    n = _sizes(2, case["nlo"], case["nhi"], S)
    cached = _sizes(1, case["lo"], case["hi"], S) if case["op"] != "prompt" else np.zeros(S, np.int64)
    T, start = int(n.sum()), np.concatenate([[0], np.cumsum(n)])
    seq, tok = np.repeat(np.arange(S), n), np.concatenate([np.arange(k) for k in n])
    pos = cached[seq] + tok
    st = dict(case=case, plan=None, T=T, max_tokens=int(n.max()), max_positions=int((cached + n).max()), start=put(start.astype(np.int32)),
              cached=put(cached.astype(np.int32)), seq=put(seq), tok=put(tok), pos=put(pos))
    # a few channels of q and k are much larger than the others, as in trained models
    wide = 1 + 4 * (torch.rand(HD, generator=gen, device=DEV) > 0.97).float()
    st["q"] = (randn(T, NH, HD) * wide).to(dt)
    if case["op"] != "cache":
        st["k"], st["v"] = (randn(T, NKV, HD) * wide).to(dt), randn(T, NKV, HD).to(dt)
    if case["op"] == "prompt":
        st["out"] = torch.empty(T, NH, HD, dtype=dt, device=DEV)
        return st
    rows, W = case.get("rows", "block8"), case.get("window", 0)
    ring = -(-(W + RING_SPARE) // PAGE) + 1 if W else 0
    need = [-(-int(c + k) // PAGE) for c, k in zip(cached, n)]
    need = [min(x, ring) if ring else x for x in need]
    table = np.zeros((S, ring or max(need)), np.int64)
    order, at = g.permutation(sum(need)), 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    P = len(order)
    pool = torch.zeros(P, _page_bytes(rows, NKV, HD), dtype=torch.uint8, device=DEV)
    parts = _views(pool, rows, NKV, HD)
    if rows == "f32":
        parts["rows"].copy_(randn(P, 2, NKV, PAGE, HD))
    else:
        for a in ("k", "v"):
            parts[a].copy_((torch.randn(parts[a].shape, generator=gen, device=DEV) * 40).round_().clamp_(-127, 127))
        parts["scales"].copy_(2.0 ** torch.randint(-6, -3, parts["scales"].shape, generator=gen, device=DEV))
    st.update(pool=pool, parts=parts, page=put(table), ring=ring)
    st["tables"] = pool.data_ptr() + st["page"] * pool.shape[1]                          # page addresses
    st["lists"] = st["tables"].data_ptr() + 8 * table.shape[1] * torch.arange(S, device=DEV)
    if case["op"] == "cache":
        st["out"] = torch.empty(T, NH, HD, dtype=dt, device=DEV)
        return st
    st["freq"] = ROPE_BASE ** (-2.0 * torch.arange(HD // 2, dtype=torch.float64, device=DEV) / HD)
    if case["norm"]:
        st["q_norm"], st["k_norm"] = 1 + 0.2 * randn(HD), 1 + 0.2 * randn(HD)
    st["q_out"] = torch.empty_like(st["q"])
    if case["kout"]:
        st["k_out"] = torch.empty_like(st["k"])
    # each token's block among those that the call touches, and each block's place
    first, last = cached // BLOCK, (cached + n - 1) // BLOCK
    base = np.concatenate([[0], np.cumsum(last - first + 1)])
    bseq = np.repeat(np.arange(S), last - first + 1)
    blk = np.concatenate([np.arange(a, b + 1) for a, b in zip(first, last)])
    st.update(block=put(base[seq] + pos // BLOCK - first[seq]), b_page=put(table[bseq, blk // (PAGE // BLOCK)]), b_in=put(blk % (PAGE // BLOCK)),
              b_old=put(np.clip(cached[bseq] - blk * BLOCK, 0, BLOCK)))
    return st


# ---------------------------------------------------------------- plain forms
def _rotated(x, st, weight):
    """Norm and rotation of every head, in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x * weight.double() / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    a = (st["pos"].double()[:, None] * st["freq"])[:, None]
    c, s, h = torch.cos(a), torch.sin(a), x.shape[-1] // 2
    return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)


def _block_scales(y, st, old):
    """Of each touched block and head the power of two that its values and codes take."""
    big = torch.zeros(st["b_page"].shape[0], y.shape[1], dtype=torch.float64, device=DEV)
    big.scatter_reduce_(0, st["block"][:, None].expand(-1, y.shape[1]), y.abs().amax(-1), "amax")
    m, e = torch.frexp(big)
    e = torch.where(m * 128 <= 127, e - 7, e - 6).clamp(min=-126)       # 127 2^e holds m 2^e
    scale = ((e.long() + 1023) << 52).view(torch.float64)
    return torch.where(st["b_old"][:, None] > 0, torch.maximum(scale, old), scale)


def _append_plain(st):
    c = st["case"]
    k, v = _rotated(st["k"], st, st.get("k_norm")), st["v"].double()
    out = dict(q_out=_rotated(st["q"], st, st.get("q_norm")).to(st["q"].dtype))
    if c["kout"]:
        out["k_out"] = k.to(st["k"].dtype)
    parts = st["parts"]
    page, slot = st["page"][st["seq"], st["pos"] // PAGE], st["pos"] % PAGE
    if c["rows"] == "f32":
        parts["rows"][page, 0, :, slot] = k.float()
        parts["rows"][page, 1, :, slot] = v.float()
        return {**out, **parts}
    sc = parts["scales"]
    places = st["b_in"][:, None] * BLOCK + torch.arange(BLOCK, device=DEV)      # positions of each block in its page
    page, byte = st["b_page"][:, None], _v_byte(places)
    parts["k"][page, :, places] = _block_codes(st, k, sc[:, 0], parts["k"][page, :, places])
    parts["v"][page, :, :, byte] = _block_codes(st, v, sc[:, 1], parts["v"][page, :, :, byte])
    return {**out, **parts}


def _block_codes(st, y, scales, old):
    """The codes [block][16][head][dim] of the touched blocks; their scales are put in place."""
    at = (st["b_page"], slice(None), st["b_in"])
    was = scales[at].double()
    s = _block_scales(y, st, was)
    before = torch.arange(BLOCK, device=DEV) < st["b_old"][:, None]
    again = torch.round(old.double() * torch.where(st["b_old"][:, None] > 0, was / s, torch.ones_like(s))[:, None, :, None])
    new = torch.where(before[:, :, None, None], again.to(torch.int8), old)
    new[st["block"], st["pos"] % BLOCK] = torch.round(y / s[st["block"]][..., None]).to(torch.int8)
    scales[at] = s.float()
    return new


def _softmax_sum(s, seen, v):
    s = s.masked_fill_(~seen, -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    return (s @ v) / s.sum(-1, keepdim=True).clamp(min=1e-30)


def _grouped(x, st, n):
    """[T][heads][HD] -> [seq][kv head][token x group][HD], zeros behind each sequence's tokens."""
    NH, NKV, HD, _ = SHAPES[st["case"]["shape"]]
    p = torch.zeros(st["case"]["seqs"], n, x.shape[1], HD, device=DEV)
    p[st["seq"], st["tok"]] = x.float()
    return p.view(p.shape[0], n, NKV, -1, HD).transpose(1, 2).reshape(p.shape[0], NKV, -1, HD)


def _ungrouped(o, st, n):
    NH, NKV, HD, _ = SHAPES[st["case"]["shape"]]
    o = o.view(o.shape[0], NKV, n, NH // NKV, HD).transpose(1, 2).reshape(o.shape[0], n, NH, HD)
    return o[st["seq"], st["tok"]].to(st["q"].dtype)


def _prompt_plain(st):
    c, n = st["case"], st["max_tokens"]
    NH, NKV, HD, _ = SHAPES[c["shape"]]
    q, k, v = _grouped(st["q"], st, n), _grouped(st["k"], st, n), _grouped(st["v"], st, n)
    t = torch.arange(n, device=DEV)
    seen = t <= t[:, None]
    if c["window"]:
        seen = seen & (t > t[:, None] - c["window"])
    s = (q @ k.transpose(2, 3).contiguous()).mul_(HD ** -0.5)
    return _ungrouped(_softmax_sum(s, seen.repeat_interleave(NH // NKV, 0), v), st, n)


def _cache_plain(st):
    c, N = st["case"], st["max_tokens"]
    NH, NKV, HD, _ = SHAPES[c["shape"]]
    W, cached = c["window"], st["cached"].long()
    first = (cached - W + 1).clamp(min=0) if W else torch.zeros_like(cached)
    n = min(st["max_positions"], W - 1 + N) if W else st["max_positions"]
    pos = first[:, None] + torch.arange(n, device=DEV)                           # [S, n]
    lp = pos // PAGE % st["ring"] if st["ring"] else pos // PAGE
    page, b = st["page"].gather(1, lp.clamp(max=st["page"].shape[1] - 1)), pos // BLOCK % (PAGE // BLOCK)
    parts = st["parts"]
    k = parts["k"][page, :, pos % PAGE].float() * parts["scales"][page, 0, :, b][..., None]
    v = parts["v"][page, :, :, _v_byte(pos)].float() * parts["scales"][page, 1, :, b][..., None]
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    at = cached[:, None] + torch.arange(N, device=DEV)                           # the tokens' positions
    seen = pos[:, None] <= at[..., None]
    if W:
        seen = seen & (pos[:, None] > at[..., None] - W)
    s = (_grouped(st["q"], st, N) @ k.transpose(2, 3).contiguous()).mul_(HD ** -0.5)
    return _ungrouped(_softmax_sum(s, seen.repeat_interleave(NH // NKV, 1)[:, None], v), st, N)


# ---------------------------------------------------------------- the library's
def _spkv():
    if "spkv" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shannon-prime-system_amd"))
    import spkv
    return spkv


def _plan(st):
    """The argument block and the buffers that a program keeps for its calls."""
    spkv, c = _spkv(), st["case"]
    NH, NKV, HD, _ = SHAPES[c["shape"]]
    common = dict(n_heads=NH, n_kv_heads=NKV, head_dim=HD, type=spkv.BF16 if c["type"] == "bf16" else spkv.F32, n_seqs=c["seqs"], n_tokens=st["T"],
                  max_tokens=st["max_tokens"], start=st["start"].data_ptr(), q=st["q"].data_ptr(), q_stride=NH * HD)
    kv = dict(k=st["k"].data_ptr(), k_stride=NKV * HD, v=st["v"].data_ptr(), v_stride=NKV * HD) if "k" in st else {}
    paged = dict(max_positions=st["max_positions"], ring_pages=st["ring"], cached=st["cached"].data_ptr(), tables=st["lists"].data_ptr()) if "ring" in st else {}
    if c["op"] == "append":
        a = spkv.AppendArgs(**common, **kv, **paged, rows=spkv.ROWS_F32 if c["rows"] == "f32" else spkv.ROWS_BLOCK8, eps=EPS, freq=st["freq"].data_ptr(),
                            q_norm=st["q_norm"].data_ptr() if c["norm"] else None, k_norm=st["k_norm"].data_ptr() if c["norm"] else None,
                            q_out=st["q_out"].data_ptr(), q_out_stride=NH * HD, k_out=st["k_out"].data_ptr() if c["kout"] else None, k_out_stride=NKV * HD)
        st["outs"] = dict(q_out=st["q_out"], **({"k_out": st["k_out"]} if c["kout"] else {}), **st["parts"])
        st["plan"] = (spkv.append, a)
        return
    out = dict(window=c["window"], scale=float(np.float32(HD ** -0.5)), out=st["out"].data_ptr(), out_stride=NH * HD)
    st["outs"] = st["out"]
    if c["op"] == "prompt":
        st["plan"] = (spkv.prompt_attention, spkv.PromptArgs(**common, **kv, **out))
        return
    a = spkv.CacheArgs(**common, **paged, **out)
    need = spkv.cache_attention_work(a)
    if need:
        st["work"] = torch.empty(need, dtype=torch.uint8, device=DEV)
        a.work, a.work_bytes = st["work"].data_ptr(), need
    st["plan"] = (spkv.cache_attention, a)


def run(st):
    if not own:
        return {"append": _append_plain, "prompt": _prompt_plain, "cache": _cache_plain}[st["case"]["op"]](st)
    if st["plan"] is None:
        _plan(st)
    call, args = st["plan"]
    call(args, torch.cuda.current_stream().cuda_stream)
    return st["outs"]


def work(case):
    """Each input read once, each output written once; pairs of a query and a position that it sees."""
    NH, NKV, HD, _ = SHAPES[case["shape"]]
    es, S, W = (4 if case["type"] == "f32" else 2), case["seqs"], case.get("window", 0)
    n = _sizes(2, case["nlo"], case["nhi"], S)
    T = int(n.sum())
    if case["op"] == "append":
        stored = 2 * NKV * HD * (4 if case["rows"] == "f32" else 1 + 4 / HD / BLOCK)
        return dict(bytes=float(T * ((2 * NH + (3 if case["kout"] else 2) * NKV) * HD * es + stored)), flops=float(T * (NH + NKV) * HD * (3 + 4 * case["norm"])))
    cached = _sizes(1, case["lo"], case["hi"], S) if case["op"] == "cache" else np.zeros(S, np.int64)
    pairs = sum(int(np.minimum(c + np.arange(k) + 1, W or 1 << 40).sum()) for c, k in zip(cached, n))
    spans = sum(int(c + k - max(0, c - W + 1 if W else 0)) for c, k in zip(cached, n))
    held = spans * 2.0 * NKV * (HD + 4 / BLOCK) if case["op"] == "cache" else T * 2.0 * NKV * HD * es
    return dict(bytes=float(2 * T * NH * HD * es + held), flops=4.0 * HD * NH * pairs)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    NH, NKV, HD, _ = SHAPES[case["shape"]]
    G, W = NH // NKV, case.get("window", 0)
    start, cached = st["start"].tolist(), st["cached"].tolist()
    if case["op"] == "append":
        return _append_exact(st, start, cached)
    out = torch.zeros(st["T"], NH, HD, dtype=torch.float64, device=DEV)
    for s in range(case["seqs"]):
        a, b = start[s], start[s + 1]
        if case["op"] == "prompt":
            lo, K, V = 0, st["k"][a:b].double(), st["v"][a:b].double()
        else:
            lo = max(0, cached[s] - W + 1) if W else 0
            K, V = _rows_exact(st, s, torch.arange(lo, cached[s] + b - a, device=DEV))
        p, t = torch.arange(K.shape[0], device=DEV) + lo, cached[s] + torch.arange(b - a, device=DEV)[:, None]
        hide = (p > t) | (p <= t - W) if W else p > t
        for h in range(NH):
            z = (st["q"][a:b, h].double() @ K[:, h // G].T.contiguous() / math.sqrt(HD)).masked_fill_(hide, -math.inf)
            out[a:b, h] = torch.softmax(z, 1) @ V[:, h // G].contiguous()
    return out


def _rows_exact(st, s, pos):
    """K and V values [position][kv head][dim] of the 8-bit pages, byte by byte."""
    NH, NKV, HD, _ = SHAPES[st["case"]["shape"]]
    lp = torch.div(pos, 64, rounding_mode="floor")
    pages = st["pool"][st["page"][s][lp % st["ring"] if st["ring"] else lp]]
    half, r = NKV * 64 * HD, pos % 64
    i = torch.arange(pos.shape[0], device=DEV)
    scales = pages[:, 2 * half:].contiguous().view(torch.float32).reshape(-1, 2, NKV, 4).double()[i, :, :, r // 16]
    k = pages[:, :half].reshape(-1, NKV, 64, HD)[i, :, r].view(torch.int8).double()
    v = pages[:, half:2 * half].reshape(-1, NKV, HD, 4, 4, 4)[i, :, :, r // 4 % 4, r // 16, r % 4].view(torch.int8).double()
    return k * scales[:, 0, :, None], v * scales[:, 1, :, None]


def _append_exact(st, start, cached):
    c = st["case"]
    NH, NKV, HD, _ = SHAPES[c["shape"]]
    pos = torch.cat([torch.arange(p, p + b - a, device=DEV) for p, a, b in zip(cached, start, start[1:])]).double()
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), torch.outer(pos, st["freq"]))[:, None]

    def rope(x, w):
        x = x.double()
        if w is not None:
            x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / HD + EPS) * w.double()
        z = torch.complex(x[..., :HD // 2], x[..., HD // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    k, v = rope(st["k"], st.get("k_norm")), st["v"].double()
    out = dict(q_out=rope(st["q"], st.get("q_norm")))
    if c["kout"]:
        out["k_out"] = k
    if c["rows"] == "f32":
        rows = st["parts"]["rows"].double()
        for s, p in enumerate(cached):
            at = torch.arange(p, p + start[s + 1] - start[s], device=DEV)
            pg = st["page"][s][at // 64]
            rows[pg, 0, :, at % 64], rows[pg, 1, :, at % 64] = k[start[s]:start[s + 1]], v[start[s]:start[s + 1]]
        return {**out, "rows": rows}
    # codes are whole numbers, compared with the plain form's one by one; the scales are powers of two
    sc = st["parts"]["scales"].double().cpu().numpy()
    page = st["page"].cpu().numpy()
    for y, which in ((k, 0), (v, 1)):
        big = y.abs().amax(-1).cpu().numpy()
        for s, p in enumerate(cached):
            end = p + start[s + 1] - start[s]
            for b in range(p // 16, (end - 1) // 16 + 1):
                a0, a1 = max(p, 16 * b), min(end, 16 * b + 16)
                e = np.ceil(np.log2(np.maximum(big[start[s] + a0 - p:start[s] + a1 - p].max(0), 1e-300) / 127))
                new = 2.0 ** np.maximum(e, -126)
                at = (page[s, b // 4], which, slice(None), b % 4)
                sc[at] = np.maximum(sc[at], new) if p > 16 * b else new
    return {**out, "k": None, "v": None, "scales": torch.from_numpy(sc)}
