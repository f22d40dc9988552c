"""The int8 K/V cache and the attention that reads it, as cases to be measured: their inputs, what a pass does and
has to move, a plain form in elementary torch operations, and the same in 64 bits.

The cache holds one layer's keys and values of a sequence and head as int8 codes with one float scale for each block
of `block` tokens:

    scale = max |x| / 127 over the block's values so far,   code = round(x / scale), half away from zero

where both quotients are rounded to 32 bits; a scale under the smallest normal float is 0, and so are its codes. A
block that is written again where it holds earlier tokens keeps its scale if that is the larger one; otherwise its
earlier codes are made again from the values that they stand for. Layout, of `slots` >= seq_len tokens:

    key codes   [sequence][layer][head][slot][lanes]             lanes: head_size rounded up to 16
    value codes [sequence][layer][head][slot / 16][lanes][16]    sixteen tokens of one dimension side by side
    scales      [sequence][layer][head][slot / block]
"""
import importlib.util
import math
import os

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TINY = 2.0 ** -126


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    def store(name, B, H, hs, S, block, pos, n, ragged, L=2):
        return dict(name=name, op="store", B=B, H=H, mul=1, hs=hs, S=S, block=block, pos=pos, n=n, ragged=ragged, L=L)

    def load(name, B, H, hs, S, block, pos, n, ragged, L=2):
        return dict(name=name, op="load", B=B, H=H, mul=1, hs=hs, S=S, block=block, pos=pos, n=n, ragged=ragged, L=L)

    def attend(name, B, H, mul, hs, S, block, pos, n, ragged, L=2):
        return dict(name=name, op="attend", B=B, H=H, mul=mul, hs=hs, S=S, block=block, pos=pos, n=n, ragged=ragged, L=L)

    return [
        # one decode step of a small chat model: the new token's K/V rows join a half-full block
        store("store_token_small", 1, 12, 64, 1024, 32, 300, 1, False),
        # one decode step of sixteen 7B conversations of different lengths
        store("store_token_batch", 16, 32, 128, 2048, 64, 1535, 1, True),
        # a ragged batch of prompt tails behind a shared beginning, heads that are no power of two
        store("store_tail_odd", 3, 5, 48, 500, 16, 211, 77, True),
        # eight whole 7B prompts at once
        store("store_prompt_batch", 8, 32, 128, 2048, 128, 0, 2048, False, L=1),
        # a prefix from the middle of short sequences, taken back to 32 bits
        load("load_prefix_odd", 3, 6, 48, 777, 16, 5, 333, True),
        # eight whole 7B sequences, taken back to 32 bits
        load("load_batch", 8, 32, 128, 2048, 64, 0, 2048, False, L=1),
        # one decode step of a small chat model
        attend("decode_small", 1, 12, 1, 64, 1024, 32, 300, 1, False),
        # one decode step of a 7B conversation at the end of its context
        attend("decode_one", 1, 32, 1, 128, 2048, 64, 2047, 1, False),
        # one decode step of sixteen 7B conversations of different lengths
        attend("decode_batch", 16, 32, 1, 128, 2048, 64, 2047, 1, True),
        # one decode step of eight long documents, four query heads to a K/V head
        attend("decode_long_shared", 8, 8, 4, 128, 32768, 128, 32767, 1, True, L=1),
        # a chunk of a 7B prompt behind what is cached
        attend("prompt_chunk", 1, 32, 1, 128, 2048, 64, 1024, 128, False),
        # four whole 7B prompts at once
        attend("prompt_batch", 4, 32, 1, 128, 2048, 64, 0, 2048, False, L=1),
    ]


def draw(rng):
    """A case of the same ranges: single tokens and prompts, small and large heads, short and long contexts, odd
    sizes, ragged batches, one to eight query heads for a K/V head."""
    spread = lambda a, b: int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))  # noqa: E731
    limit = {"store": 1.3e9, "load": 6.7e8, "attend": 3.5e8}
    while True:
        op = rng.choice(["store", "load", "attend", "attend"])
        c = dict(op=op, B=spread(1, 24), H=rng.choice([1, 2, 3, 4, 5, 6, 8, 12, 16, 24, 32]),
                 mul=rng.choice([1, 1, 2, 3, 4, 8]) if op == "attend" else 1,
                 hs=rng.choice([8, 16, 40, 48, 64, 64, 96, 128, 128, 128, 256]), block=rng.choice([16, 32, 64, 128]),
                 ragged=rng.random() < 0.6, L=rng.choice([1, 2, 3]))
        one = rng.random() < (0.5 if op != "load" else 0.1)
        c["n"] = 1 if one else spread(2, 2048)
        c["pos"] = spread(1, 32768 if one else 4096) - 1 if rng.random() < 0.8 else 0
        c["S"] = c["pos"] + c["n"] + rng.randrange(0, 200)
        w = work(c)
        scores = c["B"] * c["H"] * c["mul"] * c["n"] * (c["pos"] + c["n"]) if op == "attend" else 0
        if w["bytes"] <= limit[op] and w["flops"] <= 1.3e11 and scores <= 5e8 and c["B"] * c["L"] * c["H"] * c["S"] * c["hs"] <= 4e8:
            return c


def spans(c):
    """(first position, tokens) of each sequence of the call: with `ragged`, later ones are shorter, down to a third,
    and where three or more store or read many tokens the last one has none."""
    B = c["B"]
    got = []
    for b in range(B):
        part = 1.0 - (2.0 / 3.0) * b / max(1, B - 1) if c["ragged"] else 1.0
        pos, n = int(c["pos"] * part), max(1, int(c["n"] * part))
        if c["ragged"] and c["n"] > 1 and B > 2 and b == B - 1:
            n = 0
        got.append((pos, n))
    return got


def work(c):
    row = c["H"] * c["hs"]
    total, flops = 0, 0
    for pos, n in spans(c):
        if n == 0:
            continue
        if c["op"] == "load":  # codes and scales in, floats out, keys and values
            total += 2 * n * row * 5 + 2 * 4 * c["H"] * (n // c["block"] + 1)
            flops += 2 * n * row
        elif c["op"] == "store":  # floats in, codes and scales out, the earlier codes of a shared block, and what is read back
            back = pos + n - pos // c["block"] * c["block"]
            total += 2 * row * (4 * n + n + (back - n)) + 2 * row * 5 * back + 2 * 8 * c["H"] * (back // c["block"] + 1)
            flops += 2 * row * (4 * n + back)
        else:  # queries in, attended values out, the codes and scales of every key in sight once
            T = pos + n
            total += 8 * n * row * c["mul"] + 2 * T * row + 2 * 4 * c["H"] * (T // c["block"] + 1)
            flops += 4 * row * c["mul"] * (n * pos + n * (n + 1) // 2)
    return {"bytes": total, "flops": flops}


# --------------------------------------------------------------------------------------------------------- inputs
def sizes(c):
    unit = max(64, c["block"])
    slots = -(-c["S"] // unit) * unit
    return slots, -(-c["hs"] // 16) * 16, slots // c["block"]


def prepare(c, seed):
    """The cache as earlier calls left it (tokens below each sequence's position, behind them what other requests
    left there), the rows of this call, and the buffers that it fills."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    B, L, H, hs, S, blk = (c[k] for k in ("B", "L", "H", "hs", "S", "block"))
    slots, lanes, blocks = sizes(c)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEVICE)  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device=DEVICE)  # noqa: E731
    span = spans(c)
    pos = torch.tensor([p for p, _ in span], dtype=torch.int32, device=DEVICE)
    num = torch.tensor([n for _, n in span], dtype=torch.int32, device=DEVICE)
    held = pos + num if c["op"] != "store" else pos  # tokens that the cache holds before the call
    s = {"case": c, "pos": pos, "num": num, "layer": L - 1, "longest": max(p + n for p, n in span)}
    # keys have channels of different size, values heads of different size, and some tokens stand out
    spread = {"k": 0.3 + 1.4 * rand(H, 1, hs), "v": 0.5 + rand(H, 1, 1)}
    for w in ("k", "v"):
        if c["op"] == "attend" or c["op"] == "load" or int(pos.max()) > 0:
            x = randn(B, H, slots, hs).mul_(spread[w]).mul_(1 + 2 * rand(B, H, slots, 1).pow_(6))
            x.mul_((torch.arange(slots, device=DEVICE) < held.view(B, 1)).view(B, 1, slots, 1))
            codes, scale = quantised(x.view(B, H, blocks, blk, hs))
            del x
        else:
            codes, scale = torch.zeros(B, H, blocks, blk, hs, dtype=torch.int8, device=DEVICE), torch.zeros(B, H, blocks, device=DEVICE)
        full = torch.randint(-127, 128, (B, L, H, slots, lanes), generator=g, device=DEVICE, dtype=torch.int8)
        old = (torch.arange(slots, device=DEVICE) < held.view(B, 1)).view(B, 1, slots, 1)
        full[:, -1, :, :, :hs] = torch.where(old, codes.view(B, H, slots, hs), full[:, -1, :, :, :hs])
        every = rand(B, L, H, blocks).mul_(0.05)
        some = (torch.arange(blocks, device=DEVICE) * blk < held.view(B, 1)).view(B, 1, blocks)
        every[:, -1] = torch.where(some, scale, every[:, -1])
        if w == "v":
            full = full.view(B, L, H, slots // 16, 16, lanes).transpose(-1, -2).contiguous()
        s[w + "c"], s[w + "s"] = full, every
        del full, codes
    rows = c["n"]
    if c["op"] == "attend":
        s["q"] = randn(B, rows, H * c["mul"] * hs)
        s["out"] = torch.zeros(B, rows, H * c["mul"] * hs, device=DEVICE)
    elif c["op"] == "store":
        for w in ("k", "v"):
            x = randn(B, rows, H, hs) * spread[w].view(1, 1, H, -1) * (1 + 2 * rand(B, rows, H, 1).pow(6))
            s[w] = x.reshape(B, rows, H * hs)
    if c["op"] != "attend":  # a store's rows are read back from the start of the first block that it writes
        first = pos // blk * blk if c["op"] == "store" else pos
        back = torch.where(num > 0, pos + num - first, 0)
        s["first"], s["back"] = first.to(torch.int32), back.to(torch.int32)
        s["rows"] = int(back.max())
        s["k_out"], s["v_out"] = (torch.zeros(B, s["rows"], H * hs, device=DEVICE) for _ in range(2))
    return s


def quantised(x):
    """Codes and scales of whole blocks, [..., block, head_size]."""
    scale = x.abs().amax((-1, -2)) / 127
    scale = torch.where(scale < TINY, 0.0, scale)
    return rounded(x, scale[..., None, None]), scale


def rounded(x, scale):
    """round(x / scale), half away from zero; the quotient is rounded to 32 bits before it is rounded to a whole number."""
    y = (x.double() / scale.double()).float().double()
    y = torch.where(scale > 0, (y.abs() + 0.5).floor().clamp(max=127) * y.sign(), 0.0)
    return y.to(torch.int8)


# ---------------------------------------------------------------------------------------------------- plain forms
def seen(s, w, at):
    """The values that the codes at the positions `at` [B, T] of this call's layer stand for: [B, H, T, head_size]."""
    c = s["case"]
    codes, scale = s[w + "c"][:, s["layer"]], s[w + "s"][:, s["layer"]]
    b = torch.arange(c["B"], device=DEVICE).view(-1, 1)
    got = codes[b, :, at] if w == "k" else codes[b, :, at // 16, :, at % 16]
    got = got[..., :c["hs"]].float() * scale[b, :, at // c["block"]].unsqueeze(-1)
    return got.transpose(1, 2)


def plain_load(s):
    c, rows = s["case"], s["rows"]
    at = s["first"].view(-1, 1).long() + torch.arange(rows, device=DEVICE)
    there = (torch.arange(rows, device=DEVICE) < s["back"].view(-1, 1)).view(c["B"], rows, 1)
    at = at.clamp(max=c["S"] - 1)
    k, v = (seen(s, w, at).transpose(1, 2).reshape(c["B"], rows, -1) for w in ("k", "v"))
    return {"k": torch.where(there, k, 0.0), "v": torch.where(there, v, 0.0)}


def plain_put(s, w):
    """Brings the call's rows of keys (w = "k") or values into the cache: over a window of whole blocks that holds
    every token that a sequence may write."""
    c = s["case"]
    B, H, hs, blk, layer = c["B"], c["H"], c["hs"], c["block"], s["layer"]
    blocks = sizes(c)[2]
    wide = min(blocks, (c["n"] + blk - 2) // blk + 1)  # blocks in the window
    pos, num = s["pos"].view(B, 1).long(), s["num"].view(B, 1).long()
    which = (pos // blk).clamp(max=blocks - wide) + torch.arange(wide, device=DEVICE)  # [B, wide]
    at = which[:, :1] * blk + torch.arange(wide * blk, device=DEVICE)
    b = torch.arange(B, device=DEVICE).view(B, 1)
    split = lambda x: x.view(B, wide, blk, *x.shape[2:])  # noqa: E731
    new = split((at >= pos) & (at < pos + num)).view(B, wide, blk, 1, 1)
    old = split(at < pos).view(B, wide, blk, 1, 1)
    hit = new.any(2).view(B, wide, 1)  # blocks that are written
    x = torch.where(new, split(s[w].view(B, c["n"], H, hs)[b, (at - pos).clamp(0, c["n"] - 1)]), 0.0)
    before = split(seen(s, w, at).transpose(1, 2))
    was = s[w + "s"][:, layer][b, :, which]  # [B, wide, H]
    scale = x.abs().amax((2, 4)).double().div(127).float()
    scale = torch.where(scale < TINY, 0.0, scale)
    scale = torch.where(old[:, :, 0, 0] & hit, torch.maximum(scale, was), scale)
    codes = rounded(torch.where(old, before, x), scale.view(B, wide, 1, H, 1))
    again = (scale > was).view(B, wide, 1, H, 1)  # earlier tokens change their codes where the scale grew
    write = new | (old & again & hit.view(B, wide, 1, 1, 1))
    if w == "k":
        held = s["kc"][:, layer, :, :, :hs]
        held[b, :, at] = torch.where(write, codes, split(held[b, :, at])).flatten(1, 2)
    else:
        held = s["vc"][:, layer, :, :, :hs]
        held[b, :, at // 16, :, at % 16] = torch.where(write, codes, split(held[b, :, at // 16, :, at % 16])).flatten(1, 2)
    s[w + "s"][:, layer][b, :, which] = torch.where(hit, scale, was)


def plain_attend(s):
    c, T = s["case"], s["longest"]
    B, H, hs, mul, n = c["B"], c["H"], c["hs"], c["mul"], c["n"]
    at = torch.arange(T, device=DEVICE).expand(B, T)
    k, v = seen(s, "k", at), seen(s, "v", at)  # [B, H, T, hs]
    q = s["q"].view(B, n, H, mul, hs).permute(0, 2, 3, 1, 4).reshape(B, H, mul * n, hs)
    x = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(hs)  # [B, H, mul * n, T]
    del k
    row = torch.arange(n, device=DEVICE)
    sees = at.view(B, 1, T) <= (s["pos"].view(B, 1) + row).view(B, n, 1)
    x = torch.where(sees.view(B, 1, 1, n, T), x.view(B, H, mul, n, T), -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    total = x.sum(-1, keepdim=True)
    x = torch.matmul(x.view(B, H, mul * n, T), v).view(B, H, mul, n, hs) / total
    x = x.permute(0, 3, 1, 2, 4).reshape(B, n, H * mul * hs)
    return {"out": torch.where((row < s["num"].view(B, 1)).view(B, n, 1), x, 0.0)}


def plain(s):
    if s["case"]["op"] == "attend":
        return plain_attend(s)
    if s["case"]["op"] == "store":
        plain_put(s, "k")
        plain_put(s, "v")
    return plain_load(s)


# --------------------------------------------------------------------------------------------- the framework's own
def binding():
    """This repository's package (its folder's name has a dot, so it is loaded from its path) and its C interface."""
    if "tl" not in binding.__dict__:
        at = os.path.join(os.getcwd(), "hip_llama.cpp_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location("hip_llama_cpp_amd_boot", at)
        boot = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(boot)
        boot.load()
        from hip_llama_cpp_amd import thallama
        binding.tl = thallama
    return binding.tl


class Plan:
    """What a program that makes these calls step after step keeps: the handle on its stream, the cache's pointers and
    the workspace; for the stream and the tensors that it was made for, no others."""

    def __init__(self, s):
        tl, c = binding(), s["case"]
        lib, self.check = tl.lib(), tl.check
        self.device = s["kc"].device.index
        self.stream = raw_stream(self.device)
        self.kc, self.vc, self.ks, self.vs = (s[w] for w in ("kc", "vc", "ks", "vs"))
        cache = tl.Q8KVCache.make(c["B"], c["L"], c["H"], c["hs"], c["S"], c["block"], *(s[w].data_ptr() for w in ("kc", "vc", "ks", "vs")))
        self.handle, self.cache = tl.C.byref(tl.Handle(self.device, self.stream, None)), tl.C.byref(cache)
        self.size = lib.thaDNN_q8_attention_workspace(self.cache, c["B"], c["n"], c["H"] * c["mul"]) if c["op"] == "attend" else 0
        self.work = torch.zeros(max(1, self.size), dtype=torch.uint8, device=s["kc"].device)
        self.store, self.load, self.attend = lib.thaDNN_q8_kv_store_batch, lib.thaDNN_q8_kv_load_batch, lib.thaDNN_q8_attention_batch


raw_stream = torch._C._cuda_getCurrentRawStream if DEVICE == "cuda" else None  # torch.cuda.current_stream() takes 2.7 us


def kernels(s):
    p = s.get("plan")
    if (p is None or p.stream != raw_stream(p.device) or p.kc is not s["kc"] or p.vc is not s["vc"] or p.ks is not s["ks"]
            or p.vs is not s["vs"]):
        p = s["plan"] = Plan(s)
    c, at = s["case"], torch.Tensor.data_ptr
    op, B, n, row = c["op"], c["B"], c["n"], c["H"] * c["hs"]
    if op == "attend":
        row *= c["mul"]
        p.check(p.attend(p.handle, p.cache, s["layer"], B, n, at(s["pos"]), at(s["num"]), c["H"] * c["mul"], at(s["q"]), at(s["out"]),
                         row, row, at(p.work), p.size))
        return {"out": s["out"]}
    if op == "store":
        p.check(p.store(p.handle, p.cache, s["layer"], B, n, at(s["pos"]), at(s["num"]), at(s["k"]), at(s["v"]), row))
    p.check(p.load(p.handle, p.cache, s["layer"], B, s["rows"], at(s["first"]), at(s["back"]), at(s["k_out"]), at(s["v_out"]), row))
    return {"k": s["k_out"], "v": s["v_out"]}


def run(s):
    return kernels(s) if own else plain(s)


# ------------------------------------------------------------------------------------------------------- in 64 bits
def exact(c, seed):
    """The same from the definition, sequence after sequence and block after block, in 64 bits. What the definition
    rounds to 32 bits on its way to a code (a scale, a quotient, an earlier code's value) is rounded here too."""
    s = prepare(c, seed)
    H, hs, mul, blk, last = c["H"], c["hs"], c["mul"], c["block"], c["L"] - 1
    f64, f32 = torch.float64, torch.float32

    def held(w, b, first, count):
        """[H, count, head_size] values of sequence b in 64 bits."""
        codes = s[w + "c"][b, last]
        if w == "v":
            codes = codes.permute(0, 1, 3, 2).reshape(H, -1, codes.shape[2])
        scale = s[w + "s"][b, last].to(f64).repeat_interleave(blk, 1)
        return codes[:, first:first + count, :hs].to(f64) * scale[:, first:first + count, None]

    if c["op"] == "attend":
        out = torch.zeros(c["B"], c["n"], H, mul, hs, dtype=f64, device=DEVICE)
        for b, (pos, n) in enumerate(spans(c)):
            if n == 0:
                continue
            k, v = held("k", b, 0, pos + n), held("v", b, 0, pos + n)
            q = s["q"][b].view(c["n"], H, mul, hs).to(f64)
            hidden = torch.ones(n, pos + n, dtype=torch.bool, device=DEVICE).triu(pos + 1)
            for m in range(mul):
                x = torch.bmm(q[:n, :, m].transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) * hs ** -0.5
                out[b, :n, :, m] = torch.bmm(torch.softmax(x.masked_fill(hidden, -math.inf), -1), v).transpose(0, 1)
        return {"out": out.view(c["B"], c["n"], -1)}

    got = {}
    for w in ("k", "v"):
        res = torch.zeros(c["B"], s["rows"], H, hs, dtype=f64, device=DEVICE)
        for b, (pos, n) in enumerate(spans(c)):
            if n == 0:
                continue
            if c["op"] == "load":
                res[b, :n] = held(w, b, pos, n).transpose(0, 1)
                continue
            base = pos // blk * blk
            for at in range(base, pos + n, blk):
                lo, hi = max(at, pos), min(at + blk, pos + n)
                x = s[w][b, lo - pos:hi - pos].view(hi - lo, H, hs).transpose(0, 1).to(f64)
                scale = (x.abs().amax((1, 2)) / 127).to(f32).to(f64)
                scale[scale < TINY] = 0
                if at < pos:
                    was = s[w + "s"][b, last, :, at // blk].to(f64)
                    before = held(w, b, at, pos - at)
                    grew = scale > was
                    scale = torch.maximum(scale, was)
                    made = whole(before.to(f32).to(f64), scale)
                    before = torch.where(grew[:, None, None], made, before)
                    res[b, at - base:pos - base] = before.transpose(0, 1)
                res[b, lo - base:hi - base] = whole(x, scale).transpose(0, 1)
        got[w] = res.view(c["B"], s["rows"], -1)
    return got


def whole(x, scale):
    """What the codes of x [H, tokens, head_size] under scale [H] stand for."""
    scale = scale.view(-1, 1, 1)
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, 1.0), 0.0).to(torch.float32).to(torch.float64)
    up = torch.where(y < 0, torch.ceil(y - 0.5), torch.floor(y + 0.5))
    return up.clamp(-127, 127) * scale
