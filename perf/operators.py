"""The 8-bit key/value cache (write, read back, attention over it) and the token log probabilities: cases, plain forms
in elementary torch operations, the framework's own calls, and 64-bit values to hold both against.

Five operators: kv8_write, kv8_read, attn8, token_logprobs, linear_logprobs (mimizuku_b200's names). A case's "op" says
which of them its pass runs:
  write    kv8_write of n tokens per sequence, then kv8_read of them (the values the 8 bits stand for)
  step     one decoding step's self-attention: kv8_write of a token per sequence, attn8, kv8_read of the block written
  attend   attn8 over a filled cache, with the probabilities of chosen heads where slots > 0
  logits   token_logprobs of rows of logits
  hidden   linear_logprobs of rows of hidden states against the embedding
"""
import math

import torch

own = False

HD = 64


def listed():
    return [
        # decoder self-attention of the tiny model for one sequence early in its text: the smallest call, latency
        dict(name="step_tiny", op="step", batch=1, heads=6, cap=448, lo=38, hi=38, block=64, kind="int8"),
        # the same for a full batch of large-v3 at ragged positions
        dict(name="step_batch", op="step", batch=32, heads=20, cap=448, lo=1, hi=448, block=32, kind="e4m3"),
        # the cross k/v of an encoder group of 8 clips, the four decoder layers of large-v3-turbo
        dict(name="write_clips", op="write", batch=32, heads=20, cap=1500, n=1500, block=64, kind="int8"),
        # cross-attention of one layer, a batch of 32 clips of large-v3, 6 alignment heads recorded
        dict(name="cross_batch", op="attend", batch=32, rows=1, heads=20, group=1, cap=1500, lo=1500, hi=1500,
             block=64, kind="int8", causal=False, slots=6),
        # 5 hypotheses of each clip share its cross k/v
        dict(name="cross_beams", op="attend", batch=6, rows=5, heads=20, group=1, cap=1500, lo=1500, hi=1500,
             block=64, kind="e4m3", causal=False, slots=2),
        # a prompt of earlier text attends causally over what the cache holds, ragged lengths (one shorter than the rows)
        dict(name="prompt", op="attend", batch=8, rows=223, heads=20, group=1, cap=448, lo=150, hi=448, block=16,
             kind="int8", causal=True, slots=0),
        # a long cache with 4 query heads to a key head, one sequence of it empty
        dict(name="long", op="attend", batch=3, rows=1, heads=5, group=4, cap=131072, lo=0, hi=131072, block=128,
             kind="e4m3", causal=False, slots=0),
        # one decoding step's logits of 32 sequences, as the engine holds them, suppressed ids left out
        dict(name="logits_step", op="logits", rows=32, vocab=51866, type="fp16", top=5, masked=True),
        # scoring whole texts from stored fp32 logits, an odd vocabulary (unaligned rows)
        dict(name="logits_texts", op="logits", rows=1792, vocab=51865, type="fp32", top=8, masked=False),
        # the tiny model's next token, one sequence
        dict(name="hidden_one", op="hidden", rows=1, vocab=51865, width=384, top=5, masked=True),
        # a decoding step of large-v3, 32 sequences
        dict(name="hidden_step", op="hidden", rows=32, vocab=51866, width=1280, top=5, masked=True),
        # scoring 32 texts of 224 tokens
        dict(name="hidden_texts", op="hidden", rows=7168, vocab=51866, width=1280, top=5, masked=False),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["step", "write", "attend", "attend", "logits", "hidden", "hidden"])
    kind, block = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64, 128])
    if op == "step":
        cap = rng.randint(16, 1024)
        lo, hi = sorted((rng.randint(1, cap), rng.randint(1, cap)))
        return dict(op=op, batch=log(1, 32), heads=rng.randint(1, 20), cap=cap, lo=lo, hi=hi, block=block, kind=kind)
    if op == "write":
        n = log(1, 1500)
        return dict(op=op, batch=log(1, 32), heads=rng.randint(1, 20), cap=n + rng.choice([0, 0, 7, 100]), n=n,
                    block=block, kind=kind)
    if op == "attend":
        rows = rng.choice([1, 1, 1, rng.randint(2, 16), log(2, 224)])
        batch, heads, group = log(1, 32), rng.randint(1, 20), rng.choice([1, 1, 2, 4])
        cap = log(1, min(131072, max(1, 393216 * 5 // (batch * heads * (1 + rows * group // 32)))))
        lo, hi = sorted((rng.randint(0, cap), rng.randint(max(0, cap // 2), cap)))
        return dict(op=op, batch=batch, rows=rows, heads=heads, group=group, cap=cap, lo=lo, hi=hi, block=block,
                    kind=kind, causal=rng.random() < 0.4, slots=rng.choice([0, 0, 2]) if cap <= 4096 else 0)
    if op == "logits":
        return dict(op=op, rows=log(1, 1792), vocab=log(300, 51866), type=rng.choice(["fp16", "fp32"]),
                    top=rng.randint(0, 8), masked=rng.random() < 0.5)
    return dict(op=op, rows=log(1, 7168), vocab=log(1000, 51866), width=64 * rng.randint(1, 20), top=rng.randint(0, 8),
                masked=rng.random() < 0.5)


def _lens(case):
    """The sequences' lengths, spread evenly between the case's ends (prepare() shuffles them)."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def _codes(shape, kind, gen):
    """Stored values of a cache: the codes of normally distributed numbers whose block maximum is near the type's."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if kind == "int8":
        return (x * 36).round_().clamp_(-127, 127).to(torch.int8)
    return (x * 120).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(shape, kind, gen):
    return (0.5 + torch.rand(shape, generator=gen, device="cuda")) / (36 if kind == "int8" else 120)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    op, dev, f16 = case["op"], "cuda", torch.float16
    if op in ("step", "attend", "write"):
        b, h, cap = case["batch"], case["heads"], case["cap"]
        nb = (cap + case["block"] - 1) // case["block"]
        if op == "write":
            dtype = torch.int8 if case["kind"] == "int8" else torch.float8_e4m3fn
            st["k8"], st["v8"] = (torch.zeros((b, h, cap, HD), dtype=torch.int8, device=dev).view(dtype) for _ in "kv")
            st["ks"], st["vs"] = (torch.zeros((b, h, nb), device=dev) for _ in "kv")
            n = case["n"]
            # heads differ in size, as a model's do; keys and values lie head by head, as the encoder's projection does
            size = 0.25 + 2 * torch.rand((b, 1, h, 1), generator=gen, device=dev)
            k, v = ((torch.randn((b, h, n, HD), generator=gen, device=dev).transpose(1, 2) * size) for _ in "kv")
            st["k"], st["v"] = k.to(f16), v.to(f16)
            st["k_back"], st["v_back"] = (torch.empty((b, n, h, HD), dtype=f16, device=dev) for _ in "kv")
            return st
        st["k8"], st["v8"] = (_codes((b, h, cap, HD), case["kind"], gen) for _ in "kv")
        st["ks"], st["vs"] = (_scales((b, h, nb), case["kind"], gen) for _ in "kv")
        order = torch.randperm(b, generator=gen, device=dev)
        st["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=dev)[order]
        rows, hq = case.get("rows", 1), h * case.get("group", 1)
        if op == "step":
            # one fused projection gives the step's q, k and v, as in the decoder
            qkv = (torch.randn((b, 1, 3 * h, HD), generator=gen, device=dev) * 1.5).to(f16)
            st["q"], st["k"], st["v"] = qkv[:, :, :h], qkv[:, :, h:2 * h], qkv[:, :, 2 * h:]
            st["pos"] = st["lens"] - 1
            st["start"] = st["pos"] // case["block"] * case["block"]
            st["k_back"], st["v_back"] = (torch.empty((b, case["block"], h, HD), dtype=f16, device=dev) for _ in "kv")
        else:
            st["q"] = (torch.randn((b, rows, hq, HD), generator=gen, device=dev) * 1.5).to(f16)
            if case["slots"]:
                slots = min(case["slots"], hq)
                st["pslot"] = torch.full((hq,), -1, dtype=torch.int32, device=dev)
                st["pslot"][torch.randperm(hq, generator=gen, device=dev)[:slots]] = torch.arange(
                    slots, dtype=torch.int32, device=dev)
                st["probs"] = torch.empty((b, slots, rows, cap), dtype=f16, device=dev)
        st["out"] = torch.empty((b, rows, hq, HD), dtype=f16, device=dev)
        return st
    r, vocab, top = case["rows"], case["vocab"], case["top"]
    st["target"] = torch.randint(0, vocab, (r,), generator=gen, device=dev, dtype=torch.int32)
    st["sup"] = None
    if case["masked"]:
        st["sup"] = (torch.rand((vocab,), generator=gen, device=dev) < 0.002).to(torch.uint8)
        st["sup"][vocab // 2] = 0
    if op == "logits":
        x = torch.randn((r, vocab), generator=gen, device=dev) * 2.5
        x.scatter_add_(1, st["target"].long()[:, None], 8 * torch.rand((r, 1), generator=gen, device=dev))
        st["logits"] = x.to(f16 if case["type"] == "fp16" else torch.float32)
    else:
        # hidden states and embedding on grids (multiples of 2^-5 and 2^-10): every partial sum of a product is exact
        # in fp32, so that the order of the alternatives has one answer
        emb = torch.randn((vocab, case["width"]), generator=gen, device=dev) * (1.6 / math.sqrt(case["width"]))
        emb = (emb * 1024).round_() / 1024
        x = torch.randn((r, case["width"]), generator=gen, device=dev)
        x += emb[st["target"].long()] * (6 * torch.rand((r, 1), generator=gen, device=dev))
        st["emb"], st["x"] = emb.to(f16), ((x * 32).round_() / 32).to(f16)
    for name in ("logp", "entropy", "lse"):
        st[name] = torch.empty((r,), dtype=torch.float32, device=dev)
    st["top_id"] = torch.empty((r, top), dtype=torch.int32, device=dev) if top else None
    st["top_logp"] = torch.empty((r, top), dtype=torch.float32, device=dev) if top else None
    return st


# ---------------------------------------------------------------- the plain forms, in 32 bits

def _round_code(x, kind):
    if kind == "int8":
        return x.round().clamp(-127, 127)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).float()


def _plain_write(codes, scales, x, pos, block, kind):
    """codes [b][h][cap][64] and scales [b][h][blocks] after the tokens x [b][n][h][64] went to positions pos[b].."""
    b, h, cap, _ = codes.shape
    n, nb = x.shape[1], scales.shape[2]
    j = torch.arange(cap, device=x.device)
    at = j[None, :] - pos[:, None]                                                   # token of x at position j
    new = ((at >= 0) & (at < n))[:, None, :, None]
    xs = x.float().transpose(1, 2)
    xs = xs.gather(2, at.clamp(0, n - 1)[:, None, :, None].expand(b, h, cap, HD))
    xs = torch.where(new, xs, xs.new_zeros(()))
    blk = j // block
    amax = torch.nn.functional.pad(xs.abs().amax(3), (0, nb * block - cap)).view(b, h, nb, block).amax(3)
    first = torch.arange(nb, device=x.device) * block
    touched = ((first < (pos + n)[:, None]) & (first + block > pos[:, None]))[:, None, :]
    older = (first < pos[:, None])[:, None, :]                                       # the block has earlier tokens
    s = amax / (127.0 if kind == "int8" else 448.0)
    s = torch.where(older, torch.maximum(s, scales), s)
    s = torch.where(touched, s, scales)
    r = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    kept = torch.where(touched & (s != scales), scales * r, torch.ones_like(s))      # factor on earlier codes
    old = codes.float()
    old = torch.where((at < 0)[:, None, :, None], _round_code(old * kept[:, :, blk, None], kind), old)
    return torch.where(new, _round_code(xs * r[:, :, blk, None], kind), old), s


def _plain_values(codes, scales, block):
    return codes.float() * scales[:, :, torch.arange(codes.shape[2], device=codes.device) // block, None]


def _plain_back(values, start, n, lens):
    """values [b][h][cap][64] at positions start[b] .. + n as fp16 [b][n][h][64], zero from position lens[b] on."""
    b, h, cap, _ = values.shape
    at = start[:, None] + torch.arange(n, device=values.device)
    got = values.gather(2, at.clamp(0, cap - 1)[:, None, :, None].expand(b, h, n, HD))
    return torch.where((at < lens[:, None])[:, None, :, None], got, got.new_zeros(())).transpose(1, 2).to(torch.float16)


def _plain_attend(q, k, v, lens, causal):
    """out [b][rows][hq][64] in 32 bits and the probabilities [b][hq][rows][cap], k and v [b][h][cap][64] values."""
    b, rows, hq, _ = q.shape
    h, cap = k.shape[1], k.shape[2]
    qs = q.float().permute(0, 2, 1, 3).reshape(b, h, hq // h * rows, HD)
    s = (torch.matmul(qs, k.transpose(2, 3)) * 0.125).view(b, hq, rows, cap)
    lim = lens.long()[:, None].expand(b, rows)
    if causal:
        lim = (lim - rows + 1 + torch.arange(rows, device=q.device)).clamp(min=0)
    seen = (torch.arange(cap, device=q.device) < lim[:, :, None])[:, None]
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(3, keepdim=True).clamp(min=-3e38)
    e = torch.exp(s - m)
    p = e / e.sum(3, keepdim=True).clamp(min=1e-38)
    v = torch.where((torch.arange(cap, device=q.device) < lens.long()[:, None])[:, None, :, None], v, v.new_zeros(()))
    o = torch.matmul(p.view(b, h, -1, cap), v).view(b, hq, rows, HD)
    return o.permute(0, 2, 1, 3), p


def _plain_logprobs(x, target, sup, top):
    if sup is not None:
        x = x.masked_fill(sup.bool(), -math.inf)
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    l = e.sum(1, keepdim=True)
    lse = (m + torch.log(l))[:, 0]
    entropy = (torch.log(l) - (e * torch.where(e > 0, d, torch.zeros_like(d))).sum(1, keepdim=True) / l)[:, 0]
    logp = x.gather(1, target.long()[:, None])[:, 0] - lse
    out = dict(logp=logp, entropy=entropy, lse=lse)
    if top:
        # value and id in one integer that orders as (value, lower id first): no two are equal
        u = (x + 0.0).view(torch.int32)
        u = torch.where(u < 0, u ^ 0x7FFFFFFF, u).long()
        key = (u << 32) | (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
        key = torch.topk(key, top, dim=1, sorted=True).values
        ids = 0xFFFFFFFF - (key & 0xFFFFFFFF)
        out |= dict(top_id=ids.to(torch.int32), top_logp=x.gather(1, ids) - lse[:, None])
    return out


def run(state):
    s = state
    op = s["op"]
    if own:
        import mimizuku_b200 as m
        if op in ("write", "step"):
            cache = (s["k8"], s["v8"], s["ks"], s["vs"])
            m.kv8_write(s["k"], s["v"], *cache, block=s["block"], pos=s.get("pos"))
            if op == "step":
                m.attn8(s["q"], *cache, s["out"], block=s["block"], lens=s["lens"])
            m.kv8_read(*cache, s["k_back"], s["v_back"], block=s["block"], pos=s.get("start"),
                       lens=s.get("lens"))
            got = dict(k=s["k_back"], v=s["v_back"], ks=s["ks"], vs=s["vs"])
            return got | dict(out=s["out"]) if op == "step" else got
        if op == "attend":
            m.attn8(s["q"], s["k8"], s["v8"], s["ks"], s["vs"], s["out"], block=s["block"], lens=s["lens"],
                    causal=s["causal"], probs=s.get("probs"), pslot=s.get("pslot"))
            return dict(out=s["out"], probs=s["probs"]) if "probs" in s else dict(out=s["out"])
        more = dict(entropy=s["entropy"], lse=s["lse"], top_id=s["top_id"], top_logp=s["top_logp"], sup=s["sup"])
        if op == "logits":
            m.token_logprobs(s["logits"], s["target"], s["logp"], **more)
        else:
            m.linear_logprobs(s["x"], s["emb"], s["target"], s["logp"], **more)
        return {n: s[n] for n in ("logp", "entropy", "lse", "top_id", "top_logp") if s[n] is not None}
    if op in ("write", "step"):
        b = s["batch"]
        pos = s["pos"].long() if "pos" in s else torch.zeros((b,), dtype=torch.int64, device=s["k"].device)
        start = s["start"].long() if "start" in s else pos
        kc, ks = _plain_write(s["k8"], s["ks"], s["k"], pos, s["block"], s["kind"])
        vc, vs = _plain_write(s["v8"], s["vs"], s["v"], pos, s["block"], s["kind"])
        k, v = _plain_values(kc, ks, s["block"]), _plain_values(vc, vs, s["block"])
        n = s["k_back"].shape[1]
        lens = s["lens"] if "lens" in s else pos + n
        got = dict(k=_plain_back(k, start, n, lens), v=_plain_back(v, start, n, lens), ks=ks, vs=vs)
        if op == "step":
            got["out"] = _plain_attend(s["q"], k, v, s["lens"], False)[0].to(torch.float16)
        return got
    if op == "attend":
        k, v = _plain_values(s["k8"], s["ks"], s["block"]), _plain_values(s["v8"], s["vs"], s["block"])
        out, p = _plain_attend(s["q"], k, v, s["lens"], s["causal"])
        if "probs" not in s:
            return dict(out=out.to(torch.float16))
        heads = s["pslot"].argsort()[-s["probs"].shape[1]:]
        return dict(out=out.to(torch.float16), probs=p[:, heads].to(torch.float16))
    x = s["logits"].float() if op == "logits" else torch.matmul(s["x"].float(), s["emb"].float().t())
    return _plain_logprobs(x, s["target"], s["sup"], s["top"])


def work(case):
    op = case["op"]
    if op == "write":
        n = case["batch"] * case["heads"] * case["n"] * HD * 2
        blocks = case["batch"] * case["heads"] * -(-case["n"] // case["block"]) * 2
        return dict(bytes=n * (2 + 1 + 1 + 2) + blocks * 8, flops=n * 3)
    if op in ("step", "attend"):
        h, rows, group, block = case["heads"], case.get("rows", 1), case.get("group", 1), case["block"]
        lens = _lens(case)
        tokens = sum(lens) * h
        lim = [max(0, L - rows + 1 + i) if case.get("causal") else L for L in lens for i in range(rows)]
        pairs = sum(lim) * h * group
        b = tokens * HD * 2 + sum(-(-L // block) for L in lens) * h * 8
        b += case["batch"] * rows * h * group * HD * 4
        b += case["batch"] * min(case.get("slots", 0), h * group) * rows * case["cap"] * 2
        if op == "step":  # the new token's k and v, its codes, and the block read back
            b += case["batch"] * h * HD * 2 * (2 + 1) + case["batch"] * h * block * HD * 2 * 3
        return dict(bytes=b, flops=pairs * HD * 4)
    r, vocab, top = case["rows"], case["vocab"], case["top"]
    out = r * (4 + 12 + 8 * top) + (vocab if case["masked"] else 0)
    if op == "logits":
        return dict(bytes=r * vocab * (2 if case["type"] == "fp16" else 4) + out, flops=r * vocab * 6)
    return dict(bytes=(r + vocab) * case["width"] * 2 + out, flops=2 * r * vocab * case["width"])


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_write(st, name, pos):
    """The written cache's values in 64 bits and its scales: block by block, as the definition has it."""
    x, codes, scales = st[name].double(), st[name + "8"].double(), st[name + "s"].double().clone()
    block, cap, top = st["block"], codes.shape[2], 127.0 if st["kind"] == "int8" else 448.0

    def snap(t):
        if st["kind"] == "int8":
            return t.round().clamp(-127, 127)
        # three mantissa bits, exponents down to 2^-6, to even
        e = torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6)))
        return (torch.round(t / 2 ** (e - 3)) * 2 ** (e - 3)).clamp(-448, 448)

    values = codes * scales.repeat_interleave(block, 2)[:, :, :cap, None]
    for i in range(x.shape[0]):
        p, n = int(pos[i]), x.shape[1]
        for c in range(p // block, (p + n - 1) // block + 1):
            j0, j1 = max(p, c * block), min(p + n, (c + 1) * block, cap)
            part = x[i, j0 - p:j1 - p].transpose(0, 1)
            s = part.abs().amax((1, 2)) / top
            if c * block < p:
                s = torch.maximum(s, scales[i, :, c])
                f = (scales[i, :, c] / s)[:, None, None]
                values[i, :, c * block:p] = torch.where(f < 1, snap(codes[i, :, c * block:p] * f),
                                                        codes[i, :, c * block:p]) * s[:, None, None]
            values[i, :, j0:j1] = snap(part / s[:, None, None]) * s[:, None, None]
            scales[i, :, c] = s
    return values, scales


def _exact_attend(q, k, v, lens, causal):
    b, rows, hq, _ = q.shape
    h, cap = k.shape[1], k.shape[2]
    out = torch.zeros((b, rows, hq, HD), dtype=torch.float64, device=q.device)
    p = torch.zeros((b, hq, rows, cap), dtype=torch.float64, device=q.device)
    for i in range(b):
        n = int(lens[i])
        for c in range(h):
            if not n:
                continue
            at = slice(c * (hq // h), (c + 1) * (hq // h))
            s = torch.einsum("rgd,jd->grj", q[i, :, at].double(), k[i, c, :n].double()) / 8
            if causal:
                last = n - rows + torch.arange(rows, device=q.device)
                s = s.masked_fill(torch.arange(n, device=q.device) > last[:, None], -math.inf)
            w = torch.nan_to_num(torch.softmax(s, 2), nan=0.0)
            p[i, at, :, :n] = w
            out[i, :, at] = torch.einsum("grj,jd->rgd", w, v[i, c, :n].double())
    return out, p


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("write", "step"):
        pos = st["pos"].tolist() if op == "step" else [0] * case["batch"]
        start = st["start"].tolist() if op == "step" else pos
        got = {}
        for name in "kv":
            values, got[name + "s"] = _exact_write(st, name, pos)
            n = st[name + "_back"].shape[1]
            back = torch.zeros((case["batch"], n, case["heads"], HD), dtype=torch.float64, device=values.device)
            for i, p in enumerate(start):
                end = min(p + n, int(st["lens"][i]) if op == "step" else case["cap"])
                back[i, :end - p] = values[i, :, p:end].transpose(0, 1)
            got[name], st[name + "_values"] = back, values
        if op == "step":
            got["out"] = _exact_attend(st["q"], st["k_values"], st["v_values"], st["lens"], False)[0]
        return got
    if op == "attend":
        k, v = (st[n + "8"].double() * st[n + "s"].double().repeat_interleave(case["block"], 2)[:, :, :case["cap"], None]
                for n in "kv")
        out, p = _exact_attend(st["q"], k, v, st["lens"], case["causal"])
        if "probs" not in st:
            return dict(out=out)
        probs = torch.zeros(st["probs"].shape, dtype=torch.float64, device=out.device)
        for head, slot in enumerate(st["pslot"].tolist()):
            if slot >= 0:
                probs[:, slot] = p[:, head]
        return dict(out=out, probs=probs)
    top, got = case["top"], {"logp": [], "entropy": [], "lse": [], "top_logp": []}
    for i in range(0, case["rows"], 512):
        if op == "logits":
            x = st["logits"][i:i + 512].double()
        else:
            x = st["x"][i:i + 512].double() @ st["emb"].double().t()
        if st["sup"] is not None:
            x[:, st["sup"] != 0] = -math.inf
        lp = torch.log_softmax(x, 1)
        got["lse"].append(torch.logsumexp(x, 1))
        got["logp"].append(lp.gather(1, st["target"][i:i + 512].long()[:, None])[:, 0])
        got["entropy"].append(torch.special.entr(lp.exp()).sum(1))
        got["top_logp"].append(lp.sort(dim=1, descending=True).values[:, :top].contiguous())
    got = {n: torch.cat(v) for n, v in got.items()}
    if not top:
        del got["top_logp"]
    else:
        got["top_id"] = None
    return got
