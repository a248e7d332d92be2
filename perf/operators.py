"""Cases of the decode-step operators: what they compute and how large it is.

Three operators of a decoder layer are described here, each in a plain form of
elementary torch operations and as the call a user makes:

  norm_rope_append  RMS norm of every q and k head, rotation at the token's
                    position, and the K/V append into the paged cache
  shared_decode     one decode step of a batch whose sequences share a prefix,
                    the prefix read once for the whole batch
  w4_linear         x W^T for a few tokens, W in 4 bits with a scale (and
                    optionally a zero point) for every group of inputs

``own`` selects the call (True) or the plain form (False).  ``exact`` holds the
same results from the definitions in 64 bits.
"""
import math

import torch

own = False

BLOCK = 64  # positions per cache block
DEV = "cuda"


# ------------------------------------------------------------------ the cases

def _append(name, tokens, q_heads, kv_heads, head_dim=128, dtype="float16", packed=True,
            prompt=True, start=0, max_pos=512):
    return dict(name=name, op="norm_rope_append", tokens=tokens, q_heads=q_heads,
                kv_heads=kv_heads, head_dim=head_dim, dtype=dtype, packed=packed, prompt=prompt,
                start=start, max_pos=max_pos)


def _shared(name, seqs, q_heads, kv_heads, prefix, suffix_min, suffix_max):
    return dict(name=name, op="shared_decode", seqs=seqs, q_heads=q_heads, kv_heads=kv_heads,
                prefix=prefix, suffix_min=suffix_min, suffix_max=suffix_max)


def _linear(name, tokens, inputs, outputs, group, zeros, bias):
    return dict(name=name, op="w4_linear", tokens=tokens, inputs=inputs, outputs=outputs,
                group=group, zeros=zeros, bias=bias)


def listed():
    return [
        # one sequence decoding: the step's latency counts
        _append("append_1x28x4", 1, 28, 4, prompt=False, max_pos=2048),
        # a decode batch, every token at its own position of its own sequence
        _append("append_64x32x8", 64, 32, 8, prompt=False, max_pos=512),
        # a ragged fp32 prompt chunk with separate q, k, v and a head size that is no power of two
        _append("append_f32_1000x20x5x80", 1000, 20, 5, head_dim=80, dtype="float32",
                packed=False, start=77),
        # a long prompt chunk behind an earlier one
        _append("append_8192x32x8", 8192, 32, 8, start=4096),
        # a few chats behind a short system prompt
        _shared("shared_8x2048_28x4", 8, 28, 4, 2048, 1, 160),
        # every head its own K/V (MHA), lengths that end inside blocks
        _shared("shared_33x5001_32x32", 33, 32, 32, 5001, 0, 333),
        # a serving batch behind a long prompt with examples
        _shared("shared_64x8192_32x8", 64, 32, 8, 8192, 1, 512),
        # a batch of questions about one long document
        _shared("shared_64x32768_32x8", 64, 32, 8, 32768, 1, 1024),
        # the joint q/k/v projection of one decoding sequence
        _linear("w4_1x4096x6144", 1, 4096, 6144, 128, False, False),
        # gate and up projections of one decoding sequence, small groups with zero points
        _linear("w4_1x3584x37888_g64", 1, 3584, 37888, 64, True, False),
        # a down projection for an odd number of tokens and outputs
        _linear("w4_17x11008x4099", 17, 11008, 4099, 128, False, True),
        # the widest projection of a large model for a decode batch
        _linear("w4_8x8192x28672", 8, 8192, 28672, 128, True, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope_append", "shared_decode", "w4_linear"])
    top = {}
    for c in listed():
        w = work(c)
        t = top.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for key in t:
            t[key] = max(t[key], w[key])
    while True:
        if op == "norm_rope_append":
            kv = rng.choice([1, 2, 4, 5, 8, 16])
            prompt = rng.random() < 0.6
            case = _append(None, _log(rng, 1, 8192) if prompt else _log(rng, 1, 128),
                           kv * rng.choice([1, 2, 3, 4, 7, 8]), kv,
                           rng.choice([64, 80, 96, 128, 192, 256]),
                           rng.choice(["float16", "float16", "float32"]), rng.random() < 0.6,
                           prompt, rng.randrange(0, 4097), _log(rng, 16, 256))
        elif op == "shared_decode":
            kv = rng.choice([1, 2, 4, 8, 16, 32])
            lo = rng.randrange(0, 3)
            case = _shared(None, _log(rng, 1, 96), kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), kv,
                           _log(rng, 16, 32768), lo, lo + _log(rng, 1, 1024))
        else:
            group = rng.choice([32, 64, 128])
            case = _linear(None, _log(rng, 1, 32), group * max(1, _log(rng, 256, 14336) // group),
                           _log(rng, 64, 37888), group, rng.random() < 0.5, rng.random() < 0.5)
        w = work(case)
        if all(w[key] <= top[op][key] for key in w):
            del case["name"]
            return case


def work(case):
    if case["op"] == "norm_rope_append":
        n, hq, hkv, hd = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
        es = 2 if case["dtype"] == "float16" else 4
        rows = n if case["prompt"] else min(n, case["max_pos"])  # table rows
        return {"bytes": n * ((2 * hq + 2 * hkv) * hd * es + 2 * hkv * hd * 2) + rows * hd * 4,
                "flops": n * (hq + hkv) * hd * 7}
    if case["op"] == "shared_decode":
        s, hq, hkv, p = case["seqs"], case["q_heads"], case["kv_heads"], case["prefix"]
        suffix = s * (case["suffix_min"] + case["suffix_max"]) // 2
        return {"bytes": 4 * 128 * hkv * (p + suffix) + 4 * 128 * s * hq,
                "flops": 4 * 128 * hq * (s * p + suffix)}
    n, k, o, g = case["tokens"], case["inputs"], case["outputs"], case["group"]
    groups = o * (k // g)
    return {"bytes": o * k // 2 + 2 * groups + (groups // 2 if case["zeros"] else 0)
            + 2 * n * (k + o) + (2 * o if case["bias"] else 0),
            "flops": 2 * n * k * o}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=torch.float16):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _append_inputs(case, seed):
    g = _gen(seed)
    n, hq, hkv, hd = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"]
    dt = getattr(torch, case["dtype"])
    # projections have heads of unlike size and a few large channels
    chan = torch.exp(0.5 * torch.randn((hq + 2 * hkv) * hd, generator=g, device=DEV))
    qkv = (torch.randn((n, (hq + 2 * hkv) * hd), generator=g, device=DEV) * chan).to(dt)
    q, k, v = qkv.split([hq * hd, hkv * hd, hkv * hd], dim=1)
    if not case["packed"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if case["prompt"]:
        lengths, blocks = [case["start"] + n], _blocks(case["start"] + n)
        seq_ids = torch.zeros(n, dtype=torch.int32, device=DEV)
        positions = torch.arange(case["start"], case["start"] + n, dtype=torch.int32, device=DEV)
    else:
        lengths = (1 + torch.randint(0, case["max_pos"], (n,), generator=g, device=DEV)).tolist()
        blocks = n * _blocks(case["max_pos"])  # a pool that holds the batch at its longest
        seq_ids = torch.arange(n, dtype=torch.int32, device=DEV)
        positions = torch.tensor(lengths, dtype=torch.int32, device=DEV) - 1
    pos = torch.arange(max(lengths), dtype=torch.float64, device=DEV)
    freq = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    angle = pos[:, None] * freq
    return dict(q=q, k=k, v=v, seq_ids=seq_ids, positions=positions, lengths=lengths,
                blocks=blocks,
                qw=(1 + 0.2 * torch.randn(hd, generator=g, device=DEV)).to(dt),
                kw=(1 + 0.2 * torch.randn(hd, generator=g, device=DEV)).to(dt),
                cos=angle.cos().float(), sin=angle.sin().float(), eps=1e-6)


def _shared_inputs(case, seed):
    g = _gen(seed)
    s, hq, hkv, p = case["seqs"], case["q_heads"], case["kv_heads"], case["prefix"]
    suffix = torch.randint(case["suffix_min"], case["suffix_max"] + 1, (s,), generator=g,
                           device=DEV)
    ms = max(1, int(suffix.max()))
    # keys have an offset per channel, as they do behind a rotation
    off = torch.randn((hkv, 128), generator=g, device=DEV)
    kp = (torch.randn((p, hkv, 128), generator=g, device=DEV) + off).half()
    ks = (torch.randn((s, ms, hkv, 128), generator=g, device=DEV) + off).half()
    return dict(q=_randn(g, s, hq * 128, scale=2.0), kp=kp, vp=_randn(g, p, hkv, 128), ks=ks,
                vs=_randn(g, s, ms, hkv, 128), suffix=suffix, scale=128 ** -0.5)


def _linear_inputs(case, seed):
    g = _gen(seed)
    n, k, o, gs = case["tokens"], case["inputs"], case["outputs"], case["group"]
    codes = torch.empty((o, k), dtype=torch.uint8, device=DEV)
    for r in range(0, o, 4096):  # codes of normal weights
        part = torch.randn((min(4096, o - r), k), generator=g, device=DEV)
        codes[r:r + 4096] = (part * 2.7 + 8).round().clamp(0, 15).to(torch.uint8)
    scales = (0.004 + 0.008 * torch.rand((o, k // gs), generator=g, device=DEV)).half()
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(6, 11, (o, k // gs), generator=g, device=DEV, dtype=torch.uint8)
    return dict(x=_randn(g, n, k), codes=codes, scales=scales, zeros=zeros, group=gs,
                bias=_randn(g, o, scale=0.1) if case["bias"] else None)


def prepare(case, seed):
    if case["op"] == "norm_rope_append":
        st = _append_inputs(case, seed)
        hkv, hd, lengths = case["kv_heads"], case["head_dim"], st["lengths"]
        if own:
            from hxinfer_b200.kv import KVCache, RopeTable
            st["cache"] = KVCache(1, hkv, hd, len(lengths), max(lengths), st["blocks"])
            for s, n in enumerate(lengths):
                st["cache"].reserve(s, n)
            st["table"] = RopeTable.from_values(st.pop("cos"), st.pop("sin"))
            st["q_out"] = torch.empty((case["tokens"], case["q_heads"] * hd),
                                      dtype=st["q"].dtype, device=DEV)
        else:
            first = [0]
            for n in lengths:
                first.append(first[-1] + _blocks(n))
            st["first"] = torch.tensor(first, device=DEV)
            st["pool"] = torch.zeros((1, 2, st["blocks"], hkv, BLOCK, hd),
                                     dtype=torch.float16, device=DEV)
    elif case["op"] == "shared_decode":
        st = _shared_inputs(case, seed)
        if own:
            from hxinfer_b200.kv import KVCache
            s, hkv, p = case["seqs"], case["kv_heads"], case["prefix"]
            suffix = st["suffix"].tolist()
            cap = p + max(suffix)
            cache = KVCache(1, hkv, 128, s + 1, cap,
                            _blocks(p) + sum(1 + _blocks(n) for n in suffix))
            cache.reserve(s, p)
            cache.write(0, s, 0, st.pop("kp"), st.pop("vp"))
            for i, n in enumerate(suffix):
                cache.share(i, s, p)
                cache.reserve(i, p + n)
                if n:
                    cache.write(0, i, p, st["ks"][i, :n], st["vs"][i, :n])
            del st["ks"], st["vs"]
            st["cache"], st["prefix_seq"], st["prefix_len"] = cache, s, p
            st["seq_ids"] = torch.arange(s, dtype=torch.int32, device=DEV)
            st["lengths"] = (st["suffix"] + p).to(torch.int32)
            st["workspace"] = torch.zeros(
                cache.shared_workspace_bytes(s, case["q_heads"], p), dtype=torch.uint8, device=DEV)
            st["out"] = torch.empty_like(st["q"])
    else:
        st = _linear_inputs(case, seed)
        if own:
            from hxinfer_b200.w4 import W4Weight
            st["weight"] = W4Weight(st.pop("codes"), st.pop("scales"), st.pop("zeros"))
            st["out"] = torch.empty((case["tokens"], case["outputs"]), dtype=torch.float16,
                                    device=DEV)
    st["case"] = case
    return st


# ------------------------------------------------------------------ one pass

def run(st):
    case = st["case"]
    if case["op"] == "norm_rope_append":
        return _run_append(st, case)
    if case["op"] == "shared_decode":
        return _run_shared(st, case)
    return _run_linear(st)


def _run_append(st, case):
    if own:
        st["cache"].norm_rope_append(0, st["q"], st["k"], st["v"], st["seq_ids"], st["positions"],
                                     case["q_heads"], q_weight=st["qw"], k_weight=st["kw"],
                                     eps=st["eps"], table=st["table"], q_out=st["q_out"])
        return st["q_out"], st["cache"].pool()
    hd, hkv = case["head_dim"], case["kv_heads"]
    pos, pool = st["positions"].long(), st["pool"]
    c, s = st["cos"][pos][:, None], st["sin"][pos][:, None]

    def norm_rotate(x, w):
        x = x.float().unflatten(1, (-1, hd))
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + st["eps"]) * w.float()
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    block = st["first"][st["seq_ids"].long()] + pos // BLOCK
    pool[0, 0, block, :, pos % BLOCK] = norm_rotate(st["k"], st["kw"]).half()
    pool[0, 1, block, :, pos % BLOCK] = st["v"].unflatten(1, (hkv, hd)).half()
    return norm_rotate(st["q"], st["qw"]).flatten(1).to(st["q"].dtype), pool


def _run_shared(st, case):
    if own:
        return st["cache"].decode_shared(0, st["q"], st["seq_ids"], st["lengths"], case["q_heads"],
                                         prefix_seq=st["prefix_seq"], prefix_len=st["prefix_len"],
                                         scale=st["scale"], out=st["out"],
                                         workspace=st["workspace"])
    s, hq, hkv, p = case["seqs"], case["q_heads"], case["kv_heads"], case["prefix"]
    g = hq // hkv
    q = st["q"].float().view(s, hkv, g, 128) * st["scale"]
    dead = torch.arange(st["ks"].shape[1], device=DEV) >= st["suffix"][:, None]
    out = torch.empty((s, hkv, g, 128), device=DEV)
    for h in range(hkv):
        kp, vp = st["kp"][:, h].float(), st["vp"][:, h].float()
        ks, vs = st["ks"][:, :, h].float(), st["vs"][:, :, h].float()
        a = (q[:, h].reshape(s * g, 128) @ kp.T).view(s, g, p)
        b = (q[:, h] @ ks.transpose(1, 2)).masked_fill(dead[:, None], -math.inf)
        m = torch.maximum(a.amax(-1, keepdim=True), b.amax(-1, keepdim=True))
        a, b = torch.exp(a - m), torch.exp(b - m)
        num = (a.view(s * g, p) @ vp).view(s, g, 128) + b @ vs
        out[:, h] = num / (a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True))
    return out.view(s, hq * 128).half()


def _run_linear(st):
    if own:
        from hxinfer_b200.w4 import w4_linear
        return w4_linear(st["x"], st["weight"], bias=st["bias"], out=st["out"])
    o, k = st["codes"].shape
    w = st["codes"].float().view(o, -1, st["group"])
    zero = 8.0 if st["zeros"] is None else st["zeros"].float()[..., None]
    w = (w - zero) * st["scales"].float()[..., None]
    y = st["x"].float() @ w.view(o, k).T
    if st["bias"] is not None:
        y = y + st["bias"].float()
    return y.half()


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    if case["op"] == "norm_rope_append":
        st = _append_inputs(case, seed)
        hq, hkv, hd, half = case["q_heads"], case["kv_heads"], case["head_dim"], case["head_dim"] // 2
        pos = st["positions"].long()
        turn = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, None]

        def rotated(x, heads, w):
            x = x.double().view(len(pos), heads, hd)
            rms = torch.sqrt(x.square().sum(-1) / hd + st["eps"])
            x = x * w.double() / rms[..., None]
            z = torch.complex(x[..., :half], x[..., half:]) * turn
            return torch.cat((z.real, z.imag), -1)

        pool = torch.zeros((1, 2, st["blocks"], hkv, BLOCK, hd), dtype=torch.float64, device=DEV)
        base, starts = 0, []
        for n in st["lengths"]:
            starts.append(base)
            base += _blocks(n) * BLOCK
        slot = torch.tensor(starts, device=DEV)[st["seq_ids"].long()] + pos
        k, v = rotated(st["k"], hkv, st["kw"]), st["v"].double().view(len(pos), hkv, hd)
        for which, rows in ((0, k), (1, v)):
            flat = pool[0, which].transpose(1, 2).reshape(-1, hkv, hd)
            flat[slot] = rows
            pool[0, which] = flat.view(-1, BLOCK, hkv, hd).transpose(1, 2)
        return rotated(st["q"], hq, st["qw"]).reshape(len(pos), hq * hd), pool
    if case["op"] == "shared_decode":
        st = _shared_inputs(case, seed)
        s, hq, hkv = case["seqs"], case["q_heads"], case["kv_heads"]
        out = torch.empty((s, hkv, hq // hkv, 128), dtype=torch.float64, device=DEV)
        q = st["q"].double().view(s, hkv, hq // hkv, 128)
        for h in range(hkv):
            kp, vp = st["kp"][:, h].double(), st["vp"][:, h].double()
            for i, n in enumerate(st["suffix"].tolist()):
                keys = torch.cat((kp, st["ks"][i, :n, h].double()))
                vals = torch.cat((vp, st["vs"][i, :n, h].double()))
                out[i, h] = torch.softmax(q[i, h] @ keys.T * st["scale"], -1) @ vals
        return out.view(s, hq * 128)
    st = _linear_inputs(case, seed)
    gs, x = st["group"], st["x"].double()
    y = torch.zeros((case["tokens"], case["outputs"]), dtype=torch.float64, device=DEV)
    for i in range(case["inputs"] // gs):  # y = sum over groups of s (q . x - z sum x)
        part = x[:, i * gs:(i + 1) * gs]
        dot = part @ st["codes"][:, i * gs:(i + 1) * gs].double().T
        zero = 8.0 if st["zeros"] is None else st["zeros"][:, i].double()
        y += (dot - part.sum(1, keepdim=True) * zero) * st["scales"][:, i].double()
    return y if st["bias"] is None else y + st["bias"].double()
