"""Performance cases of the 4-bit KV cache's operators: what a program that
serves sequences over such a cache has them do.

Kinds of case (each over a batch of sequences whose cache rows lie in pages):
  prep    q and k heads normalised and rotated at their tokens' positions
  store   new tokens' k and v quantised into the cache, and their rows read back
  read    whole sequences' rows read back out of the cache
  attn    causal attention of the last tokens of each sequence over its cache,
          optionally gated by sigmoid(gate)

The cache: K and V each are n_pages pages; a page holds, for each kv head,
page_rows rows of codes (hd / 2 bytes: byte 16 b + i of a row holds element
32 b + i in its low and 32 b + 16 + i in its high four bits), then page_rows
rows of hd / 32 f16 scales.  Element = scale * (code - 8), the values of
ggml's Q4_0 with magnitudes up to 65504.

With `own` false `run` computes all of it with elementary torch operations in
32 bits; with `own` true it calls the library's entry points.
"""
import ctypes as C
import math
import os
import random
import sys

import numpy as np
import torch

own = False

PKG = os.path.join(os.getcwd(), "sinter-qwen36-nomtp-tu102_amd")
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
# the 27B hybrid's rotary dimensions and base (sinter.qwen36_27b_config)
ROPE, BASE = 64, 1e7


def listed():
    return [
        # one token of one reply on the 27B hybrid's attention heads: the
        # shortest call, all latency
        {"name": "prep_reply", "kind": "prep", "type": "f32", "nq": 24, "nkv": 4, "hd": 256, "page": 64,
         "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 4097, "past_hi": 4097, "gate": True},
        # ubatches of three prompts far into long documents
        {"name": "prep_prompts_far", "kind": "prep", "type": "bf16", "nq": 24, "nkv": 4, "hd": 256, "page": 64,
         "seqs": 3, "new_lo": 300, "new_hi": 1300, "past_lo": 60000, "past_hi": 120000, "gate": False},
        # one new token of each of 48 replies
        {"name": "store_replies_48", "kind": "store", "type": "f32", "nq": 24, "nkv": 4, "hd": 256, "page": 64,
         "seqs": 48, "new_lo": 1, "new_hi": 1, "past_lo": 100, "past_hi": 9000, "gate": False},
        # two prompts, small pages, the middle head size
        {"name": "store_prompts", "kind": "store", "type": "bf16", "nq": 32, "nkv": 8, "hd": 128, "page": 16,
         "seqs": 2, "new_lo": 3000, "new_hi": 5000, "past_lo": 0, "past_hi": 77, "gate": False},
        # one sequence taken out of the cache, e.g. to keep it elsewhere
        {"name": "read_sequence_8k", "kind": "read", "type": "f16", "nq": 24, "nkv": 4, "hd": 256, "page": 256,
         "seqs": 1, "new_lo": 8191, "new_hi": 8191, "past_lo": 0, "past_hi": 0, "gate": False},
        # many short ones of a model with a kv head per q head
        {"name": "read_sequences_20", "kind": "read", "type": "f32", "nq": 16, "nkv": 16, "hd": 64, "page": 32,
         "seqs": 20, "new_lo": 1, "new_hi": 2900, "past_lo": 0, "past_hi": 0, "gate": False},
        # the first tokens of a reply to a short question
        {"name": "attn_reply_300", "kind": "attn", "type": "f32", "nq": 24, "nkv": 4, "hd": 256, "page": 64,
         "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 299, "past_hi": 299, "gate": True},
        # one token of a reply at the end of a very long document
        {"name": "attn_reply_128k", "kind": "attn", "type": "f32", "nq": 24, "nkv": 4, "hd": 256, "page": 1024,
         "seqs": 1, "new_lo": 1, "new_hi": 1, "past_lo": 131000, "past_hi": 131000, "gate": True},
        # one token of each of 64 replies of very different lengths
        {"name": "attn_replies_64", "kind": "attn", "type": "bf16", "nq": 24, "nkv": 4, "hd": 256, "page": 64,
         "seqs": 64, "new_lo": 1, "new_hi": 1, "past_lo": 200, "past_hi": 16000, "gate": False},
        # four drafted tokens of each of eight sequences checked at once
        {"name": "attn_verify_8x4", "kind": "attn", "type": "f16", "nq": 32, "nkv": 8, "hd": 128, "page": 16,
         "seqs": 8, "new_lo": 4, "new_hi": 4, "past_lo": 2000, "past_hi": 9000, "gate": False},
        # two prompts from their first token
        {"name": "attn_prompts_2k", "kind": "attn", "type": "bf16", "nq": 24, "nkv": 4, "hd": 256, "page": 64,
         "seqs": 2, "new_lo": 1900, "new_hi": 2200, "past_lo": 0, "past_hi": 0, "gate": False},
        # a later turn of a long chat
        {"name": "attn_turn_32k", "kind": "attn", "type": "f32", "nq": 24, "nkv": 4, "hd": 256, "page": 256,
         "seqs": 1, "new_lo": 500, "new_hi": 500, "past_lo": 32000, "past_hi": 32000, "gate": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prep", "store", "read", "attn", "attn", "attn"])
    nq, nkv, hd = rng.choice([(24, 4, 256), (24, 4, 256), (16, 2, 256), (32, 8, 128), (28, 4, 128), (8, 8, 128),
                              (16, 16, 64), (12, 1, 64), (40, 2, 64)])
    case = {"kind": kind, "type": rng.choice(["f32", "f16", "bf16"]), "nq": nq, "nkv": nkv, "hd": hd,
            "page": rng.choice([16, 32, 64, 256, 1024]), "gate": rng.random() < 0.5, "lens": rng.randrange(1 << 30)}
    if kind in ("prep", "store"):
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 8000 // seqs))
        past = _log(rng, 1, 20000)
        case |= {"seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "past_lo": past // 3, "past_hi": past}
    elif kind == "read":
        seqs = _log(rng, 1, 40)
        hi = _log(rng, 1, 30000 // seqs)
        case |= {"seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "past_lo": 0, "past_hi": 0}
    elif rng.random() < 0.6:   # replies, drafted tokens
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 8, min(131000, 500000 // seqs))
        new = rng.choice([1, 1, 1, 2, 3, 5])
        case |= {"seqs": seqs, "new_lo": 1 if rng.random() < 0.5 else new, "new_hi": new,
                 "past_lo": hi // rng.choice([1, 2, 50]), "past_hi": hi}
    else:                      # prompts, later turns
        seqs = rng.choice([1, 1, 2, 3, 5])
        hi = _log(rng, 8, 2000 // seqs)
        past = rng.choice([0, 0, _log(rng, 1, min(32000, 14_000_000 // (seqs * hi)))])
        case |= {"seqs": seqs, "new_lo": rng.randint(1, hi), "new_hi": hi, "past_lo": past // 2, "past_hi": past}
    return case


def _lens(case):
    """The new tokens and the rows before them of each sequence."""
    rng = random.Random(case.get("lens", 5))
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    past = [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    return new, past


# ---------------------------------------------------------------- the cache in torch

def _quantise(x):
    """Codes (uint8, one an element) and f16 scales of x [..., hd], f32."""
    xb = x.reshape(*x.shape[:-1], -1, 32).clamp(-65504.0, 65504.0)
    top = xb.abs().argmax(-1, keepdim=True)          # (the first of equal ones)
    d = torch.gather(xb, -1, top) / -8.0
    d16 = d.half()
    inv = torch.where(d16 != 0, 1.0 / d, torch.zeros_like(d))
    q = (xb * inv + 8.5).to(torch.int32).clamp(0, 15).to(torch.uint8)
    return q, torch.where(d16 != 0, d16, torch.zeros_like(d16)).squeeze(-1)


def _planes(st, cache):
    """Views of a cache's codes [pages, nkv, rows, hd / 2] and scales [pages, nkv, rows, hd / 32]."""
    c = st["case"]
    rows, hd, nkv = c["page"], c["hd"], c["nkv"]
    per = cache.view(-1, nkv, rows * (hd // 2 + hd // 16))
    codes = per[..., :rows * hd // 2].view(-1, nkv, rows, hd // 2)
    return codes, per[..., rows * hd // 2:].view(torch.float16).view(-1, nkv, rows, hd // 32)


def _write(st, cache, x, page, row):
    """Quantise x [n, nkv, hd] into rows `row` of pages `page`."""
    codes, scales = _planes(st, cache)
    q, d = _quantise(x)
    packed = q[..., :16] | (q[..., 16:] << 4)
    codes[page, :, row] = packed.reshape(*packed.shape[:2], -1)
    scales[page, :, row] = d


def _values(st, cache, page, row):
    """The f32 values [n, nkv, hd] of rows `row` of pages `page`."""
    codes, scales = _planes(st, cache)
    b = codes[page, :, row]
    b = b.view(*b.shape[:2], -1, 16)
    q = torch.cat([b & 15, b >> 4], -1).to(torch.float32) - 8.0
    return (q * scales[page, :, row].float().unsqueeze(-1)).reshape(*b.shape[:2], -1)


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    new, past = _lens(case)
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["type"]]
    nq, nkv, hd, rows, n_seq = case["nq"], case["nkv"], case["hd"], case["page"], case["seqs"]
    total = [n + p for n, p in zip(new, past)]
    n_tok = sum(new)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    st = {"case": case, "new": new, "past": past, "n_tok": n_tok}
    st["tok_start"] = torch.tensor([sum(new[:i]) for i in range(n_seq + 1)], dtype=torch.int32, device="cuda")
    st["kv_len"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(p, t, device="cuda") for p, t in zip(past, total)])
    seq = torch.cat([torch.full((n,), s, device="cuda") for s, n in enumerate(new)])
    st["pos"], st["seq"] = pos, seq
    # a few heads' channels are much larger than the rest, as in real keys
    loud = 1.0 + 4.0 * (torch.rand(nkv, hd, generator=gen, device="cuda") < 0.03)
    if case["kind"] == "prep":
        st["q"] = normal(n_tok, nq, hd * (2 if case["gate"] else 1)).to(dt)[..., :hd]
        st["k"] = (normal(n_tok, nkv, hd) * loud).to(dt)
        st["q_norm"], st["k_norm"] = 1.0 + 0.1 * normal(hd), 1.0 + 0.1 * normal(hd)
        st["q_out"], st["k_out"] = torch.zeros(n_tok, nq, hd, dtype=dt, device="cuda"), torch.zeros_like(st["k"])
        if own:
            _plan(st)
        return st
    # pages in any order, two of them nobody's
    need = [(t + rows - 1) // rows for t in total]
    order = torch.randperm(sum(need) + 2, generator=gen, device="cuda").to(torch.int32)
    st["max_pages"] = max(need) + 1
    st["pages"] = torch.zeros(n_seq, st["max_pages"], dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        st["pages"][s, :n] = order[at:at + n]
        at += n
    st["n_pages"] = sum(need) + 2
    page_bytes = nkv * rows * hd * 9 // 16
    st["kc"] = torch.zeros(st["n_pages"] * page_bytes, dtype=torch.uint8, device="cuda")
    st["vc"] = torch.zeros_like(st["kc"])
    if case["kind"] == "store":
        st["k"], st["v"] = (normal(n_tok, nkv, hd) * loud).to(dt), normal(n_tok, nkv, hd).to(dt)
    else:
        for s, t in enumerate(total):
            for r0 in range(0, t, 32768):
                p = torch.arange(r0, min(r0 + 32768, t), device="cuda")
                page = st["pages"][s, p // rows].long()
                _write(st, st["kc"], normal(len(p), nkv, hd) * loud, page, p % rows)
                _write(st, st["vc"], normal(len(p), nkv, hd), page, p % rows)
    if case["kind"] == "attn":
        # queries that look for something: scores of a few units' spread
        st["q"] = (1.5 * normal(n_tok, nq, hd)).to(dt)
        st["out"] = torch.zeros(n_tok, nq, hd, dtype=dt, device="cuda")
        if case["gate"]:
            st["gate"] = normal(n_tok, nq, hd).to(dt)
    else:
        out = torch.float32 if case["kind"] == "store" else dt
        st["k_out"] = torch.zeros(n_tok, nkv, hd, dtype=out, device="cuda")
        st["v_out"] = torch.zeros_like(st["k_out"])
    if own:
        _plan(st)
    return st


# ---------------------------------------------------------------- the library's calls

def _plan(st):
    """The argument records a program keeps for these buffers."""
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import sinter
    case, L = st["case"], sinter.lib()
    rec = {"lib": L, "check": sinter.check, "type": TYPE_IDS[case["type"]]}
    b = sinter.Kv4Batch(tok_start=st["tok_start"].data_ptr(), kv_len=st["kv_len"].data_ptr(), n_seq=case["seqs"],
                        n_tok=st["n_tok"], page_rows=case["page"], nkv=case["nkv"], hd=case["hd"])
    if case["kind"] != "prep":
        b.pages, b.kc, b.vc = st["pages"].data_ptr(), st["kc"].data_ptr(), st["vc"].data_ptr()
        b.max_pages, b.n_pages = st["max_pages"], st["n_pages"]
    rec["batch"] = b

    def heads(name):
        t = st.get(name)
        return sinter.Heads() if t is None else sinter.Heads(p=t.data_ptr(), ld=t.stride(0), hs=t.stride(1))

    if case["kind"] == "prep":
        rec["args"] = sinter.Kv4PrepArgs(q=heads("q"), q_out=heads("q_out"), k=heads("k"), k_out=heads("k_out"),
                                         q_norm=st["q_norm"].data_ptr(), k_norm=st["k_norm"].data_ptr(),
                                         nq=case["nq"], rope_dims=ROPE, rope_base=BASE, eps=EPS, type=rec["type"])
    elif case["kind"] == "attn":
        new, total = max(st["new"]), max(n + p for n, p in zip(st["new"], st["past"]))
        a = sinter.Kv4AttnArgs(q=heads("q"), gate=heads("gate"), out=heads("out"), nq=case["nq"], max_q=new,
                               max_kv=total, scale=1.0 / math.sqrt(case["hd"]), type=rec["type"])
        size = L.sinter_kv4_attn_ws_bytes(C.byref(b), C.byref(a))
        st["ws"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        a.ws, a.ws_bytes = st["ws"].data_ptr(), size
        rec["args"] = a
    else:
        rec["in"], rec["out"] = (heads("k"), heads("v")), (heads("k_out"), heads("v_out"))
    st["plan"] = rec


def _run_own(st):
    if "plan" not in st:
        _plan(st)
    r, case = st["plan"], st["case"]
    L, ref, stream = r["lib"], C.byref, C.c_void_p(torch.cuda.current_stream().cuda_stream)
    b = ref(r["batch"])
    if case["kind"] == "prep":
        r["check"](L.sinter_kv4_prep(b, ref(r["args"]), stream), "prep")
        return st["q_out"], st["k_out"]
    if case["kind"] == "attn":
        r["check"](L.sinter_kv4_attn(b, ref(r["args"]), stream), "attn")
        return st["out"]
    if case["kind"] == "store":
        r["check"](L.sinter_kv4_append(b, ref(r["in"][0]), ref(r["in"][1]), r["type"], stream), "append")
    out = TYPE_IDS["f32"] if case["kind"] == "store" else r["type"]
    r["check"](L.sinter_kv4_read(b, ref(r["out"][0]), ref(r["out"][1]), out, stream), "read")
    return st["k_out"], st["v_out"]


# ---------------------------------------------------------------- the plain form

def _rope(x, w, pos, dt):
    x = x.float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    half = ROPE // 2
    freq = BASE ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    ang = pos.double()[:, None, None] * freq
    c, s = ang.cos().float(), ang.sin().float()
    a, b = y[..., :half], y[..., half:ROPE]
    return torch.cat([a * c - b * s, a * s + b * c, y[..., ROPE:]], -1).to(dt)


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    dt, rows = DTYPES[case["type"]], case["page"]
    if case["kind"] == "prep":
        return _rope(st["q"], st["q_norm"], st["pos"], dt), _rope(st["k"], st["k_norm"], st["pos"], dt)
    if case["kind"] != "attn":
        page, row = st["pages"][st["seq"], st["pos"] // rows].long(), st["pos"] % rows
        if case["kind"] == "store":
            _write(st, st["kc"], st["k"].float(), page, row)
            _write(st, st["vc"], st["v"].float(), page, row)
        out = torch.float32 if case["kind"] == "store" else dt
        return _values(st, st["kc"], page, row).to(out), _values(st, st["vc"], page, row).to(out)
    gqa, outs, at = case["nq"] // case["nkv"], [], 0
    for s, (n, p) in enumerate(zip(st["new"], st["past"])):
        pos = torch.arange(n + p, device="cuda")
        page, row = st["pages"][s, pos // rows].long(), pos % rows
        k = _values(st, st["kc"], page, row).transpose(0, 1).contiguous()     # [nkv, rows, hd]
        v = _values(st, st["vc"], page, row).transpose(0, 1).contiguous()
        q = st["q"][at:at + n].float().transpose(0, 1).reshape(case["nkv"], gqa * n, -1)
        score = q @ k.transpose(1, 2) * (1.0 / math.sqrt(case["hd"]))
        seen = pos[None, :] <= pos[p:, None]                                   # [n, rows]
        score = score.view(case["nkv"], gqa, n, -1).masked_fill(~seen, float("-inf"))
        w = (score - score.amax(-1, keepdim=True)).exp()
        o = (w.view(case["nkv"], gqa * n, -1) @ v).view(case["nq"], n, -1) / w.sum(-1).view(case["nq"], n, 1)
        outs.append(o.transpose(0, 1))
        at += n
    o = torch.cat(outs)
    if case["gate"]:
        o = o * (1.0 / (1.0 + (-st["gate"].float()).exp()))
    return o.to(dt)


# ---------------------------------------------------------------- floors

def work(case):
    new, past = _lens(case)
    n_tok, total = sum(new), sum(new) + sum(past)
    nq, nkv, hd, e = case["nq"], case["nkv"], case["hd"], BYTES[case["type"]]
    row = nkv * hd * 9 // 16                              # a cache row of K (or V)
    if case["kind"] == "prep":
        n = n_tok * (nq + nkv) * hd
        return {"bytes": 2 * e * n, "flops": 6 * n}
    if case["kind"] == "store":                           # in, quantised, read back in f32
        n = n_tok * nkv * hd
        return {"bytes": 2 * (e * n + 2 * n_tok * row + 4 * n), "flops": 2 * 6 * n}
    if case["kind"] == "read":
        return {"bytes": 2 * n_tok * (row + e * nkv * hd), "flops": 2 * n_tok * nkv * hd}
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    return {"bytes": 2 * total * row + e * n_tok * nq * hd * (3 if case["gate"] else 2),
            "flops": 4 * pairs * nq * hd}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_values(case, st, name, s, pos):
    """f64 values [nkv, rows, hd] of sequence s at positions pos, from the cache's bytes."""
    rows, hd, nkv = case["page"], case["hd"], case["nkv"]
    head = rows * hd * 9 // 16
    raw = st[name].view(-1, nkv, head)
    page, row = st["pages"][s, pos // rows].long(), pos % rows
    out = torch.empty(nkv, len(pos), hd, dtype=torch.float64, device="cuda")
    byte = torch.arange(hd // 2, device="cuda")
    for g in range(nkv):
        b = raw[page[:, None], g, row[:, None] * (hd // 2) + byte].int()
        at = rows * hd // 2 + row[:, None] * (hd // 16) + torch.arange(hd // 16, device="cuda")
        d = raw[page[:, None], g, at].contiguous().view(torch.float16).double()
        low = 32 * (byte // 16) + byte % 16
        out[g][:, low] = ((b % 16) - 8).double() * d[:, byte // 16]
        out[g][:, low + 16] = ((b // 16) - 8).double() * d[:, byte // 16]
    return out


def _exact_stored(x):
    """What the cache gives back for x, the format's own f32 roundings spelled out in f64."""
    x = np.clip(x.astype(np.float64), -65504.0, 65504.0).reshape(-1, 32)
    top = x[np.arange(len(x)), np.abs(x).argmax(1)]
    d = (top / -8.0).astype(np.float32)
    d16 = d.astype(np.float16)
    with np.errstate(divide="ignore"):
        inv = np.where(d16 != 0, (1.0 / d.astype(np.float64)).astype(np.float32), np.float32(0)).astype(np.float64)
    prod = (x * inv[:, None]).astype(np.float32).astype(np.float64)
    code = np.minimum(np.trunc((prod + 8.5).astype(np.float32)), 15.0)
    return (code - 8.0) * d16.astype(np.float64)[:, None]


def exact(case, seed):
    st = prepare(case, seed)
    new, past = st["new"], st["past"]
    if case["kind"] == "prep":
        outs = []
        for x, w in ((st["q"], st["q_norm"]), (st["k"], st["k_norm"])):
            x, w = x.double(), w.double()
            y = x / (x.pow(2).sum(-1, keepdim=True) / case["hd"] + EPS).sqrt() * w
            for i in range(ROPE // 2):
                ang = st["pos"].double() * math.pow(BASE, -2.0 * i / ROPE)
                c, s = ang.cos()[:, None], ang.sin()[:, None]
                lo, hi = y[..., i].clone(), y[..., i + ROPE // 2].clone()
                y[..., i], y[..., i + ROPE // 2] = lo * c - hi * s, hi * c + lo * s
            outs.append(y)
        return tuple(outs)
    if case["kind"] == "store":
        return tuple(torch.from_numpy(_exact_stored(st[n].float().cpu().numpy()).reshape(st[n].shape))
                     for n in ("k", "v"))
    if case["kind"] == "read":
        outs = []
        for name in ("kc", "vc"):
            parts = [_exact_values(case, st, name, s, torch.arange(p, p + n, device="cuda")).transpose(0, 1)
                     for s, (n, p) in enumerate(zip(new, past))]
            outs.append(torch.cat(parts))
        return tuple(outs)
    nkv, gqa = case["nkv"], case["nq"] // case["nkv"]
    out, at = torch.zeros(st["n_tok"], case["nq"], case["hd"], dtype=torch.float64, device="cuda"), 0
    for s, (n, p) in enumerate(zip(new, past)):
        pos = torch.arange(n + p, device="cuda")
        k, v = (_exact_values(case, st, name, s, pos) for name in ("kc", "vc"))
        for h in range(case["nq"]):
            q = st["q"][at:at + n, h].double()
            score = q.matmul(k[h // gqa].t().contiguous()) / math.sqrt(case["hd"])
            if n > 1:
                score += torch.full_like(score, float("-inf")).triu(p + 1)
            out[at:at + n, h] = torch.softmax(score, -1).matmul(v[h // gqa])
        at += n
    if case["gate"]:
        out *= torch.sigmoid(st["gate"].double())
    return out
