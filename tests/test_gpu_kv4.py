"""The 4-bit paged KV cache's operators (sinter_kv4_*) on the GPU against the
64-bit reference (kv4_ref.py).

Append and read back are compared byte for byte and value for value: the
quantiser's fp32 steps are the format's definition.  The tolerances of prep
and attention count roundings (u = 2^-24, the fp32 half step):

prep: the sum of squares adds at most 9 roundings (a product, two sums within
the lane, six across lanes), halved by the root, the mean, eps, root and
reciprocal 4 more, the three products 3, the rotation 3 (cos and sin rounded,
product, sum): 16 u of |y| + |partner|, then the type's half step.

attention: a score is a sum of hd products of q and k, in fp32 within a block
and over the blocks: at most 40 u of sum |q k| (32 products and at most 8
scaled sums), to which F32's q in two f16 parts adds 2^-22; its
rounding in log2 units and the exponential add 8 u of the score's size and 8 u.
A weight's relative error is that of its score twice (its own and the sum's);
the product with the V scale enters as f16 (2^-11; two parts 2^-22), the sums
over rows add at most 2^-18 (tiles, waves and chunks of at most 64 each on top
of the 32 rows of a tile), and a term of a row of n is off by at least f16's
smallest step, 2^-25 at a largest weight of at least 2^4 / (scale bound): n 2^-26
of the largest |v|.  All of it in sum w |v|, then the gate's 8 u and the
type's half step.  Sequences of many (token, head) rows (more than 96, or 256
where the batch is little work) run on tiles unpacked to f16, which the
tolerance allows from 32 rows on: V's scale * code is rounded (2^-11 of sum w |v|; F32 keeps the
rest in a second part), and for BF16 K's too, 2^-11 of sum |q k| in a score.
"""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = 0, 1, 30
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
SMALLEST = {F32: 2.0 ** -126, F16: 2.0 ** -24, BF16: 2.0 ** -126}


def tdtype(torch, t):
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[t]


class Batch:
    """Device and host copies of a batch over a cache of shuffled pages."""

    def __init__(self, sn, torch, new, kv_len, page, nkv, hd, pad=0, spare=1, seed=0, fill=None):
        rng = np.random.default_rng(seed)
        self.sn, self.torch, self.page, self.nkv, self.hd = sn, torch, page, nkv, hd
        self.tok_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.kv_len = np.array(kv_len, np.int32)
        self.n_tok = int(self.tok_start[-1]) + pad
        need = [max(0, -(-int(n) // page)) for n in kv_len]
        self.max_pages = max(need + [1]) + 1
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.pages = np.full((len(kv_len), self.max_pages), -7, np.int32)   # (no entry behind the rows is ever read)
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = order[at:at + n]
            at += n
        nbytes = self.n_pages * ref.page_bytes(page, nkv, hd)
        self.kc = np.full(nbytes, 0x7E, np.uint8) if fill is None else fill(nbytes)   # scales 0x7e7e: NaN
        self.vc = self.kc.copy()
        self.up()

    def up(self):
        self.d = {n: self.torch.from_numpy(np.ascontiguousarray(getattr(self, n)).reshape(-1)).to("cuda")
                  for n in ("tok_start", "kv_len", "pages", "kc", "vc")}

    def rec(self):
        d = self.d
        return self.sn.Kv4Batch(tok_start=d["tok_start"].data_ptr(), kv_len=d["kv_len"].data_ptr(),
                                pages=d["pages"].data_ptr(), kc=d["kc"].data_ptr(), vc=d["vc"].data_ptr(),
                                n_seq=len(self.kv_len), n_tok=self.n_tok, max_pages=self.max_pages,
                                n_pages=self.n_pages, page_rows=self.page, nkv=self.nkv, hd=self.hd)

    def rows(self, s, n):
        """K and V values [nkv][n][hd] of sequence s."""
        out = []
        for cache in (self.kc, self.vc):
            out.append(np.array([[ref.get(cache, self.pages[s, r // self.page], r % self.page, g, self.page, self.nkv,
                                          self.hd) for r in range(n)] for g in range(self.nkv)]).reshape(self.nkv, n, self.hd))
        return out

    def fill_rows(self, seed, loud=True):
        """Random K and V in every row that a sequence has."""
        rng = np.random.default_rng(seed)
        ch = 1.0 + 4.0 * (rng.random((self.nkv, self.hd)) < 0.05)
        for s, n in enumerate(self.kv_len):
            for cache, c in ((self.kc, ch), (self.vc, 1.0)):
                x = (rng.standard_normal((max(0, n), self.nkv, self.hd)) * c).astype(np.float32)
                code, d16 = ref.quantise(x)
                for r in range(max(0, n)):
                    for g in range(self.nkv):
                        ref.put(cache, self.pages[s, r // self.page], r % self.page, g, self.page, self.nkv, self.hd,
                                code[r, g], d16[r, g])
        self.up()


def heads(sn, t):
    return sn.Heads(p=t.data_ptr(), ld=t.stride(0), hs=t.stride(1))


def stream(torch):
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def strided(torch, x, t, extra_head=0, extra_tok=0):
    """x [n, heads, hd] on the device as `t`, inside a larger buffer of 7s."""
    n, h, hd = x.shape
    buf = torch.full((n, h * (hd + extra_head) + extra_tok), 7.0, dtype=tdtype(torch, t), device="cuda")
    view = torch.as_strided(buf, (n, h, hd), (buf.stride(0), hd + extra_head, 1))
    view.copy_(torch.from_numpy(x).to("cuda").to(tdtype(torch, t)))
    return buf, view


def ok(sn, rc, torch):
    sn.check(rc, "kv4")
    torch.cuda.synchronize()
    assert sn.op_error()[0] == 0


# ---------------------------------------------------------------- append, read

def awkward_rows(n, nkv, hd, seed):
    """Rows with the values at which a quantiser goes wrong."""
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((n, nkv, hd)) * 10.0 ** rng.integers(-3, 3, (n, nkv, 1))).astype(np.float32)
    flat = x.reshape(-1, 32)
    k = 0
    for special in (np.zeros(32), np.full(32, -2.0), np.where(np.arange(32) % 2, 3.0, -3.0),
                    np.where(np.arange(32) % 2, -3.0, 3.0), np.full(32, 1e-8), np.full(32, 3e-7), rng.standard_normal(32) * 1e-40,
                    rng.standard_normal(32) * 1e6, np.full(32, 65504.0), np.full(32, np.inf), np.full(32, -np.inf),
                    np.where(np.arange(32) == 5, np.nan, 1.0), np.where(np.arange(32) == 31, np.nan, np.inf),
                    np.arange(32) - 15.5, (np.arange(32) - 16) / 2.0, np.where(np.arange(32) == 31, 8.0, 0.5)):
        if k < len(flat):
            flat[k] = special
        k += 3
    return x


STORE = [(F32, 4, 256, 64, [1, 5, 0, 3], [70, 5, 9, 200]), (F16, 2, 128, 16, [1], [1]), (BF16, 8, 128, 32, [33, 40], [33, 100]),
         (BF16, 1, 64, 16, [17, 1, 1], [17, 3, 65]), (F32, 3, 64, 1024, [9], [1030]), (F16, 16, 64, 16, [4, 4], [2, 4])]


@pytest.mark.parametrize("t,nkv,hd,page,new,kv", STORE)
def test_append_and_read(sn, torch_gpu, t, nkv, hd, page, new, kv):
    """The cache's bytes, every other byte of it left alone, padding and tokens
    without a row skipped, strided inputs and outputs; the rows read back."""
    torch = torch_gpu
    b = Batch(sn, torch, new, kv, page, nkv, hd, pad=3, seed=hd + page)
    x = [torch.from_numpy(awkward_rows(b.n_tok, nkv, hd, 5 + i)).to(tdtype(torch, t)) for i in range(2)]
    print(f"append t={t} nkv={nkv} hd={hd} page={page}", flush=True)
    views = [strided(torch, a.float().numpy(), t, 16 * i, 32 - 16 * i) for i, a in enumerate(x)]
    ok(sn, sn.lib().sinter_kv4_append(C.byref(b.rec()), C.byref(heads(sn, views[0][1])), C.byref(heads(sn, views[1][1])), t,
                                     stream(torch)), torch)
    want = [b.kc.copy(), b.vc.copy()]
    pos = ref.positions(b.tok_start, b.kv_len, b.n_tok)
    back = [np.full((b.n_tok, nkv, hd), np.nan), np.full((b.n_tok, nkv, hd), np.nan)]
    for i in range(2):
        code, d16 = ref.quantise(x[i].float().numpy())
        for j, (s, p) in enumerate(pos):
            if s < 0 or p < 0:
                continue
            for g in range(nkv):
                ref.put(want[i], b.pages[s, p // page], p % page, g, page, nkv, hd, code[j, g], d16[j, g])
                back[i][j, g] = ref.values(code[j, g], d16[j, g])
    assert np.array_equal(b.d["kc"].cpu().numpy(), want[0])
    assert np.array_equal(b.d["vc"].cpu().numpy(), want[1])
    for ot in (F32, F16, BF16):
        outs = [strided(torch, np.full((b.n_tok, nkv, hd), 3.0, np.float32), ot, 8 * i, 64) for i in range(2)]
        ok(sn, sn.lib().sinter_kv4_read(C.byref(b.rec()), C.byref(heads(sn, outs[0][1])), C.byref(heads(sn, outs[1][1])), ot,
                                        stream(torch)), torch)
        for i in range(2):
            exp, _ = strided(torch, np.full((b.n_tok, nkv, hd), 3.0, np.float32), ot, 8 * i, 64)
            ev = torch.as_strided(exp, outs[i][1].shape, outs[i][1].stride())
            for j, (s, p) in enumerate(pos):
                if s >= 0 and p >= 0:
                    ev[j] = torch.from_numpy(back[i][j]).to("cuda").float().to(tdtype(torch, ot))
            assert torch.equal(torch.nan_to_num(outs[i][0].float(), nan=99.0), torch.nan_to_num(exp.float(), nan=99.0))


def test_read_one_of_the_two(sn, torch_gpu):
    torch = torch_gpu
    b = Batch(sn, torch, [4], [20], 16, 2, 64)
    b.fill_rows(3)
    k, v = b.rows(0, 20)
    for i, want in enumerate((k, v)):
        out = torch.zeros(4, 2, 64, device="cuda")
        args = [C.byref(heads(sn, out)), None]
        ok(sn, sn.lib().sinter_kv4_read(C.byref(b.rec()), args[i], args[1 - i], F32, stream(torch)), torch)
        assert np.array_equal(out.cpu().numpy(), want.transpose(1, 0, 2)[16:].astype(np.float32))


# ---------------------------------------------------------------- prep

PREP = [(F32, 24, 4, 256, 64, [1], [4098], True, 1e7), (BF16, 24, 4, 256, 64, [3, 0, 2], [131000, 4, 1], True, 1e7),
        (F16, 3, 1, 64, 64, [9, 2], [9, 1], True, 1e4), (F32, 5, 5, 128, 128, [7], [100000], False, 5e5),
        (BF16, 2, 2, 64, 0, [3], [3], True, 1e4), (F32, 1, 1, 256, 8, [1100], [1100], True, 1e4),
        (F16, 33, 1, 128, 24, [1030], [40000], True, 1e6)]


@pytest.mark.parametrize("t,nq,nkv,hd,rope,new,kv,weights,base", PREP)
def test_prep(sn, torch_gpu, t, nq, nkv, hd, rope, new, kv, weights, base):
    torch = torch_gpu
    rng = np.random.default_rng(hd + nq)
    b = Batch(sn, torch, new, kv, 1 << 17, 1, 64, pad=2)   # (only its positions are used)
    b.nkv, b.hd = nkv, hd
    q, k = (rng.standard_normal((b.n_tok, n, hd)).astype(np.float32) * 3 for n in (nq, nkv))
    wq, wk = (torch.from_numpy((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)).to("cuda") for _ in range(2))
    (_, qv), (_, kv_) = strided(torch, q, t, hd), strided(torch, k, t, 16)   # q as the halves of q | gate rows
    qbuf, qo = strided(torch, np.full(q.shape, 3.0, np.float32), t, 0, 16)
    kin = kv_.float().cpu().numpy()
    a = sn.Kv4PrepArgs(q=heads(sn, qv), q_out=heads(sn, qo), k=heads(sn, kv_), k_out=heads(sn, kv_),   # k in place
                       q_norm=wq.data_ptr() if weights else None, k_norm=wk.data_ptr() if weights else None, nq=nq,
                       rope_dims=rope, rope_base=base, eps=1e-6, type=t)
    print(f"prep t={t} nq={nq} hd={hd} rope={rope}", flush=True)
    ok(sn, sn.lib().sinter_kv4_prep(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    pos = ref.positions(b.tok_start, b.kv_len, b.n_tok)
    for x, got, w in ((qv.float().cpu().numpy(), qo.float().cpu().numpy(), wq), (kin, kv_.float().cpu().numpy(), wk)):
        for j, (s, p) in enumerate(pos):
            if s < 0 or p < 0:   # left as it was
                assert np.array_equal(got[j], x[j] if x is kin else np.full_like(x[j], 3.0)), j
                continue
            want, mag = ref.prep(x[j], w.cpu().numpy() if weights else None, p, 1e-6, rope, base)
            tol = 16 * U * mag + HALF_STEP[t] * (1 + 16 * U) * np.abs(want) + 16 * U * HALF_STEP[t] * mag + SMALLEST[t]
            assert (np.abs(got[j] - want) <= tol).all(), (j, np.abs(got[j] - want).max())


def test_prep_one_of_the_two(sn, torch_gpu):
    torch = torch_gpu
    b = Batch(sn, torch, [2], [5], 16, 2, 64)
    x = torch.randn(2, 3, 64, device="cuda")
    full, part = (torch.zeros(2, 3, 64, device="cuda") for _ in range(2))
    k, ko = torch.randn(2, 2, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    base = dict(nq=3, rope_dims=32, rope_base=1e4, eps=1e-5, type=F32)
    L, r, s = sn.lib(), C.byref(b.rec()), stream(torch)
    ok(sn, L.sinter_kv4_prep(r, C.byref(sn.Kv4PrepArgs(q=heads(sn, x), q_out=heads(sn, full), k=heads(sn, k), k_out=heads(sn, ko),
                                                       **base)), s), torch)
    ok(sn, L.sinter_kv4_prep(r, C.byref(sn.Kv4PrepArgs(q=heads(sn, x), q_out=heads(sn, part), **base)), s), torch)
    assert torch.equal(full, part) and float(ko.abs().sum()) > 0
    kp = torch.zeros_like(ko)
    ok(sn, L.sinter_kv4_prep(r, C.byref(sn.Kv4PrepArgs(k=heads(sn, k), k_out=heads(sn, kp), **base)), s), torch)
    assert torch.equal(ko, kp)


# ---------------------------------------------------------------- attention

def attn_args(sn, torch, b, nq, t, q, out, gate=None, max_q=None, max_kv=None, scale=None):
    new = np.diff(b.tok_start)
    a = sn.Kv4AttnArgs(q=heads(sn, q), out=heads(sn, out), nq=nq, max_q=int(max_q or new.max()),
                       max_kv=int(max_kv or max(1, b.kv_len.max())), scale=scale or b.hd ** -0.5, type=t)
    if gate is not None:
        a.gate = heads(sn, gate)
    n = sn.lib().sinter_kv4_attn_ws_bytes(C.byref(b.rec()), C.byref(a))
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    ws.fill_(0xff)   # (NaN wherever a record is read that was not written)
    a.ws, a.ws_bytes = ws.data_ptr(), n
    return a, ws


def check_attn(b, nq, t, q, got, gate, scale, untouched=3.0, only=None):
    """got [n_tok, nq, hd] against the reference; q, gate f64 as the kernel read them."""
    pos = ref.positions(b.tok_start, b.kv_len, b.n_tok)
    gqa = nq // b.nkv
    kv = {}
    for j, (s, p) in enumerate(pos):
        if s < 0:
            assert (got[j] == untouched).all(), j
            continue
        if only is not None and j not in only:
            continue
        if s not in kv:
            kv[s] = b.rows(s, max(0, int(b.kv_len[s])))
        for h in range(nq):
            k, v = kv[s][0][h // gqa, :max(0, p + 1)], kv[s][1][h // gqa, :max(0, p + 1)]
            with np.errstate(all="ignore"):
                want, mag, qk = ref.attention(q[j, h], k, v, scale)
            n, many = len(k), int(b.tok_start[s + 1] - b.tok_start[s]) * gqa > 32
            score = 40 * U * qk + (2.0 ** -22 * qk if t == F32 else 0) + 8 * U * qk + 8 * U
            if many and t == BF16:
                score += 2.0 ** -11 * qk
            rel = 2 * score + (2.0 ** -22 if t == F32 else 2.0 ** -11) + 2.0 ** -18
            if many and t != F32:
                rel += 2.0 ** -11
            err = rel * mag + n * 2.0 ** -26 * (np.abs(v).max() if n else 0)
            if gate is not None:
                sg = 1.0 / (1.0 + np.exp(-gate[j, h]))
                want, err = want * sg, err * sg + 8 * U * np.abs(want)
            tol = err + HALF_STEP[t] * (np.abs(want) + err) + SMALLEST[t]
            assert np.isfinite(got[j, h]).all(), (j, h)
            bad = np.abs(got[j, h] - want) > tol
            assert not bad.any(), (j, h, float(np.abs(got[j, h] - want).max()), float(tol[bad].min()))


ATTN = [
    # t, nq, nkv, hd, page, new, kv_len, gate
    (F32, 24, 4, 256, 64, [1], [1], True), (F32, 24, 4, 256, 64, [1, 1, 1], [300, 33, 32], False),
    (BF16, 24, 4, 256, 16, [1, 0, 1, 1], [31, 50, 17, 129], True), (F16, 8, 8, 128, 32, [1, 2, 5], [700, 2, 64], False),
    (F16, 32, 8, 128, 16, [4, 4], [1100, 4], False), (F32, 12, 1, 64, 64, [3, 1], [90, 1500], True),
    (BF16, 40, 2, 64, 16, [5, 1, 2], [5, 640, 100], True), (F32, 16, 16, 64, 128, [2, 1], [600, 47], False),
    (F32, 6, 1, 256, 2048, [1], [2500], True), (BF16, 7, 1, 128, 64, [19, 40], [19, 75], False),
    (F16, 5, 5, 256, 32, [37], [100], True), (F32, 28, 4, 128, 16, [21, 3, 1], [530, 3, 16], False),
    # more tokens than rows: the first have none
    (F32, 6, 2, 64, 16, [5, 2], [3, 0], True), (BF16, 4, 1, 256, 16, [40], [33], False),
]


def run_attn(sn, torch, t, nq, nkv, hd, page, new, kv, gated, seed, poison=True, **kw):
    b = Batch(sn, torch, new, kv, page, nkv, hd, pad=2, spare=3, seed=seed)
    b.fill_rows(seed + 1)
    rng = np.random.default_rng(seed + 2)
    q = rng.standard_normal((b.n_tok, nq, hd)).astype(np.float32) * 1.5
    g = rng.standard_normal((b.n_tok, nq, hd)).astype(np.float32) * 2
    (_, qv), (_, gv) = strided(torch, q, t, 32), strided(torch, g, t, 0, 16)
    obuf, ov = strided(torch, np.full(q.shape, 3.0, np.float32), t, 16, 8)
    a, ws = attn_args(sn, torch, b, nq, t, qv, ov, gv if gated else None, **kw)
    print(f"attn t={t} nq={nq} nkv={nkv} hd={hd} page={page} new={new} kv={kv}", flush=True)
    ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    got = ov.float().cpu().numpy()
    rest = obuf.clone()
    torch.as_strided(rest, ov.shape, ov.stride()).fill_(7.0)
    assert bool((rest == 7.0).all())   # nothing between the rows written
    return b, qv.double().cpu().numpy(), gv.double().cpu().numpy() if gated else None, got


@pytest.mark.parametrize("t,nq,nkv,hd,page,new,kv,gated", ATTN)
def test_attention(sn, torch_gpu, t, nq, nkv, hd, page, new, kv, gated):
    """Every cache byte that no sequence has is NaN in its scales."""
    b, q, g, got = run_attn(sn, torch_gpu, t, nq, nkv, hd, page, new, kv, gated, 40 + hd + nq)
    check_attn(b, nq, t, q, got, g, hd ** -0.5)


@pytest.mark.parametrize("t,hd", [(F32, 256), (BF16, 128)])
def test_attention_split_over_many_chunks(sn, torch_gpu, t, hd):
    """Long and short sequences in one batch: several chunks each, joined."""
    b, q, g, got = run_attn(sn, torch_gpu, t, 6, 1, hd, 64, [1, 2, 1, 1], [5000, 1700, 513, 40], True, 9)
    check_attn(b, 6, t, q, got, g, hd ** -0.5)


@pytest.mark.parametrize("n_seq", [65, 130])
def test_attention_many_sequences(sn, torch_gpu, n_seq):
    rng = np.random.default_rng(n_seq)
    kv = rng.integers(0, 40, n_seq)
    kv[3], kv[-1] = 900, 700
    new = rng.integers(0, 3, n_seq)
    new[3] = new[-1] = 1
    b, q, g, got = run_attn(sn, torch_gpu, BF16, 2, 1, 64, 16, list(new), list(kv), False, 17)
    check_attn(b, 2, BF16, q, got, g, 64 ** -0.5)


@pytest.mark.parametrize("t,nkv,hd,n_seq", [(F32, 16, 256, 40), (BF16, 8, 256, 80), (F16, 16, 64, 70)])
def test_attention_more_sequences_than_slots(sn, torch_gpu, t, nkv, hd, n_seq):
    """Long sequences that share the slots of a call, each divided where a
    slot's share ends; all read one sequence's pages."""
    torch = torch_gpu
    rng = np.random.default_rng(hd + n_seq)
    kv = rng.integers(500, 1200, n_seq)
    kv[0], kv[5], kv[7] = 1200, 1, 40
    new = np.ones(n_seq, int)
    new[3], new[9] = 2, 0
    b = Batch(sn, torch, list(new), list(kv), 64, nkv, hd, seed=n_seq)
    b.pages[:] = b.pages[0]
    b.kv_len = b.kv_len[:1]
    b.fill_rows(7)
    b.kv_len = kv.astype(np.int32)
    b.up()
    q = rng.standard_normal((b.n_tok, nkv, hd)).astype(np.float32)
    (_, qv), (_, ov) = strided(torch, q, t), strided(torch, np.full(q.shape, 3.0, np.float32), t)
    a, ws = attn_args(sn, torch, b, nkv, t, qv, ov)
    print(f"{n_seq} sequences over {nkv} heads of {hd}", flush=True)
    ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    check_attn(b, nkv, t, qv.double().cpu().numpy(), ov.float().cpu().numpy(), None, hd ** -0.5,
               only={0, 3, 4, 5, 7, *range(9, b.n_tok, 9)})


@pytest.mark.parametrize("t", [F32, BF16])
def test_attention_many_sequences_of_many_rows(sn, torch_gpu, t):
    """More than 64 sequences, prompts among them, empty ones between."""
    rng = np.random.default_rng(8)
    new = rng.integers(0, 3, 90)
    new[[2, 40, 41, 70, 89]] = [50, 20, 33, 140, 17]
    kv = new + rng.integers(0, 60, 90)
    kv[[5, 41, 70]] = [300, 700, 140]
    b, q, g, got = run_attn(sn, torch_gpu, t, 2, 1, 64, 16, list(new), list(kv), True, 18)
    check_attn(b, 2, t, q, got, g, 64 ** -0.5)


@pytest.mark.parametrize("t,nq,new,kv", [(BF16, 40, [1, 0, 3, 1], [70, 9, 900, 1]), (F32, 33, [1, 1], [600, 31]), (F16, 256, [1, 2], [33, 2])])
def test_attention_large_groups(sn, torch_gpu, t, nq, new, kv):
    """More q heads to a kv head than the split kernel's rows."""
    b, q, g, got = run_attn(sn, torch_gpu, t, nq, 1, 64, 32, new, kv, False, 19)
    check_attn(b, nq, t, q, got, g, 64 ** -0.5)


@pytest.mark.parametrize("n_seq", [300, 4500])
def test_batches_of_many_sequences(sn, torch_gpu, n_seq):
    """Replies of thousands of sequences, some without a token, and prompts of
    hundreds (several tokens a workgroup, across sequences): stored, read back
    and attended to."""
    torch = torch_gpu
    rng = np.random.default_rng(n_seq)
    new = rng.integers(0, 60, n_seq) if n_seq < 1000 else rng.integers(0, 3, n_seq)
    kv = np.maximum(new + rng.integers(-1, 5, n_seq), 0)
    b = Batch(sn, torch, list(new), list(kv), 16, 1, 64, pad=5, seed=n_seq)
    x = [rng.standard_normal((b.n_tok, 1, 64)).astype(np.float32) for _ in range(2)]
    dev = [torch.from_numpy(a).to("cuda") for a in x]
    print(f"{n_seq} sequences, {b.n_tok} tokens", flush=True)
    L, r, st = sn.lib(), b.rec(), stream(torch)
    ok(sn, L.sinter_kv4_append(C.byref(r), C.byref(heads(sn, dev[0])), C.byref(heads(sn, dev[1])), F32, st), torch)
    pos = ref.positions(b.tok_start, b.kv_len, b.n_tok)
    want = [b.kc.copy(), b.vc.copy()]
    back = [np.full((b.n_tok, 1, 64), 3.0, np.float32) for _ in range(2)]
    for i in range(2):
        code, d16 = ref.quantise(x[i])
        for j, (s, p) in enumerate(pos):
            if s >= 0 and p >= 0:
                ref.put(want[i], b.pages[s, p // 16], p % 16, 0, 16, 1, 64, code[j, 0], d16[j, 0])
                back[i][j, 0] = ref.values(code[j, 0], d16[j, 0])
        assert np.array_equal(b.d["kc" if i == 0 else "vc"].cpu().numpy(), want[i])
    out = [torch.full((b.n_tok, 1, 64), 3.0, device="cuda") for _ in range(2)]
    ok(sn, L.sinter_kv4_read(C.byref(r), C.byref(heads(sn, out[0])), C.byref(heads(sn, out[1])), F32, st), torch)
    for i in range(2):
        assert np.array_equal(out[i].cpu().numpy(), back[i])
    # attention to the rows of this call (the rows before them: as they are)
    b.kc, b.vc = want
    b.fill_rows(n_seq)
    q = rng.standard_normal((b.n_tok, 2, 64)).astype(np.float32)
    (_, qv), (_, ov) = strided(torch, q, BF16), strided(torch, np.full(q.shape, 3.0, np.float32), BF16)
    a, ws = attn_args(sn, torch, b, 2, BF16, qv, ov)
    ok(sn, L.sinter_kv4_attn(C.byref(b.rec()), C.byref(a), st), torch)
    check_attn(b, 2, BF16, qv.double().cpu().numpy(), ov.float().cpu().numpy(), None, 64 ** -0.5,
               only=set(range(0, b.n_tok, 7)))


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("toks", [2, 30])
def test_attention_magnitudes(sn, torch_gpu, t, toks):
    """Tiny and huge values, scales that grow along the sequence and differ by
    block, scores that keep growing: the weights' reference moves."""
    torch = torch_gpu
    hd, n = 128, 700
    b = Batch(sn, torch, [toks], [n], 64, 1, hd, seed=4)
    rng = np.random.default_rng(8)
    q = rng.standard_normal((toks, 4, hd)).astype(np.float32)
    q[0, 1] *= 1e-3
    if t == F32:
        q[1, 2] *= 1e20
        q[1, 2] /= 1e20
    grow = np.linspace(0, 6, n)[:, None]
    k = (rng.standard_normal((n, hd)) + grow * q[0, 0] / 4).astype(np.float32)
    v = (rng.standard_normal((n, hd)) * 10.0 ** np.linspace(-3, 3, n)[:, None] * 10.0 ** -np.repeat([0, 2, 1, 3], 32)).astype(np.float32)
    for cache, x in ((b.kc, k), (b.vc, v)):
        code, d16 = ref.quantise(x)
        for r in range(n):
            ref.put(cache, b.pages[0, r // 64], r % 64, 0, 64, 1, hd, code[r], d16[r])
    b.up()
    (_, qv), (_, ov) = strided(torch, q, t), strided(torch, np.full(q.shape, 3.0, np.float32), t)
    a, ws = attn_args(sn, torch, b, 4, t, qv, ov)
    ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    check_attn(b, 4, t, qv.double().cpu().numpy(), ov.float().cpu().numpy(), None, hd ** -0.5)


@pytest.mark.parametrize("nan", [0x7e00, 0x7c00])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("nq", [6, 14])
def test_attention_rows_not_seen_stay_out(sn, torch_gpu, nan, t, nq):
    """A later token's row that is not finite reaches only the tokens that see it."""
    torch = torch_gpu
    half = nq // 2
    b = Batch(sn, torch, [9], [50], 16, 2, 64, seed=3)
    b.fill_rows(5)
    for cache in (b.kc, b.vc):
        for r in (45, 48):
            _, sc = ref.head_view(cache, b.pages[0, r // 16], 1, 16, 2, 64)
            sc.view(np.uint16)[r % 16, 1] = nan
    b.up()
    q = np.random.default_rng(1).standard_normal((9, nq, 64)).astype(np.float32)
    (_, qv), (_, ov) = strided(torch, q, t), strided(torch, np.zeros_like(q), t)
    a, ws = attn_args(sn, torch, b, nq, t, qv, ov)
    ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    got = ov.float().cpu().numpy()
    assert np.isfinite(got[:4]).all() and np.isfinite(got[:, :half]).all()
    assert not np.isfinite(got[4:, half:]).all(-1).any()
    check_attn(b, nq, t, qv.double().cpu().numpy(), got, None, 64 ** -0.5, only=(0, 1, 2, 3))


@pytest.mark.parametrize("n", [3, 20])
def test_attention_nonfinite_query_stays_alone(sn, torch_gpu, n):
    torch = torch_gpu
    b = Batch(sn, torch, [n], [70], 16, 1, 64, seed=3)
    b.fill_rows(5)
    q = np.random.default_rng(1).standard_normal((n, 2, 64)).astype(np.float32)
    q[1, 0, 7] = np.nan
    q[2, 1, 9] = np.inf
    (_, qv), (_, ov) = strided(torch, q, F32), strided(torch, np.zeros_like(q), F32)
    a, ws = attn_args(sn, torch, b, 2, F32, qv, ov)
    ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    got = ov.cpu().numpy()
    assert np.isnan(got[1, 0]).all()
    fine = np.ones((n, 2), bool)
    fine[1, 0] = fine[2, 1] = False
    assert np.isfinite(got[fine]).all()


# More than 256 rows a sequence, beside shorter ones: the kernel for many rows
MANY = [
    (F32, 16, 1, 256, 16, [20, 1, 40], [100, 30, 41], True), (BF16, 32, 2, 128, 64, [33, 2], [600, 2], False),
    (F16, 16, 1, 64, 16, [18, 70], [18, 400], True), (F16, 64, 2, 256, 32, [9], [40], False),
    (BF16, 18, 1, 256, 16, [40], [33], True), (F32, 256, 1, 128, 16, [2, 1], [130, 1], False),
    (F32, 40, 2, 64, 128, [17, 0, 14], [1500, 3, 14], False), (BF16, 6, 1, 64, 16, [50, 3], [1400, 700], True),
    (F16, 3, 1, 128, 32, [100, 1], [100, 900], False), (BF16, 2, 2, 256, 16, [300], [301], False),
]


@pytest.mark.parametrize("t,nq,nkv,hd,page,new,kv,gated", MANY)
def test_attention_of_many_rows(sn, torch_gpu, t, nq, nkv, hd, page, new, kv, gated):
    b, q, g, got = run_attn(sn, torch_gpu, t, nq, nkv, hd, page, new, kv, gated, 60 + hd + nq)
    check_attn(b, nq, t, q, got, g, hd ** -0.5)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_many_rows_magnitudes(sn, torch_gpu, t):
    test_attention_magnitudes(sn, torch_gpu, t, 80)


@pytest.mark.parametrize("nan", [0x7e00, 0x7c00])
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_many_rows_not_seen_stay_out(sn, torch_gpu, nan, t):
    test_attention_rows_not_seen_stay_out(sn, torch_gpu, nan, t, 70)


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_many_rows_nonfinite_query_stays_alone(sn, torch_gpu, t):
    torch = torch_gpu
    b = Batch(sn, torch, [20], [70], 16, 1, 64, seed=3)
    b.fill_rows(5)
    q = np.random.default_rng(1).standard_normal((20, 20, 64)).astype(np.float32)
    q[1, 0, 7] = np.nan
    q[2, 1, 9] = np.inf
    (_, qv), (_, ov) = strided(torch, q, t), strided(torch, np.zeros_like(q), t)
    a, ws = attn_args(sn, torch, b, 20, t, qv, ov)
    ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    got = ov.float().cpu().numpy()
    assert np.isnan(got[1, 0]).all()
    fine = np.ones((20, 20), bool)
    fine[1, 0] = fine[2, 1] = False
    assert np.isfinite(got[fine]).all()


@pytest.mark.parametrize("page", [16, 64])
def test_many_rows_missing_pages(sn, torch_gpu, page):
    torch = torch_gpu
    b = Batch(sn, torch, [2, 20], [60, 90], page, 1, 64, seed=3)
    b.fill_rows(5)
    q = np.random.default_rng(1).standard_normal((22, 20, 64)).astype(np.float32)
    (_, qv), (_, ov) = strided(torch, q, F32), strided(torch, np.zeros_like(q), F32)
    b.pages[1, 0] = b.n_pages
    b.up()
    a, ws = attn_args(sn, torch, b, 20, F32, qv, ov)
    sn.check(sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), "attn")
    torch.cuda.synchronize()
    assert sn.op_error() == (sn.E_BAD_SHAPE, 1)
    got = ov.cpu().numpy()
    check_attn(b, 20, F32, q.astype(np.float64), got, None, 0.125, only=(0, 1))
    for j in (2, 21):
        rows = range(page, 90 - 20 + (j - 2) + 1)   # (without the first page's)
        k, v = (np.array([ref.get(c, b.pages[1, r // page], r % page, 0, page, 1, 64) for r in rows]).reshape(-1, 64) for c in (b.kc, b.vc))
        want, mag, _ = ref.attention(q[j, 7].astype(np.float64), k, v, 0.125)
        assert np.abs(got[j, 7] - want).max() <= 2.0 ** -15 * mag.max()


@pytest.mark.parametrize("what", ["max_q", "max_kv", "tokens"])
def test_many_rows_over_the_bounds(sn, torch_gpu, what):
    torch = torch_gpu
    b = Batch(sn, torch, [1, 30], [30, 600], 16, 1, 64, seed=3)
    b.fill_rows(5)
    q = np.random.default_rng(1).standard_normal((31, 16, 64)).astype(np.float32)
    kw = dict(max_q=30, max_kv=700)
    if what == "tokens":
        b.tok_start[2] = 90
        b.up()
    else:
        kw[what] -= 150 if what == "max_kv" else 4
    (_, qv), (_, ov) = strided(torch, q, BF16), strided(torch, np.zeros_like(q), BF16)
    a, ws = attn_args(sn, torch, b, 16, BF16, qv, ov, **kw)
    sn.check(sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), "attn")
    torch.cuda.synchronize()
    assert sn.op_error() == (sn.E_BAD_SHAPE, 1)
    b.tok_start[2] = 31
    check_attn(b, 16, BF16, qv.double().cpu().numpy(), ov.float().cpu().numpy(), None, 0.125, only=(0,))


# ---------------------------------------------------------------- errors seen on the device

def test_missing_pages(sn, torch_gpu):
    """A page outside the cache: reported, nothing read or written there, the
    other rows and sequences as without it."""
    torch = torch_gpu
    b = Batch(sn, torch, [2, 2], [60, 40], 16, 2, 64, seed=3)
    b.fill_rows(5)
    q = np.random.default_rng(1).standard_normal((4, 2, 64)).astype(np.float32)
    good = b.pages[1].copy()
    for bad in (-1, b.n_pages, 2 ** 31 - 1):
        b.pages[1, 1] = bad
        b.up()
        (_, qv), (_, ov) = strided(torch, q, F32), strided(torch, np.zeros_like(q), F32)
        a, ws = attn_args(sn, torch, b, 2, F32, qv, ov)
        sn.check(sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), "attn")
        assert sn.op_error() == (sn.E_BAD_SHAPE, 1)
        assert sn.op_error() == (0, 0)   # read and cleared
        got = ov.cpu().numpy()
        check_attn(b, 2, F32, q.astype(np.float64), got, None, 0.125, only=(0, 1))
        b.pages[1] = good
        k, v = b.rows(1, 40)
        keep = np.r_[0:16, 32:39]       # token 2 is at position 38
        want, mag, _ = ref.attention(q[2, 0].astype(np.float64), k[0][keep], v[0][keep], 0.125)
        assert np.abs(got[2, 0] - want).max() <= 2.0 ** -15 * mag.max()
    # append and read skip the row
    b.pages[1, 2] = -5
    b.up()
    x = torch.ones(4, 2, 64, device="cuda")
    before = b.kc.copy()
    sn.check(sn.lib().sinter_kv4_append(C.byref(b.rec()), C.byref(heads(sn, x)), C.byref(heads(sn, x)), F32, stream(torch)), "append")
    assert sn.op_error() == (sn.E_BAD_SHAPE, 1)
    code, d16 = ref.quantise(np.ones((1, 64), np.float32))
    for p in (58, 59):
        for g in range(2):
            ref.put(before, b.pages[0, p // 16], p % 16, g, 16, 2, 64, code[0], d16[0])
    assert np.array_equal(b.d["kc"].cpu().numpy(), before)
    out = torch.full((4, 2, 64), 3.0, device="cuda")
    sn.check(sn.lib().sinter_kv4_read(C.byref(b.rec()), C.byref(heads(sn, out)), None, F32, stream(torch)), "read")
    assert sn.op_error() == (sn.E_BAD_SHAPE, 1)
    assert bool((out[:2] == 1).all()) and bool((out[2:] == 3.0).all())


@pytest.mark.parametrize("what", ["max_q", "max_kv", "table", "tokens"])
def test_lengths_over_the_bounds(sn, torch_gpu, what):
    """A sequence longer than the call was told, than its page table, or than
    the token arrays is reported; the others keep their results."""
    torch = torch_gpu
    b = Batch(sn, torch, [1, 3], [30, 600], 16, 1, 64, seed=3)
    b.fill_rows(5)
    q = np.random.default_rng(1).standard_normal((4, 2, 64)).astype(np.float32)
    kw = {}
    if what == "max_q":
        kw["max_q"] = 2
    elif what == "max_kv":
        kw["max_kv"] = 500
    elif what == "table":
        b.kv_len[1] = b.max_pages * 16 + 3
    else:
        b.tok_start[2] = 9
    b.d["tok_start"].copy_(torch.from_numpy(b.tok_start)), b.d["kv_len"].copy_(torch.from_numpy(b.kv_len))
    if what == "table":
        b.pages[1, -1] = b.pages[1, 0]
        b.up()
    (_, qv), (_, ov) = strided(torch, q, F32), strided(torch, np.zeros_like(q), F32)
    kw.setdefault("max_q", 3), kw.setdefault("max_kv", 700)
    a, ws = attn_args(sn, torch, b, 2, F32, qv, ov, **kw)
    sn.check(sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), "attn")
    assert sn.op_error() == (sn.E_BAD_SHAPE, 1)
    b.tok_start[2] = 4
    check_attn(b, 2, F32, q.astype(np.float64), ov.cpu().numpy(), None, 0.125, only=(0,))


# ---------------------------------------------------------------- how they are used

def test_many_bytes_of_cache(sn, torch_gpu):
    """Pages behind the 4 GiB that 32-bit offsets reach."""
    torch = torch_gpu
    page, nkv, hd = 64, 2, 64
    per = ref.page_bytes(page, nkv, hd)
    n_pages = (5 << 30) // per
    big = [torch.empty(n_pages * per, dtype=torch.uint8, device="cuda") for _ in range(2)]
    b = Batch(sn, torch, [100, 3], [100, 3], page, nkv, hd)
    b.pages = np.array([[n_pages - 1, n_pages // 2, 0], [n_pages - 3, 0, 0]], np.int32)
    b.n_pages, b.max_pages = n_pages, 3
    b.d["pages"] = torch.from_numpy(b.pages.reshape(-1)).to("cuda")
    b.d["kc"], b.d["vc"] = big
    rng = np.random.default_rng(2)
    x = [torch.from_numpy(rng.standard_normal((103, nkv, hd)).astype(np.float32)).to("cuda") for _ in range(2)]
    ok(sn, sn.lib().sinter_kv4_append(C.byref(b.rec()), C.byref(heads(sn, x[0])), C.byref(heads(sn, x[1])), F32, stream(torch)), torch)
    out = [torch.zeros_like(a) for a in x]
    ok(sn, sn.lib().sinter_kv4_read(C.byref(b.rec()), C.byref(heads(sn, out[0])), C.byref(heads(sn, out[1])), F32, stream(torch)), torch)
    vals = [ref.values(*ref.quantise(a.cpu().numpy())) for a in x]
    for o, w in zip(out, vals):
        assert np.array_equal(o.cpu().numpy(), w.astype(np.float32))
    q = rng.standard_normal((103, 4, hd)).astype(np.float32)
    (_, qv), (_, ov) = strided(torch, q, F32), strided(torch, np.zeros_like(q), F32)
    a, ws = attn_args(sn, torch, b, 4, F32, qv, ov)
    ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
    b.rows = lambda s, n: [w[b.tok_start[s]:b.tok_start[s] + n].transpose(1, 0, 2) for w in vals]
    check_attn(b, 4, F32, q.astype(np.float64), ov.cpu().numpy(), None, hd ** -0.5, only=(0, 63, 64, 99, 100, 102))


class Replies:
    """Sequences served over one cache: prep, append and attention per step."""

    def __init__(self, sn, torch, t, nq, nkv, hd, page, lens, room, seed):
        self.sn, self.torch, self.t, self.nq, self.nkv, self.hd = sn, torch, t, nq, nkv, hd
        self.b = Batch(sn, torch, [0] * len(lens), [n + room for n in lens], page, nkv, hd, seed=seed)
        self.b.kv_len[:] = 0
        self.rng = np.random.default_rng(seed)
        self.wq, self.wk = (torch.from_numpy((1 + 0.1 * self.rng.standard_normal(hd)).astype(np.float32)).to("cuda") for _ in range(2))
        self.max_kv = max(lens) + room

    def buffers(self, new):
        torch, b = self.torch, self.b
        n = int(sum(new))
        b.n_tok = n
        b.tok_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        b.kv_len = (b.kv_len + np.array(new)).astype(np.int32)
        b.d["tok_start"] = torch.from_numpy(b.tok_start).to("cuda")
        b.d["kv_len"] = torch.from_numpy(b.kv_len).to("cuda")
        def mk(h):
            return torch.from_numpy(self.rng.standard_normal((n, h, self.hd)).astype(np.float32)).to("cuda").to(tdtype(torch, self.t))
        self.qg, self.k, self.v = mk(2 * self.nq).view(n, self.nq, 2 * self.hd), mk(self.nkv), mk(self.nkv)
        self.q, self.kr = torch.zeros(n, self.nq, self.hd, dtype=self.k.dtype, device="cuda"), torch.zeros_like(self.k)
        self.out = torch.full_like(self.q, 3.0)
        sn = self.sn
        self.prep = sn.Kv4PrepArgs(q=sn.Heads(self.qg.data_ptr(), self.qg.stride(0), 2 * self.hd), q_out=heads(sn, self.q),
                                   k=heads(sn, self.k), k_out=heads(sn, self.kr), q_norm=self.wq.data_ptr(),
                                   k_norm=self.wk.data_ptr(), nq=self.nq, rope_dims=self.hd // 4, rope_base=1e7, eps=1e-6, type=self.t)
        gate = self.qg[..., self.hd:]
        self.attn, self.ws = attn_args(sn, torch, b, self.nq, self.t, self.q, self.out, gate, max_kv=self.max_kv)
        self.attn.gate = sn.Heads(gate.data_ptr(), gate.stride(0), gate.stride(1))
        self.rec = b.rec()

    def launch(self):
        L, s, r = self.sn.lib(), stream(self.torch), C.byref(self.rec)
        self.sn.check(L.sinter_kv4_prep(r, C.byref(self.prep), s))
        self.sn.check(L.sinter_kv4_append(r, C.byref(heads(self.sn, self.kr)), C.byref(heads(self.sn, self.v)), self.t, s))
        self.sn.check(L.sinter_kv4_attn(r, C.byref(self.attn), s))

    def check(self):
        torch, b = self.torch, self.b
        torch.cuda.synchronize()
        assert self.sn.op_error()[0] == 0
        b.kc, b.vc = b.d["kc"].cpu().numpy(), b.d["vc"].cpu().numpy()
        # the cache holds the rotated k of this step, quantised
        pos = ref.positions(b.tok_start, b.kv_len, b.n_tok)
        code, d16 = ref.quantise(self.kr.float().cpu().numpy())
        for j, (s, p) in enumerate(pos):
            for g in range(self.nkv):
                assert np.array_equal(ref.get(b.kc, b.pages[s, p // b.page], p % b.page, g, b.page, self.nkv, self.hd),
                                      ref.values(code[j, g], d16[j, g]))
        gate = self.qg[..., self.hd:].double().cpu().numpy()
        check_attn(b, self.nq, self.t, self.q.double().cpu().numpy(), self.out.float().cpu().numpy(), gate, self.hd ** -0.5)


@pytest.mark.parametrize("t,nq,nkv,hd,page", [(F32, 6, 1, 256, 16), (BF16, 8, 2, 64, 32), (F16, 4, 4, 128, 16)])
def test_prompts_then_replies(sn, torch_gpu, t, nq, nkv, hd, page):
    """Prompts of several lengths, a second turn beside single tokens, then
    replies token by token across page ends."""
    r = Replies(sn, torch_gpu, t, nq, nkv, hd, page, [30, 3, 70], 12, seed=hd)
    for new in ([28, 2, 66], [1, 9, 1], [1, 1, 1], [3, 0, 1], [1, 1, 2], [1, 1, 1]):
        r.buffers(new)
        r.launch()
        r.check()


def test_graph_replays_follow_the_lengths(sn, torch_gpu):
    """One captured step replayed as the sequences grow, the program's own
    eager work in between; every replay equal to the eager step, bit for bit."""
    replay_steps(sn, torch_gpu, 6, 2, [20, 500], [1, 1])


def test_graph_replays_of_many_rows(sn, torch_gpu):
    replay_steps(sn, torch_gpu, 16, 1, [20, 300], [1, 20])


def replay_steps(sn, torch, nq, nkv, first, step):
    r = Replies(sn, torch, F32, nq, nkv, 64, 16, first, 40, seed=5)
    r.buffers(first)
    r.launch()
    r.check()
    r.buffers(step)
    r.launch()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r.launch()
    for step in range(6):
        r.b.kv_len += 1
        r.b.d["kv_len"] += 1
        r.qg.normal_()
        r.k.normal_()
        r.v.normal_()
        r.out.fill_(3.0)
        r.ws.fill_(0xff)
        g.replay()
        torch.cuda.synchronize()
        got, kc = r.out.clone(), r.b.d["kc"].clone()
        r.out.fill_(5.0)
        r.launch()
        torch.cuda.synchronize()
        assert torch.equal(got, r.out) and torch.equal(kc, r.b.d["kc"])
        r.check()


def test_two_streams_at_once(sn, torch_gpu):
    """Two batches over one cache on two streams, a workspace each."""
    torch = torch_gpu
    b = Batch(sn, torch, [1, 1], [2000, 1500], 64, 2, 128, seed=2)
    b.fill_rows(3)
    q = torch.randn(2, 8, 128, device="cuda")
    outs, runs = [], []
    for i in range(2):
        out = torch.zeros_like(q)
        runs.append((torch.cuda.Stream(), *attn_args(sn, torch, b, 8, F32, q, out)))
        outs.append(out)
    rec = b.rec()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, a, ws in runs:
            sn.check(sn.lib().sinter_kv4_attn(C.byref(rec), C.byref(a), C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1]) and sn.op_error()[0] == 0
    check_attn(b, 8, F32, q.double().cpu().numpy(), outs[0].cpu().numpy(), None, 128 ** -0.5)


def test_two_streams_at_once_of_many_rows(sn, torch_gpu):
    """Prompts on one stream, replies and another step's append on the other."""
    torch = torch_gpu
    many, few = Batch(sn, torch, [150, 90], [700, 300], 64, 2, 64, seed=2), Batch(sn, torch, [1, 2], [1500, 40], 64, 2, 64, seed=3)
    qs, outs, runs = [], [], []
    for b in (many, few):
        b.fill_rows(3)
        q = torch.randn(b.n_tok, 8, 64, device="cuda", dtype=torch.float16)
        out = torch.zeros_like(q)
        qs.append(q), outs.append(out)
        runs.append((torch.cuda.Stream(), b.rec(), *attn_args(sn, torch, b, 8, F16, q, out)))
    other = Batch(sn, torch, [40, 40], [40, 64], 16, 2, 64, seed=4)
    x = torch.randn(80, 2, 64, device="cuda")
    torch.cuda.synchronize()
    L = sn.lib()
    for _ in range(10):
        for s, r, a, ws in runs:
            sn.check(L.sinter_kv4_attn(C.byref(r), C.byref(a), C.c_void_p(s.cuda_stream)))
        sn.check(L.sinter_kv4_append(C.byref(other.rec()), C.byref(heads(sn, x)), C.byref(heads(sn, x)), F32, C.c_void_p(runs[1][0].cuda_stream)))
    torch.cuda.synchronize()
    assert sn.op_error()[0] == 0
    for b, q, out, n in zip((many, few), qs, outs, (11, 1)):
        check_attn(b, 8, F16, q.double().cpu().numpy(), out.float().cpu().numpy(), None, 0.125, only=set(range(0, b.n_tok, n)))


def test_same_bits_every_time(sn, torch_gpu):
    torch = torch_gpu
    b = Batch(sn, torch, [2, 1, 30], [1800, 900, 700], 64, 2, 64, seed=2)
    b.fill_rows(3)
    q = torch.randn(33, 8, 64, device="cuda")
    first = None
    for _ in range(5):
        out = torch.zeros_like(q)
        a, ws = attn_args(sn, torch, b, 8, F32, q, out)
        ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
        first = out if first is None else first
        assert torch.equal(first, out)


def test_same_bits_every_time_of_many_rows(sn, torch_gpu):
    torch = torch_gpu
    b = Batch(sn, torch, [2, 70, 90], [1800, 900, 700], 64, 2, 64, seed=2)
    b.fill_rows(3)
    q = torch.randn(162, 8, 64, device="cuda", dtype=torch.bfloat16)
    first = None
    for _ in range(5):
        out = torch.zeros_like(q)
        a, ws = attn_args(sn, torch, b, 8, BF16, q, out)
        ok(sn, sn.lib().sinter_kv4_attn(C.byref(b.rec()), C.byref(a), stream(torch)), torch)
        first = out if first is None else first
        assert torch.equal(first, out)
