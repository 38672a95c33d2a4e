"""GPU: attention over the paged 4-bit cache where keys and values differ in size, against a float64 softmax over the values that the
cache holds (read back by load, whose values are exact).

Tolerances, for a row and a 64-dim block, V the largest |v| of the block that the row sees, S the largest scale sum_d |q_d k_d| of a key
that it sees. fp32 rows: products and sums keep some 22 bits, 2e-5 V as in tests/test_kv4_gpu.py; a score is kept to 2^-20 S, which
changes a weight by that share and an output by twice that of V at most. bf16 rows: half an ulp of the output, 2^-8 |out| at
most, P and V rounded to 11 bits each (2^-10 V), and keys rounded to 11 bits (2^-12 of each product, 2^-11 S V).
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def kv4(fn):
    import kv4 as m
    return m


@pytest.fixture(scope="module")
def ws(fn, kv4):
    return kv4.KV4Workspace(fn)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """One request of `length` tokens, keys [length][nkv][hd] and values of any sizes, its last `new` tokens as rows."""

    def __init__(self, fn, kv4, ws, k, v, q, bs=16, dtype="f32"):
        self.length, self.nkv, self.hd = k.shape
        n = -(-self.length // bs)
        perm = torch.randperm(n, generator=torch.Generator().manual_seed(1))
        self.c = kv4.KV4Cache(fn, self.nkv, self.hd, bs, n, ws)
        self.table = perm.to(torch.int32).cuda()[None].contiguous()
        slots = (perm[:, None] * bs + torch.arange(bs)[None]).reshape(-1)[:self.length].cuda()
        self.c.store(torch.from_numpy(k).float().cuda(), torch.from_numpy(v).float().cuda(), slots)
        self.q = torch.from_numpy(q).float().cuda().to(DT[dtype])
        self.k, self.v = (x.double().cpu().numpy() for x in self.c.load(slots))
        self.fn, self.dtype, self.new = fn, dtype, q.shape[0]

    def run(self, scale=None, max_new=None):
        out = self.c.attn(self.q, i32(0, self.new), i32(self.length), self.table, max_new or self.new, scale=scale)
        self.fn.sync(torch.cuda.current_stream().cuda_stream)
        return out.double().cpu().numpy()

    def rows(self, scale=None):
        """Per row and head: what it should be [hd], V per block, S."""
        scale = 1 / np.sqrt(self.hd) if scale is None else scale
        q = self.q.double().cpu().numpy()
        group = q.shape[1] // self.nkv
        for i in range(self.new):
            see = self.length - self.new + i + 1
            for h in range(q.shape[1]):
                k, v = self.k[:see, h // group], self.v[:see, h // group]
                s = scale * (k @ q[i, h])
                p = np.exp(s - s.max())
                yield i, h, p @ v / p.sum(), np.abs(v).reshape(see, -1, 64).max((0, 2)), abs(scale) * (np.abs(k) @ np.abs(q[i, h])).max()

    def check(self, scale=None, max_new=None, cap=None):
        """cap: rows whose S is above it are only looked at for finite outputs."""
        got, worst = self.run(scale, max_new), 0.0
        assert np.isfinite(got).all()
        for i, h, want, V, S in self.rows(scale):
            if cap is not None and S > cap:
                continue
            V = np.repeat(V, 64)
            if self.dtype == "f32":
                tol = (2e-5 + 2.0 ** -19 * S) * V
            else:
                tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -10 + 2.0 ** -11 * S) * V
            worst = max(worst, float((np.abs(got[i, h] - want) / np.maximum(tol, 1e-300)).max()))
        assert worst <= 1, worst


# new tokens, heads of a group: the two forms of the kernel for few rows, the kernel for prompts
FORMS = [pytest.param(1, 8, id="one"), pytest.param(5, 3, id="few"), pytest.param(70, 2, id="prompt")]


def normal(rng, *shape):
    return rng.standard_normal(shape)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", FORMS)
@pytest.mark.parametrize("size", [1e-6, 1e-5, 1e-4, 1e-3, 1.0, 1e3, 3e4])
def test_keys_of_any_size(fn, kv4, ws, size, new, group, dtype):
    """Scores of the same spread from keys of any size. (Scales below fp16's normal numbers have few bits; those are the cache's values.)"""
    rng = np.random.default_rng(1)
    q = normal(rng, new, 2 * group, 128) * 2 / size
    Case(fn, kv4, ws, normal(rng, 150, 2, 128) * size, normal(rng, 150, 2, 128), q, dtype=dtype).check()


@pytest.mark.parametrize("new, group", FORMS)
@pytest.mark.parametrize("scale", [0.3, -0.1, 0.0, -0.0, 1e-20])
def test_scales_given(fn, kv4, ws, scale, new, group):
    rng = np.random.default_rng(2)
    for size in (1e-4, 1.0):
        q = normal(rng, new, 2 * group, 64) / size
        Case(fn, kv4, ws, normal(rng, 100, 2, 64) * size, normal(rng, 100, 2, 64), q, bs=32).check(scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", FORMS)
@pytest.mark.parametrize("hd, spread", [(64, 2.0), (128, 4.0), (256, 3.0)])
def test_keys_of_sizes_beside_each_other(fn, kv4, ws, hd, spread, new, group, dtype):
    """Tokens whose keys differ by powers of ten, within a tile too: the scores stay right beside each other."""
    rng = np.random.default_rng(3)
    k = normal(rng, 200, 1, hd) * 10 ** rng.uniform(-spread, 0, (200, 1, 1))
    Case(fn, kv4, ws, k, normal(rng, 200, 1, hd), normal(rng, new, group, hd) * 2, dtype=dtype).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", FORMS)
@pytest.mark.parametrize("hd, spread", [(64, 6.0), (128, 3.0), (256, 8.0)])
def test_values_of_sizes_beside_each_other(fn, kv4, ws, hd, spread, new, group, dtype):
    """Tokens, and 64-dim blocks, whose values differ by powers of ten: each block keeps its precision."""
    rng = np.random.default_rng(4)
    v = normal(rng, 200, 1, hd) * 10 ** rng.uniform(-spread / 2, spread / 2, (200, 1, 1))
    v = np.clip((v.reshape(200, 1, -1, 64) * 10.0 ** rng.uniform(-2, 2, (1, 1, hd // 64, 1))).reshape(200, 1, hd), -5e5, 5e5)
    Case(fn, kv4, ws, normal(rng, 200, 1, hd), v, normal(rng, new, group, hd), dtype=dtype).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", FORMS)
@pytest.mark.parametrize("block", [1e-1, 1e-2, 1e-3, 1e-4])
def test_blocks_of_small_values_beside_large_ones(fn, kv4, ws, block, new, group, dtype):
    """One 64-dim block of every token is smaller: its outputs are right to their own size. Few tokens, whose errors do not average out,
    and small scores, whose errors would cover it."""
    rng = np.random.default_rng(5)
    for length in (new + 2, new + 100):
        v = normal(rng, length, 1, 256)
        v[..., 64:128] *= block
        Case(fn, kv4, ws, normal(rng, length, 1, 256), v, normal(rng, new, group, 256) * 0.05, dtype=dtype).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", [pytest.param(5, 3, id="few"), pytest.param(70, 2, id="prompt")])
@pytest.mark.parametrize("base, factor", [(0.05, 1e6), (1e-3, 1e4), (1e-3, 1e6), (1e-3, 1e8)])
def test_values_hidden_from_a_row_do_not_matter(fn, kv4, ws, base, factor, new, group, dtype):
    """The last token's values (one block of them in the second case) are far larger; the rows before it do not see them."""
    rng = np.random.default_rng(6)
    for dims in (slice(0, 128), slice(64, 128)):
        v = normal(rng, 128, 1, 128) * base
        v[-1, 0, dims] *= factor
        v = np.clip(v, -5e5, 5e5)  # scales within fp16
        Case(fn, kv4, ws, normal(rng, 128, 1, 128), v, normal(rng, new, group, 128), dtype=dtype).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", [pytest.param(5, 3, id="few"), pytest.param(70, 2, id="prompt")])
@pytest.mark.parametrize("factor", [1e4, 1e6, 1e8])
def test_keys_hidden_from_a_row_do_not_matter(fn, kv4, ws, factor, new, group, dtype):
    rng = np.random.default_rng(7)
    k = normal(rng, 128, 1, 128) * 1e-3
    k[-1] = np.clip(k[-1] * factor, -5e5, 5e5)
    q = normal(rng, new, group, 128) * 1e3
    Case(fn, kv4, ws, k, normal(rng, 128, 1, 128), q, dtype=dtype).check(cap=1e3)


@pytest.mark.parametrize("new, group", FORMS)
@pytest.mark.parametrize("factor", [1e2, 1e5, 1e8])
def test_large_values_of_no_weight(fn, kv4, ws, factor, new, group):
    """A token that everyone sees, whose values are large and whose weight is nothing beside the others': the kernel for prompts keeps
    the precision of what counts. The one for few rows is held to the largest value seen."""
    rng = np.random.default_rng(8)
    k, v = normal(rng, 128, 1, 128) * 0.1, normal(rng, 128, 1, 128) * 1e-3
    q = np.abs(normal(rng, new, group, 128)) + 1
    k[20], v[20] = -20.0, v[20] * factor  # scores of -200 and less
    c = Case(fn, kv4, ws, k, v, q)
    c.check()
    if new >= 64:
        got = c.run()
        for i, h, want, _, S in c.rows():
            # without that token the largest |v| is 5e-3 and S is at most a fortieth (keys of 0.5 beside its 20)
            assert np.abs(got[i, h] - want).max() <= (2e-5 + 2.0 ** -19 * S / 40) * 5e-3


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", FORMS)
@pytest.mark.parametrize("qsize", [1e5, 1e7, 3e7, 1e8, 1e9, 1e12])
def test_scores_of_any_size(fn, kv4, ws, qsize, new, group, dtype):
    """Scores of up to 1e13: the row is its best key's value where that key's lead passes the scores' rounding (2^-18 S)."""
    rng = np.random.default_rng(9)
    c = Case(fn, kv4, ws, normal(rng, 150, 1, 64), normal(rng, 150, 1, 64), normal(rng, new, group, 64) * qsize, dtype=dtype)
    got, q, led = c.run(), c.q.double().cpu().numpy(), 0
    assert np.isfinite(got).all()
    for i, h, want, V, S in c.rows():
        s = np.sort(c.k[:c.length - new + i + 1, 0] @ q[i, h] / 8)
        if s[-1] - s[-2] > (2.0 ** -18 if dtype == "f32" else 2.0 ** -10) * S + 60:
            led += 1
            tol = (2e-5 if dtype == "f32" else 2.0 ** -8) * V[0]
            assert np.abs(got[i, h] - want).max() <= tol, (i, h)
    assert led > 0


def test_nan_and_infinite_values_beside_sizes(fn, kv4, ws):
    """What is not finite reaches the rows that see it, whatever the sizes around it are."""
    rng = np.random.default_rng(10)
    for new, group in ((5, 3), (70, 2)):
        k, v = normal(rng, 128, 1, 128), normal(rng, 128, 1, 128) * 10 ** rng.uniform(-4, 4, (128, 1, 1))
        bad = 125
        v[bad, 0, 70] = np.nan
        c = Case(fn, kv4, ws, k, v, normal(rng, new, group, 128))
        got = c.run()
        sees = np.arange(128 - new, 128) >= bad
        assert np.isnan(got[sees][..., 64:]).all() and np.isfinite(got[sees][..., :64]).all() and np.isfinite(got[~sees]).all()
        # a key that is not finite: all of the rows that see it, none before
        k[bad, 0, 3] = np.inf
        c = Case(fn, kv4, ws, k, normal(rng, 128, 1, 128), normal(rng, new, group, 128))
        got = c.run()
        assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()


@pytest.mark.parametrize("lead", [100.0, 300.0])
def test_a_nan_value_of_no_weight_is_seen(fn, kv4, ws, lead):
    """0 x NaN is NaN, in a tile that some rows see a part of as in one that all see: both kernels agree."""
    rng = np.random.default_rng(11)
    for new, group, length in ((1, 4, 20), (1, 4, 64), (3, 4, 60), (70, 2, 100), (70, 2, 128)):
        k, v = normal(rng, length, 1, 64) * 1e-3, normal(rng, length, 1, 64)
        q = np.ones((new, group, 64))
        k[5], v[5, 0, 9] = -lead / 8, np.nan  # scale sum q k = 64 k / 8
        got = Case(fn, kv4, ws, k, v, q).run()
        sees = np.arange(length - new, length) >= 5
        assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all(), (new, length)


def test_long_sums_of_one_sign_keep_bf16_rows(fn, kv4, ws):
    """Flat rows over two million tokens, one request to a CTA, all products of one sign: a sum that were cut at every step would
    end low by 1e-3 and more. Averaged over 512 outputs, whose own rounding (2^-9 at most, spread) then counts 2^-9 / sqrt(512),
    twice that allowed; the weights' common rounding to 11 bits is 2^-12."""
    tokens, bs, hd, n = 1 << 21, 64, 64, 444
    c = kv4.KV4Cache(fn, 1, hd, bs, tokens // bs, ws)
    g = torch.Generator("cuda").manual_seed(3)
    v = -0.55 - 0.4 * torch.arange(hd, device="cuda") / hd + 0.1 * torch.rand(tokens, 1, hd, device="cuda", generator=g)
    v[..., 17] = 1.1  # the value of largest magnitude: the others' codes are 11 to 15 of 15
    k = torch.zeros(tokens, 1, hd, device="cuda")
    slots = torch.arange(tokens, device="cuda")
    c.store(k, v, slots)
    table = torch.arange(tokens // bs, dtype=torch.int32, device="cuda")[None].expand(n, -1).contiguous()
    q = torch.randn(n, 8, hd, device="cuda", generator=g).bfloat16()
    out = c.attn(q, torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.full((n,), tokens, dtype=torch.int32, device="cuda"),
                 table, 1).double()
    fn.sync(torch.cuda.current_stream().cuda_stream)
    want = c.load(slots)[1].double().mean((0, 1))
    rel = (out / want - 1)[..., torch.arange(hd) != 17]
    # every request has the same answer; its 8 x 63 outputs round alike, so the dims are what is averaged over
    tol = 2.0 ** -12 + 2 * 2.0 ** -9 / 63 ** 0.5
    assert float(rel.mean((1, 2)).abs().max()) <= tol, rel.mean()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new, group", FORMS)
def test_outputs_in_the_place_of_the_rows(fn, kv4, ws, new, group, dtype):
    """out is q's own memory: the same values, also where the kernel for prompts has to do a call again (values past 65504)."""
    rng = np.random.default_rng(12)
    for size in (1.0, 2e5):
        v = np.clip(normal(rng, 300, 1, 128) * size, -5e5, 5e5)  # scales within fp16
        c = Case(fn, kv4, ws, normal(rng, 300, 1, 128), v, normal(rng, new, group, 128), dtype=dtype)
        c.check()
        want, q = c.run(), c.q.clone()
        c.c.attn(q, i32(0, new), i32(300), c.table, new, out=q)
        fn.sync(torch.cuda.current_stream().cuda_stream)
        # another form of the kernel may round apart by twice what each is allowed
        tol = (4e-5 + 2.0 ** -18 * 10 if dtype == "f32" else 2.0 ** -6) * 5 * size
        assert np.abs(q.double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, bs", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("large", ["values", "keys", "scores", "none"])
def test_many_prompts_with_large_values(fn, kv4, ws, hd, bs, dtype, large):
    """Several row tiles and some 70 tiles to a CTA, split row tiles among them, with scales past 8188 here and there: both forms of the
    kernel for prompts over long runs."""
    n, nkv, group, new, length = 4, 4, 2, 600, 1500
    g = torch.Generator("cuda").manual_seed(hd)
    per = -(-length // bs)
    table = torch.randperm(n * per, generator=torch.Generator().manual_seed(2)).to(torch.int32).reshape(n, per).cuda()
    slots = (table.long()[:, :, None] * bs + torch.arange(bs, device="cuda")).reshape(n, -1)[:, :length].contiguous()
    k, v = torch.randn(2, n, length, nkv, hd, device="cuda", generator=g)
    few = (torch.rand(n, length, nkv, 1, device="cuda", generator=g) < 0.01).float()
    q = torch.randn(n * new, nkv * group, hd, device="cuda", generator=g) * (1e7 if large == "scores" else 0.5)
    if large == "values":
        v *= 1 + 1e5 * few
    if large == "keys":  # tiny but for a few, which only some rows weigh
        k *= 1e-3 + 1e5 * few
        q *= 1e-5
    c = kv4.KV4Cache(fn, nkv, hd, bs, n * per, ws)
    c.store(k.flatten(0, 1), v.flatten(0, 1), slots.flatten())
    q = q.to(DT[dtype])
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda") * new
    args = (cu, torch.full((n,), length, dtype=torch.int32, device="cuda"), table, new)
    out = c.attn(q, *args)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out, c.attn(q, *args))  # the same bits again
    hide = torch.arange(length, device="cuda")[None, :] > torch.arange(length - new, length, device="cuda")[:, None]
    for r in range(n):
        lk, lv = (x.double() for x in c.load(slots[r]))
        for h in range(nkv * group):
            qh, kh, vh = q[r * new:(r + 1) * new, h].double(), lk[:, h // group], lv[:, h // group]
            s = (qh @ kh.T / hd ** 0.5).masked_fill(hide, float("-inf"))
            want = torch.softmax(s, -1) @ vh
            S = (qh.abs() @ kh.abs().T / hd ** 0.5).masked_fill(hide, 0.0).amax(-1, keepdim=True)
            V = torch.cummax(vh.abs().reshape(length, -1, 64).amax(-1), 0).values[length - new:].repeat_interleave(64, 1)
            got = out[r * new:(r + 1) * new, h].double()
            assert got.isfinite().all()
            if dtype == "f32":
                tol = (2e-5 + 2.0 ** -19 * S) * V
            else:
                tol = 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2.0 ** -11 * S) * V
            if large != "scores":
                assert ((got - want).abs() <= tol).all(), (r, h)
            else:  # rows whose best key leads by more than the scores' rounding are its value
                two = s.topk(2, -1).values
                led = two[:, 0] - two[:, 1] > (2.0 ** -18 if dtype == "f32" else 2.0 ** -10) * S[:, 0] + 60
                assert led.any() and ((got - want).abs()[led] <= ((2e-5 if dtype == "f32" else 2.0 ** -8) * V)[led]).all(), (r, h)


@pytest.mark.parametrize("new, group", FORMS)
def test_rows_and_outputs_as_columns_of_one_buffer(fn, kv4, ws, new, group):
    """q, gate and out beside each other in the rows of one buffer: the same bits as apart."""
    rng = np.random.default_rng(13)
    c = Case(fn, kv4, ws, normal(rng, 300, 1, 128), normal(rng, 300, 1, 128), normal(rng, new, group, 128))
    a = (i32(0, new), i32(300), c.table, new)
    gate = torch.from_numpy(normal(rng, new, group, 128)).float().cuda()
    want = c.c.attn(c.q, *a, gate=gate)
    w = group * 128
    for order in ((0, 1, 2), (2, 0, 1), (1, 2, 0)):
        buf = torch.zeros(new, 3 * w, device="cuda")
        q, g, out = (buf[:, i * w:(i + 1) * w].unflatten(1, (group, 128)) for i in order)
        q.copy_(c.q)
        g.copy_(gate)
        c.c.attn(q, *a, gate=g, out=out)
        fn.sync(torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out, want) and torch.equal(q, c.q) and torch.equal(g, gate)


@pytest.mark.parametrize("new, group", [(1, 8), (6, 2)])
def test_flat_rows_over_long_contexts(fn, kv4, ws, new, group):
    """fp32 rows whose weights are spread over 60000 tokens, none near the largest: errors of a weight (exp2's 2^-22.5, its two halves' 2^-23
    of the largest among 32 tokens) average out as the output itself does, which is some 2.5 times below the sum that the codes' 8 is
    taken back from: 2.5 x 2^-22 = 6e-7 of the output's norm, 1e-6 allowed."""
    n, nkv, hd, bs, length = 2, 1, 64, 64, 60000
    per = -(-length // bs)
    c = kv4.KV4Cache(fn, nkv, hd, bs, n * per, ws)
    g = torch.Generator("cuda").manual_seed(1)
    k, v = torch.randn(2, n * per * bs, nkv, hd, device="cuda", generator=g)
    slots = torch.arange(n * per * bs, device="cuda")
    c.store(k, v, slots)
    q = torch.randn(n * new, nkv * group, hd, device="cuda", generator=g)
    table = torch.arange(n * per, dtype=torch.int32, device="cuda").reshape(n, per)
    out = c.attn(q, i32(0, new, 2 * new), i32(length, length), table, new).double()
    fn.sync(torch.cuda.current_stream().cuda_stream)
    hide = torch.arange(length, device="cuda")[None, :] > torch.arange(length - new, length, device="cuda")[:, None]
    for r in range(n):
        lk, lv = (x[:, 0].double() for x in c.load(slots[r * per * bs:r * per * bs + length]))
        for h in range(group):
            rows = slice(r * new, (r + 1) * new)
            s = (q[rows, h].double() @ lk.T / 8).masked_fill(hide, float("-inf"))
            want = torch.softmax(s, -1) @ lv
            assert float((out[rows, h] - want).norm() / want.norm()) <= 1e-6
