"""Host parts of the latent-attention operators: the rotary table, and what the
C entries and the binding refuse."""
import ctypes
import math

import numpy as np
import pytest
import torch

P = ctypes.c_void_p


def at(i):
    """An aligned address far from those of other i: what is refused is refused before use."""
    return (i + 1) << 44


def refused(nvb, code, overlap=False):
    message = nvb.library().nvb_last_error().decode()
    return code == -1 and ("overlaps" in message) == overlap and message != ""


# ------------------------------------------------------------ rotary table
def angles(positions, dim, theta, change=lambda f: f):
    f = change(theta ** (-2.0 * np.arange(dim // 2) / dim))
    return np.arange(positions)[:, None] * f


def assert_table(table, angle, magnitude=1.0):
    # one rounding to FP32 of a 64-bit cosine; the angle's own rounding is 2^-53 of it
    want = np.concatenate([np.cos(angle), np.sin(angle)], 1) * magnitude
    assert np.abs(table.astype(np.float64) - want).max() <= magnitude * (2.0 ** -24 + angle.max() * 2.0 ** -50)


@pytest.mark.parametrize("positions, dim, theta", [(1, 2, 10000.0), (5, 64, 10000.0), (3000, 64, 1e6), (70, 128, 500.0)])
def test_rope_table(nvb, positions, dim, theta):
    table = nvb.host.rope_table(positions, dim, theta)
    assert table.shape == (positions, dim) and table.dtype == np.float32
    assert_table(table, angles(positions, dim, theta))


def test_rope_table_scalings(nvb):
    table = nvb.host.rope_table
    n, dim, theta, orig = 500, 64, 10000.0, 4096.0
    assert_table(table(n, dim, theta, "linear", 8.0), angles(n, dim, theta) / 8.0)
    assert_table(table(n, dim, theta, "base", 4.0), angles(n, dim, theta * 4.0 ** (64 / 62)))

    def by_wavelength(f):
        turns = orig * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0, 1)
        return f * keep + f / 8.0 * (1 - keep)

    assert_table(table(n, dim, theta, "wavelength", 8.0, orig, 1.0, 4.0), angles(n, dim, theta, by_wavelength))

    def by_pair(f):
        at = [dim * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        slowed = np.clip((np.arange(dim // 2) - lo) / (hi - lo), 0, 1)
        return f * (1 - slowed) + f / 40.0 * slowed

    got = table(n, dim, theta, "yarn", 40.0, orig, 1.0, 32.0, magnitude=1.25)
    assert_table(got, angles(n, dim, theta, by_pair), 1.25)
    # a factor of one changes nothing
    for kind in ("linear", "base", "wavelength", "yarn"):
        assert np.array_equal(table(n, dim, theta, kind, 1.0, orig, 1.0, 32.0), table(n, dim, theta))


@pytest.mark.parametrize("original, slow", [(4, 1.0), (60, 20.0), (4096, 5000.0)])
def test_rope_table_by_pair_where_every_pair_is_slow(nvb, original, slow):
    # the first pair turns original / (2 pi) times, fewer than `slow`, by more than a pair: all are divided
    assert 64 * math.log(original / (slow * 2 * math.pi)) / (2 * math.log(10000.0)) < -1
    got = nvb.host.rope_table(300, 64, 10000.0, "yarn", 8.0, original, slow, 2 * slow)
    assert_table(got, angles(300, 64, 10000.0) / 8.0)


@pytest.mark.parametrize("bad", [dict(positions=0), dict(dim=3), dict(dim=0), dict(theta=1.0), dict(theta=math.inf),
                                 dict(scaling="other"), dict(scaling="linear", factor=0.5),
                                 dict(scaling="base", factor=math.nan), dict(scaling="base", factor=2.0, dim=2),
                                 dict(scaling="yarn", factor=2.0),
                                 dict(scaling="yarn", factor=2.0, original_positions=10, slow=4.0, fast=4.0),
                                 dict(scaling="wavelength", factor=2.0, original_positions=10, slow=0.0),
                                 dict(magnitude=math.inf)])
def test_rope_table_refusals(nvb, bad):
    with pytest.raises(nvb.host.HostError):
        nvb.host.rope_table(**{**dict(positions=4, dim=64, theta=10000.0), **bad})


# --------------------------------------------------------------- C entries
def store(nvb, **kw):
    a = dict(kv=at(0), kv_stride=576, weight=at(1), positions=at(2), slots=at(3), cache=at(4), q=at(5), qr=192, qh=64, out=at(6), outr=1024,
             outh=64, rows=2, heads=2, inter=0, bs=64, blocks=2, eps=1e-6, table=at(7), maxp=4)
    a.update(kw)
    return nvb.library().nvb_latent_store(
        None, a["kv"], a["kv_stride"], a["weight"], a["positions"], a["slots"], a["cache"], a["q"], a["qr"], a["qh"],
        a["out"], a["outr"], a["outh"], a["rows"], a["heads"], a["inter"], a["bs"], a["blocks"], a["eps"], a["table"],
        a["maxp"])


@pytest.mark.parametrize("bad", [
    dict(kv=None, q=None), dict(positions=None), dict(table=None), dict(weight=None), dict(slots=None),
    dict(cache=None), dict(out=None), dict(rows=0), dict(heads=0), dict(heads=1025), dict(maxp=0), dict(bs=0),
    dict(blocks=0), dict(bs=65536, blocks=65536), dict(eps=-1.0), dict(eps=0.0), dict(eps=math.nan), dict(kv_stride=568),
    dict(kv_stride=580), dict(qr=100), dict(qh=-64), dict(outr=96), dict(outh=32), dict(outr=64, outh=64),
    dict(outr=1024, outh=1024), dict(outr=2 ** 40), dict(kv=at(60) + 2), dict(q=at(60) + 8), dict(out=at(60) + 8),
    dict(cache=at(60) + 8), dict(table=at(60) + 4), dict(positions=at(60) + 2), dict(slots=at(60) + 1),
    dict(rows=2 ** 31 - 1, outr=64, outh=2 ** 31 - 8)])
def test_store_refusals(nvb, bad):
    assert refused(nvb, store(nvb, **bad))


def gather(nvb, **kw):
    a = dict(cache=at(0), table=at(1), cu=at(2), latent=at(3), ls=512, rope=at(4), rs=64, batch=1, total=1, bs=64, stride=1, blocks=1)
    a.update(kw)
    return nvb.library().nvb_latent_gather(None, a["cache"], a["table"], a["cu"], a["latent"], a["ls"], a["rope"],
                                           a["rs"], a["batch"], a["total"], a["bs"], a["stride"], a["blocks"])


@pytest.mark.parametrize("bad", [
    dict(cache=None), dict(table=None), dict(cu=None), dict(latent=None), dict(rope=None), dict(batch=0),
    dict(batch=65536), dict(total=0), dict(bs=0), dict(stride=0), dict(blocks=0), dict(bs=2 ** 16, blocks=2 ** 16),
    dict(ls=504), dict(ls=516), dict(rs=32), dict(rs=66), dict(cache=at(60) + 8), dict(latent=at(60) + 2), dict(rope=at(60) + 8),
    dict(table=at(60) + 2), dict(cu=at(60) + 1)])
def test_gather_refusals(nvb, bad):
    assert refused(nvb, gather(nvb, **bad))


def absorbed(nvb, **kw):
    L = nvb.library()
    a = dict(q=at(0), cache=at(1), out=at(2), cu=at(3), lens=at(4), table=at(5), batch=1, total=1, max_q=1, heads=16, bs=64, stride=1,
             blocks=1, scale=1.0, lse=None, scratch=at(6), floats=L.nvb_latent_scratch_floats(1))
    a.update(kw)
    return L.nvb_paged_latent_fwd(None, a["q"], a["cache"], a["out"], a["cu"], a["lens"], a["table"], a["batch"],
                                  a["total"], a["max_q"], a["heads"], a["bs"], a["stride"], a["blocks"], a["scale"],
                                  a["lse"], a["scratch"], a["floats"])


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(cache=None), dict(out=None), dict(cu=None), dict(lens=None), dict(table=None),
    dict(scratch=None), dict(batch=0), dict(batch=65536), dict(total=0), dict(max_q=0), dict(heads=0), dict(heads=257),
    dict(bs=0), dict(bs=32), dict(bs=96), dict(stride=0), dict(bs=2 ** 16, stride=2 ** 16),
    dict(total=2 ** 30, heads=16), dict(blocks=0), dict(bs=2 ** 16, blocks=2 ** 16), dict(scale=0.0),
    dict(scale=math.nan), dict(scale=math.inf), dict(scale=-1.0), dict(q=at(60) + 8), dict(cache=at(60) + 2), dict(out=at(60) + 8),
    dict(scratch=at(60) + 4), dict(cu=at(60) + 2), dict(lens=at(60) + 1), dict(table=at(60) + 2), dict(lse=at(60) + 2), dict(floats=0),
    dict(floats=-5)])
def test_absorbed_refusals(nvb, bad):
    assert refused(nvb, absorbed(nvb, **bad))


def test_scratch_goes_by_the_sms(nvb):
    floats = nvb.library().nvb_latent_scratch_floats
    assert floats(0) == floats(-1) == floats(1025) == 0
    assert floats(1) > 0 and floats(148) == 148 * floats(1)


def expanded(nvb, **kw):
    a = dict(q=at(0), kv=at(1), rope=at(2), rs=64, out=at(3), cu_q=at(4), cu_k=at(5), batch=1, total_q=1, total_k=1, max_q=1, heads=16,
             scale=1.0, lse=None)
    a.update(kw)
    return nvb.library().nvb_latent_prefill_fwd(None, a["q"], a["kv"], a["rope"], a["rs"], a["out"], a["cu_q"],
                                                a["cu_k"], a["batch"], a["total_q"], a["total_k"], a["max_q"],
                                                a["heads"], a["scale"], a["lse"])


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(kv=None), dict(rope=None), dict(out=None), dict(cu_q=None), dict(cu_k=None), dict(batch=0),
    dict(batch=65536), dict(total_q=0), dict(total_k=0), dict(max_q=0), dict(heads=0), dict(heads=257),
    dict(total_q=2 ** 30), dict(rs=56), dict(rs=68), dict(rs=2 ** 40), dict(scale=0.0), dict(scale=math.nan),
    dict(q=at(60) + 8), dict(kv=at(60) + 2), dict(rope=at(60) + 8), dict(out=at(60) + 4), dict(cu_q=at(60) + 2), dict(cu_k=at(60) + 1),
    dict(lse=at(60) + 3)])
def test_expanded_refusals(nvb, bad):
    assert refused(nvb, expanded(nvb, **bad))


# --------------------------------------------------------------- overlaps
@pytest.mark.parametrize("bad", [
    dict(cache=at(0)), dict(cache=at(0) - 64 * 2 * 1152 + 16), dict(out=at(0) + 1024), dict(q=at(6), qr=1152),
    dict(q=at(6) + 128), dict(q=at(4) + 16), dict(table=at(6) + 2048 + 112), dict(positions=at(4)),
    dict(slots=at(6) + 4), dict(weight=at(4) + 64 * 2 * 1152 - 16)])
def test_store_overlaps(nvb, bad):
    assert refused(nvb, store(nvb, **bad), overlap=True)


# queries and latents in rows of one projection, 10 heads of 192 and the 576 of kv in either order: what fits is only
# refused for its number of rows, looked at last
@pytest.mark.parametrize("q, kv, stride, fits", [
    (256, 3840, 2496, True), (1152 + 256, 0, 2496, True), (0, 3600, 2496, True), (256, 3824, 2496, False),
    (256, 3856, 2496, True),   # kv ends at element 2504, the next row's first part begins at 2496 + 128
    (256, 3840, 2488, True),   # 2496 and 2488 + 128
    (256, 3840, 2368, True), (256, 3840, 2360, False),  # 2496 and 2368 + 128, 2360 + 128
    (1152 - 16, 0, 2496, False), (1152 + 256, 0, 2488, False)])
def test_store_of_one_projection(nvb, q, kv, stride, fits):
    part = dict(q=at(8) + q, qr=stride, qh=192, out=at(8) + q, outr=stride, outh=192, heads=10)
    code = store(nvb, rows=2 ** 31 - 1, kv=at(8) + kv, kv_stride=stride, **part)
    assert refused(nvb, code, overlap=not fits)
    assert not fits or "too many rows" in nvb.library().nvb_last_error().decode()


@pytest.mark.parametrize("bad", [
    dict(latent=at(0)), dict(rope=at(0) + 64 * 1152 - 16), dict(rope=at(3) + 16), dict(rope=at(3) + 1008),
    dict(latent=at(4) - 16), dict(total=3, ls=576, rs=576, rope=at(3) + 1008),
    dict(total=3, ls=576, rs=576, rope=at(3) + 1040), dict(total=3, ls=576, rs=584, rope=at(3) + 1024),
    dict(cu=at(3)), dict(table=at(4) + 124)])
def test_gather_overlaps(nvb, bad):
    assert refused(nvb, gather(nvb, **bad), overlap=True)


@pytest.mark.parametrize("bad", [
    dict(out=at(0)), dict(out=at(0) + 16 * 1152 - 16), dict(out=at(1) - 16), dict(scratch=at(2) + 16 * 1024 - 16),
    dict(lse=at(6) + 64), dict(lse=at(2)), dict(cu=at(2) + 4), dict(lens=at(6)), dict(table=at(2) + 8),
    dict(scratch=at(1) + 64 * 1152 - 16)])
def test_absorbed_overlaps(nvb, bad):
    assert refused(nvb, absorbed(nvb, **bad), overlap=True)


@pytest.mark.parametrize("bad", [
    dict(out=at(0) + 16), dict(out=at(1) + 16 * 512 - 16), dict(out=at(2) + 112), dict(lse=at(3) + 4),
    dict(cu_q=at(3)), dict(cu_k=at(3) + 16 * 256 - 4), dict(total_k=5, rs=576, out=at(2) + 4 * 1152 + 112)])
def test_expanded_overlaps(nvb, bad):
    assert refused(nvb, expanded(nvb, **bad), overlap=True)


# ------------------------------------------------- the binding's own checks
@pytest.mark.gpu
def test_the_binding_refuses_what_does_not_fit(nvb):
    bf, i32 = dict(dtype=torch.bfloat16, device="cuda"), dict(dtype=torch.int32, device="cuda")
    cache, table = torch.zeros(4, 64, 576, **bf), torch.zeros(1, 2, **i32)
    cu, lens = torch.tensor([0, 1], **i32), torch.tensor([1], **i32)
    q, out = torch.zeros(1, 16, 576, **bf), torch.zeros(1, 16, 512, **bf)
    scratch = nvb.latent_scratch("cuda")
    good = dict(q=q, cache=cache, out=out, cu_q=cu, kv_lens=lens, block_table=table, max_q=1, scale=1.0, scratch=scratch)
    nvb.paged_latent_fwd(**good)
    for bad in (dict(q=q.float()), dict(q=q[..., :512]), dict(cache=cache[..., :512]), dict(cache=cache.cpu()),
                dict(out=q), dict(cu_q=cu.long()), dict(kv_lens=lens[:0]), dict(block_table=table[0]),
                dict(out=cache.view(-1)[:16 * 512].view(1, 16, 512)), dict(scratch=scratch[:100]),
                dict(lse=torch.zeros(1, 15, device="cuda")), dict(cache=torch.zeros(4, 32, 576, **bf))):
        with pytest.raises(nvb.NvbError):
            nvb.paged_latent_fwd(**{**good, **bad})
    rope_table, weight = torch.zeros(8, 64, device="cuda"), torch.ones(512, **bf)
    kv, heads = torch.zeros(2, 576, **bf), torch.zeros(2, 4, 192, **bf)
    good = dict(kv=kv, weight=weight, positions=torch.zeros(2, **i32), slots=torch.arange(2, **i32), cache=cache,
                rope_table=rope_table, q=heads[..., 128:])
    nvb.latent_store(**good)
    for bad in (dict(kv=None), dict(kv=kv[:, :575]), dict(kv=kv.T.contiguous().T), dict(weight=weight[:256]),
                dict(q=heads[..., :128]), dict(q_out=heads[..., 120:184]), dict(q_out=heads[:1, :, :64]),
                dict(cache=cache.transpose(0, 1)), dict(rope_table=rope_table[:, :32]), dict(positions=None),
                dict(q=None, q_out=heads[..., 128:]), dict(kv=cache.view(-1, 576)[:2]), dict(q=heads[..., 1:65])):
        with pytest.raises((nvb.NvbError, AttributeError)):
            nvb.latent_store(**{**good, **bad})
    latent, rope = torch.zeros(5, 512, **bf), torch.zeros(5, 64, **bf)
    wide = torch.zeros(5, 576, **bf)
    cu5 = torch.tensor([0, 5], **i32)
    nvb.latent_gather(cache, table, cu5, latent, rope)
    nvb.latent_gather(cache, table, cu5, wide[:, :512], wide[:, 512:])
    for args in ((cache, table, cu5, latent, rope[:4]), (cache, table, cu5, latent, latent[:, :64]),
                 (cache, table, cu5, cache.view(-1, 576)[:5, :512], rope), (cache, table, cu5[:1], latent, rope),
                 (cache, table, cu5, wide[:, :512], wide[:, 448:512])):
        with pytest.raises(nvb.NvbError):
            nvb.latent_gather(*args)
    q, kv, out = torch.zeros(3, 2, 192, **bf), torch.zeros(5, 2, 256, **bf), torch.zeros(3, 2, 128, **bf)
    good = dict(q=q, kv=kv, k_rope=rope, out=out, cu_q=torch.tensor([0, 3], **i32), cu_k=cu5, max_q=3, scale=1.0)
    nvb.latent_prefill_fwd(**good)
    for bad in (dict(q=q[..., :128]), dict(kv=kv[:, :1]), dict(k_rope=rope[:4]), dict(out=kv[:3, :, :128]),
                dict(cu_k=cu5[:1]), dict(k_rope=out.view(-1)[:320].view(5, 64)), dict(out=q.view(-1)[:768].view(3, 2, 128))):
        with pytest.raises(nvb.NvbError):
            nvb.latent_prefill_fwd(**{**good, **bad})
    torch.cuda.synchronize()
