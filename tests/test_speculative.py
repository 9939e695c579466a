"""Host side of the speculative-decoding operators: ancestor masks, forks and
truncation of page lists, and the argument checks of the device entry points,
which run before any CUDA call."""
import ctypes

import numpy as np
import pytest

import spec_ref

P = ctypes.c_void_p
NZ = P(256)  # any non-null aligned address: the checks fail before it is used


@pytest.fixture(scope="module")
def host(nvb):
    from importlib import import_module

    return import_module("nano_vllm_rs_b200.host")


# ------------------------------------------------------------------ tree masks
@pytest.mark.parametrize("sizes", [[1], [5], [1, 3, 0, 7], [64], [65, 130], [200]])
def test_tree_mask_is_each_nodes_ancestors(host, sizes):
    rng = np.random.RandomState(sum(sizes))
    parents, cu = [], [0]
    for n in sizes:
        parents += [-1] + [int(rng.randint(-1 if i > 2 else 0, i)) for i in range(1, n)] if n else []
        cu.append(cu[-1] + n)
    mask, depth = host.tree_mask(parents, cu)
    for s, n in enumerate(sizes):
        seen = spec_ref.ancestors(parents[cu[s]:cu[s + 1]])
        assert np.array_equal(mask[cu[s]:cu[s + 1]], spec_ref.pack_bits(seen, mask.shape[1]))
        assert np.array_equal(depth[cu[s]:cu[s + 1]], seen.sum(1) - 1)


@pytest.mark.parametrize("parents, cu, words", [([0], [0, 1], 1), ([-1, 1], [0, 2], 1), ([-1, 5], [0, 2], 1),
                                                ([-1, -2], [0, 2], 1), ([-1] * 65, [0, 65], 1),
                                                ([-1, 0], [1, 2], 1), ([-1, 0], [0, 2, 1], 1), ([-1], [0, 1], 0)])
def test_tree_mask_refuses(host, parents, cu, words):
    with pytest.raises(host.HostError):
        host.tree_mask(parents, cu, words)


def test_tree_mask_refuses_more_rows_than_parents(host):
    with pytest.raises(host.HostError):
        host.tree_mask([-1], [0, 2])


@pytest.mark.parametrize("cu", [[0, 10, 5], [0, 3, 12, 2, 5], [0, 5, 100, 5], [0, 6, -1, 5]])
def test_tree_mask_refuses_falling_offsets_before_it_writes(host, cu):
    # the rows that such offsets reach in between lie behind the arrays, which end at the last offset's
    with pytest.raises(host.HostError):
        host.tree_mask([-1] * 5, cu)
    parents, offsets = np.full(128, -1, np.int32), np.array(cu, np.int32)
    mask, depth = np.full((128, 2), 77, np.uint64), np.full(128, 77, np.int32)
    ptr = lambda x: x.ctypes.data_as(P)  # noqa: E731
    assert host.library().nvbh_tree_mask(ptr(parents), ptr(offsets), len(cu) - 1, 2, ptr(mask), ptr(depth)) == -1
    assert (mask == 77).all() and (depth == 77).all()


# ------------------------------------------------------------ forked page lists
@pytest.mark.parametrize("tokens", [0, 1, 255, 256, 257, 512, 700])
def test_fork_shares_full_pages_and_copies_the_partial_one(host, tokens):
    pool = host.BlockPool(8)
    blocks = [pool.allocate() for _ in range(3)]
    child, copy = pool.fork(blocks, tokens, 256)
    full, part = divmod(tokens, 256)
    assert child[:full] == blocks[:full] and len(child) == full + (part > 0)
    assert [pool.references(x) for x in blocks] == [2] * full + [1] * (3 - full)
    if part:
        assert copy == (blocks[full], child[full], part) and child[full] not in blocks
        assert pool.references(child[full]) == 1
    else:
        assert copy is None
    for x in child:
        pool.release(x)
    assert pool.in_use() == 3


def test_fork_failures_leave_the_pool_as_it_was(host):
    pool = host.BlockPool(2)
    blocks = [pool.allocate(), pool.allocate()]
    for bad, tokens in ((blocks, 300), (blocks, 600), (blocks[:1], 257), ([0, 7], 400), ([-1], 5)):
        with pytest.raises(host.HostError):
            pool.fork(bad, tokens, 256)
        assert [pool.references(x) for x in blocks] == [1, 1] and pool.available() == 0
    assert pool.fork(blocks, 512, 256) == (blocks, None)  # whole pages need no free one
    with pytest.raises(host.HostError):
        pool.fork(blocks, 512, 0)


def test_fork_of_a_fork_and_a_cached_page(host):
    pool = host.BlockPool(4)
    a = [pool.allocate()]
    pool.publish(a[0], list(range(256)))
    b, _ = pool.fork(a, 256, 256)
    c, copy = pool.fork(b, 100, 256)
    assert b == a and pool.references(a[0]) == 2 and copy == (a[0], c[0], 100)
    pool.release(a[0])
    pool.release(b[0])
    assert pool.find(list(range(256))) == a[0]  # free, and still found by its prefix


@pytest.mark.parametrize("tokens, kept", [(0, 0), (1, 1), (256, 1), (257, 2), (768, 3)])
def test_truncate_releases_the_pages_behind(host, tokens, kept):
    pool = host.BlockPool(3)
    blocks = [pool.allocate() for _ in range(3)]
    assert pool.truncate(blocks, tokens, 256) == blocks[:kept]
    assert pool.in_use() == kept


def test_truncate_refuses_and_keeps(host):
    pool = host.BlockPool(3)
    blocks = [pool.allocate(), pool.allocate()]
    for bad, tokens in ((blocks, 513), (blocks + [2], 100), ([blocks[0], -1], 0)):
        with pytest.raises(host.HostError):
            pool.truncate(bad, tokens, 256)
        assert pool.in_use() == 2
    child, _ = pool.fork(blocks, 512, 256)
    pool.truncate(child, 256, 256)
    assert [pool.references(x) for x in blocks] == [2, 1]  # a shared page loses one user


def test_truncate_into_a_published_page_takes_it_out_of_the_cache(host):
    # the sequence writes over what is behind its 300 tokens: nobody may find the page under its 512 any more
    pool, tokens = host.BlockPool(4), list(range(600))
    blocks = [pool.allocate(), pool.allocate()]
    for i in range(2):
        pool.publish(blocks[i], tokens[:256 * (i + 1)])
    assert pool.truncate(blocks, 300, 256) == blocks
    assert pool.find(tokens[:512]) is None and pool.find(tokens[:256]) == blocks[0] and pool.cached_keys() == 1
    other = tokens[:300] + [7] * 212
    pool.publish(blocks[1], other)  # filled anew
    assert pool.find(other) == blocks[1] and pool.find(tokens[:512]) is None


@pytest.mark.parametrize("tokens", [0, 256, 512])
def test_truncate_at_a_pages_end_keeps_the_cache(host, tokens):
    pool, text = host.BlockPool(4), list(range(512))
    blocks = [pool.allocate(), pool.allocate()]
    for i in range(2):
        pool.publish(blocks[i], text[:256 * (i + 1)])
    pool.truncate(blocks, tokens, 256)
    assert [pool.find(text[:256]), pool.find(text)] == blocks  # whole, and free or in use


def test_truncate_into_a_page_that_another_sequence_holds_keeps_it_for_that_one(host):
    pool, text = host.BlockPool(4), list(range(512))
    blocks = [pool.allocate(), pool.allocate()]
    for i in range(2):
        pool.publish(blocks[i], text[:256 * (i + 1)])
    child, _ = pool.fork(blocks, 512, 256)
    assert pool.truncate(child, 300, 256) == blocks and pool.references(blocks[1]) == 2
    assert pool.find(text) == blocks[1]  # the child copies it before it writes
    assert pool.truncate(blocks, 256, 256) == blocks[:1] and pool.find(text) == blocks[1]


def test_truncate_keeps_a_page_published_for_no_more_than_is_kept(host):
    pool, text = host.BlockPool(4), list(range(300))
    blocks = [pool.allocate(), pool.allocate()]
    pool.publish(blocks[1], text)
    pool.truncate(blocks, 300, 256)
    assert pool.find(text) == blocks[1]


@pytest.mark.parametrize("page", [-1, 3, 2 ** 31 - 1, -2 ** 31])
def test_truncate_into_a_page_that_the_pool_does_not_have_keeps_it_as_it_is(host, page):
    pool = host.BlockPool(3)
    blocks = [page, pool.allocate()]
    assert pool.truncate(blocks, 100, 256) == [page] and pool.in_use() == 0


# -------------------------------------------------- argument checks of the ABI
def _tree(lib, **kw):
    a = dict(q=NZ, mask=NZ, words=1, batch=1, total_q=2, max_q=2, max_k=300, qh=4, kvh=2, bs=256, stride=2, splits=1,
             lse_accum=NZ, out_accum=NZ, blocks=2)
    a.update(kw)
    return lib.nvb_paged_tree_fwd(P(0), a["q"], NZ, NZ, NZ, NZ, NZ, NZ, a["mask"], a["words"], a["batch"],
                                  a["total_q"], a["max_q"], a["max_k"], a["qh"], a["kvh"], a["bs"], a["stride"],
                                  a["splits"], NZ, a["lse_accum"], a["out_accum"], a["blocks"])


@pytest.mark.parametrize("bad", [dict(q=P(0)), dict(mask=P(0)), dict(mask=P(257)), dict(words=0), dict(words=17),
                                 dict(max_q=65), dict(batch=0), dict(batch=65536), dict(total_q=0), dict(max_q=0),
                                 dict(max_k=0), dict(max_k=513), dict(qh=5), dict(qh=258, kvh=2), dict(kvh=0),
                                 dict(bs=128), dict(stride=0), dict(stride=1 << 24), dict(splits=0),
                                 dict(splits=129), dict(splits=16, lse_accum=P(0)), dict(splits=11, out_accum=P(0)),
                                 dict(blocks=0), dict(blocks=1 << 24), dict(q=P(264)),
                                 dict(total_q=1 << 30)])
def test_tree_refuses_on_the_host(nvb, bad):
    lib = nvb.library()
    assert _tree(lib, **bad) == -1
    assert lib.nvb_last_error().decode()


@pytest.mark.parametrize("at, off", [(i, o) for i in (5, 6, 7) for o in (1, 2)] + [(8, 4)] +
                         [(i, o) for i in (19, 20, 21) for o in (1, 2)] + [(21, 4)])
def test_tree_refuses_addresses_that_its_types_cannot_have(nvb, at, off):
    lib = nvb.library()
    args = [P(0), *[NZ] * 8, 1, 1, 2, 2, 300, 4, 2, 256, 2, 11, NZ, NZ, NZ, 2]
    args[at] = P(256 + off)
    assert lib.nvb_paged_tree_fwd(*args) == -1
    assert "aligned" in lib.nvb_last_error().decode()


def test_tree_num_splits(nvb):
    lib = nvb.library()
    assert [lib.nvb_tree_parts(s) for s in (0, 1, 2, 7, 8, 9, 11, 16, 128, 129)] == [0, 1, 1, 1, 1, 3, 11, 2, 16, 0]
    for bad in ((0, 4, 16, 8, 100, 148), (1, 0, 16, 8, 100, 148), (1, 4, 16, 5, 100, 148), (1, 4, 16, 8, 0, 148),
                (1, 4, 16, 8, 100, 0)):
        assert lib.nvb_tree_num_splits(*bad) == 0
    for batch in (1, 7, 64):
        for nodes in (1, 8, 64, 200):
            for max_k in (1, 300, 5000, 1 << 20):
                assert 1 <= nvb.tree_num_splits(batch, nodes, 32, 8, max_k, 148) <= 128


@pytest.mark.parametrize("splits", [1, 2, 8, 9, 11, 24, 64, 97, 128])
def test_tree_scratch_has_a_row_for_each_part(nvb, splits):
    parts = nvb.library().nvb_tree_parts(splits)
    lse, out = nvb.tree_scratch(splits, 5, 4, "cpu")
    if parts == 1:
        assert lse is None and out is None
    else:
        assert lse.shape == (parts, 5, 4) and out.shape == (parts, 5, 4, 128)


def test_tree_num_splits_joins_on_chip_and_cuts_long_ranges(nvb):
    for batch in (1, 2, 5, 16, 37, 64, 300):
        for max_k in (64, 400, 2048, 8192, 32768, 131072):
            splits = nvb.tree_num_splits(batch, 8, 32, 8, max_k, 148)
            assert splits & (splits - 1) == 0 and (splits == 1 or max_k >= 128 * splits)
            # past the CTAs that fit the GPU only for long ranges, and then only what one cluster joins
            if splits > 1 and batch * 8 * splits > 296:
                assert splits <= 8 and max_k >= 2560 * splits and batch * 8 * splits <= 8 * 148
    assert nvb.tree_num_splits(64, 8, 32, 8, 4200, 148) == 1 and nvb.tree_num_splits(64, 8, 32, 8, 16384, 148) == 2


def _layers(*values):
    return (P * len(values))(*values)


def _copy(lib, **kw):
    a = dict(k=_layers(4096, 8192), v=_layers(12288, 16384), layers=2, src=NZ, dst=NZ, rows=P(0), pairs=1, kvh=2,
             dim=128, bs=256, blocks=4)
    a.update(kw)
    return lib.nvb_cache_copy_pages(P(0), a["k"], a["v"], a["layers"], a["src"], a["dst"], a["rows"], a["pairs"],
                                    a["kvh"], a["dim"], a["bs"], a["blocks"])


BAD_CACHES = [dict(k=None), dict(layers=0), dict(layers=1025), dict(kvh=0), dict(dim=0), dict(bs=0), dict(blocks=0),
              dict(blocks=1 << 24), dict(kvh=1 << 20), dict(k=_layers(4096, 0)), dict(k=_layers(4096, 8193)),
              dict(v=_layers(4096, 16384))]


@pytest.mark.parametrize("bad", BAD_CACHES + [dict(src=P(0)), dict(dst=P(0)), dict(pairs=-1), dict(pairs=5)])
def test_copy_pages_refuses_on_the_host(nvb, bad):
    lib = nvb.library()
    assert _copy(lib, **bad) == -1
    assert lib.nvb_last_error().decode()


def test_copy_of_no_pages_is_nothing(nvb):
    assert _copy(nvb.library(), pairs=0, src=P(0), dst=P(0)) == 0


@pytest.mark.parametrize("bad", BAD_CACHES + [dict(path=P(0)), dict(batch=0), dict(batch=65536), dict(stride=0),
                                              dict(table=0), dict(new=P(512))])
def test_compact_paths_refuses_on_the_host(nvb, bad):
    lib = nvb.library()
    a = dict(k=_layers(4096, 8192), v=_layers(12288, 16384), layers=2, path=NZ, new=NZ, batch=1, stride=4, kvh=2,
             dim=128, bs=256, table=2, blocks=4)
    a.update(bad)
    rc = lib.nvb_cache_compact_paths(P(0), a["k"], a["v"], a["layers"], NZ, P(512), NZ, a["path"], NZ, a["new"],
                                     a["batch"], a["stride"], a["kvh"], a["dim"], a["bs"], a["table"], a["blocks"])
    assert rc == -1
    assert lib.nvb_last_error().decode()


@pytest.mark.parametrize("off", [1, 2])
@pytest.mark.parametrize("at", range(6))
def test_cache_copies_refuse_addresses_that_their_types_cannot_have(nvb, at, off):
    lib = nvb.library()
    caches = [_layers(4096, 8192), _layers(12288, 16384), 2]
    ints = [P(1024 * (i + 1) + (off if i == at else 0)) for i in range(6)]
    assert lib.nvb_cache_compact_paths(P(0), *caches, *ints, 1, 4, 2, 128, 256, 2, 4) == -1
    assert "aligned" in lib.nvb_last_error().decode()
    if at < 3:
        assert lib.nvb_cache_copy_pages(P(0), *caches, *ints[:3], 1, 2, 128, 256, 4) == -1
        assert "aligned" in lib.nvb_last_error().decode()


@pytest.mark.parametrize("bad", [dict(logits=P(0)), dict(rows=0), dict(batch=0), dict(batch=65536), dict(max_q=0),
                                 dict(max_q=1025), dict(vocab=0), dict(ws=P(0)), dict(ws=P(264)), dict(size=8)])
def test_verify_refuses_on_the_host(nvb, bad):
    lib = nvb.model.library()
    a = dict(logits=NZ, rows=2, batch=1, max_q=2, vocab=10, ws=NZ, size=1 << 20)
    a.update(bad)
    rc = lib.nvbe_layer_verify(P(0), a["logits"], P(0), NZ, NZ, NZ, NZ, NZ, NZ, NZ, NZ, NZ, NZ, a["rows"], a["batch"],
                               a["max_q"], a["vocab"], a["ws"], a["size"])
    assert rc == -1
    assert lib.nvbe_model_last_error().decode()


@pytest.mark.parametrize("vocab", [(1 << 30) + 1, (1 << 31) - 1])
def test_verify_refuses_vocabularies_past_its_index_arithmetic(nvb, vocab):
    lib = nvb.model.library()
    assert lib.nvbe_layer_verify(P(0), *[NZ] * 12, 2, 1, 2, vocab, NZ, 1 << 20) == -1
    assert "vocab" in lib.nvbe_model_last_error().decode()


VERIFY_POINTERS = ["logits", "draft", "tokens", "parents", "uniforms", "seeds", "temperatures", "cu_q", "out_tokens",
                   "path", "counts", "accept"]


@pytest.mark.parametrize("name, off", [(n, 1) for n in VERIFY_POINTERS] + [(n, 2) for n in VERIFY_POINTERS[2:]] +
                         [("seeds", 4)])
def test_verify_refuses_addresses_that_its_types_cannot_have(nvb, name, off):
    # (the kernels would read them, which no library catches)
    lib = nvb.model.library()
    pointers = [P(256 + off) if n == name else NZ for n in VERIFY_POINTERS]
    assert lib.nvbe_layer_verify(P(0), *pointers, 2, 1, 2, 10, NZ, 1 << 20) == -1
    assert "aligned" in lib.nvbe_model_last_error().decode()


def test_verify_workspace_grows_with_the_rows(nvb):
    size = nvb.model.verify_workspace_bytes
    assert size(0, 1) == 0 and size(1, 0) == 0
    assert 0 < size(1, 1) < size(100, 1) < size(100, 7)


def test_engine_header_functions_are_exported(nvb):
    lib = nvb.model.library()
    assert lib.nvbe_layer_verify and lib.nvbe_verify_workspace_bytes


# ------------------------------------------------- the drawn token's tolerance
def test_tokens_that_may_be_drawn_are_those_that_rounding_reaches():
    rng, vocab = np.random.RandomState(1), 50
    logits, draft = rng.randn(3, vocab) * 2, rng.randn(3, vocab) * 2
    tokens, parents, seeds = np.array([0, 4, 9]), np.array([-1, 0, 0]), np.array([5, 6, 7])
    args = (tokens, parents, seeds, [1.0], [0, 3], [[0]], [1])
    for d, eps in ((draft, 0.2), (None, 0.9)):
        one, = spec_ref.drawn_from(logits, d, *args)
        more, = spec_ref.drawn_from(logits, d, *args, eps=eps)
        assert len(one) == 1 and one < more and len(more) < vocab
    assert spec_ref.drawn_from(logits, draft, tokens, parents, seeds, [0.0], [0, 3], [[0]], [1]) == [None]
    assert spec_ref.drawn_from(logits, draft, tokens, parents, seeds, [1.0], [0, 3], [[0, 2]], [2]) == [None]
    # drafts equal to the target but for one token: what is left is that token and the rounding of the likely ones; a
    # token without probability is never among them
    near = logits.copy()
    near[0, 7] += 1e-9
    logits[0, 20:] = near[0, 20:] = -np.inf
    few, = spec_ref.drawn_from(near, logits, *args)
    assert few and max(few) < 20


# ------------------------------------------------- memory that a graph holds on to
def test_a_graph_keeps_the_workspaces_of_its_calls(nvb, monkeypatch):
    class Library:
        def __getattr__(self, name):
            return lambda *a: 0

    monkeypatch.setattr(nvb, "library", lambda: Library())
    monkeypatch.setattr(nvb, "_stream", lambda stream=None: P(0))
    given, first, second, failed = object(), object(), object(), object()
    nvb._hold(failed)  # no capture is under way: the call's own memory goes back

    def broken():
        nvb._hold(failed)
        raise ValueError

    def outer():
        nvb._hold(first)
        with pytest.raises(ValueError):
            nvb.capture(broken)
        nvb._hold(second)

    graph = nvb.capture(outer, keep=[given])
    assert graph._keep == [given, first, second] and nvb._captures == []
