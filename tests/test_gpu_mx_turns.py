"""The microscaled products where a workgroup computes several tiles in turn:
every tile shape, dense, for experts and with the SwiGLU fold, with scales in
16-byte pieces and without, K of one, three and fifteen 128s (a tile's last
stage is a half one there, and the next tile's first follows it) and of whole
stages.  Each case says which shape it is for and is checked to take it, with
more than two tiles a workgroup, against the plain 64-bit form; test_gpu_mx.py
derives the bounds."""
import numpy as np
import pytest

import test_gpu_mx_tiles as edges
from conftest import load_oracle
from helpers import device
from mx_tiles import count, tiles_of
from test_gpu_mx import Encoded, check_product, close, encoded, run_experts, want_experts

load_oracle()
import mx_oracle as mx  # noqa: E402

# (tile of C x tile of B, m, n): 16 x 64 tiles take no dense product of so many tiles
DENSE = [((16, 128), 3, 140503), ((32, 128), 18, 140501), ((64, 64), 69700, 45), ((128, 128), 90, 150001),
         ((256, 256), 190, 152003)]
DENSE_K = [1, 129, 384, 450, 512]
# (tile, routes, experts, n, swiglu)
EXPERTS = [((16, 64), 19300, 1024, 46, False), ((16, 64), 19300, 1024, 44, True),
           ((16, 128), 2820, 130, 404, False), ((16, 128), 2820, 130, 410, True),
           ((32, 128), 5660, 130, 404, False), ((32, 128), 5660, 130, 410, True),
           ((64, 64), 61000, 130, 42, False), ((64, 64), 61000, 130, 40, True),
           ((128, 128), 122500, 130, 51, False), ((128, 128), 122500, 130, 50, True),
           ((256, 256), 106600, 130, 132, False), ((256, 256), 106600, 130, 132, True)]
EXPERTS_K = [100, 384, 1900, 450, 1024]


def fits(values, k, tile):
    """The plain form's time bounds the sizes; narrow scales do not run on 256 x 256 tiles."""
    return values * k < 1.1e8 and (tile != (256, 256) or -(-k // 128) % 4 == 0)


def dense_cases():
    return [(tile, m, n, k) for tile, m, n in DENSE for k in DENSE_K if fits(m + n, k, tile)]


def expert_cases():
    return [(tile, routes, experts, n, swiglu, k) for tile, routes, experts, n, swiglu in EXPERTS
            for k in EXPERTS_K if fits(routes + experts * n, k, tile)]


def ids_of(routes, experts):
    """Even routing with some dropped routes."""
    rng = np.random.default_rng(routes + experts)
    ids = rng.permutation(routes).astype(np.int32).reshape(routes, 1) % experts
    ids[rng.random(ids.shape) < 0.02] = -1
    return ids


def test_every_form_takes_turns():
    """Each case takes its shape with more than two tiles a workgroup, and the cases hold every
    shape and form that can: narrow scales do not run on 256 x 256 tiles."""
    seen = set()
    for tile, m, n, k in dense_cases():
        t = tiles_of(m, n, k)
        assert (t.rows, t.columns) == tile and t.at_most > 2 * t.workgroups, (tile, m, n, k, t)
        seen.add((tile, "dense", t.wide, -(-k // 128) % 2))
    for tile, routes, experts, n, swiglu, k in expert_cases():
        t = tiles_of(routes, n, k, experts, swiglu)
        assert (t.rows, t.columns) == tile, (tile, routes, n, k, t)
        offsets, _, _ = mx.sort_routes(ids_of(routes, experts), experts)
        assert count(t, n, swiglu, offsets) > 2 * t.workgroups and not t.streamed, (tile, routes, experts, n, k, t)
        seen.add((tile, "swiglu" if swiglu else "plain", t.wide, -(-k // 128) % 2))
    for tile in ((16, 64), (16, 128), (32, 128), (64, 64), (128, 128), (256, 256)):
        for form in ("dense", "plain", "swiglu"):
            if (tile, form) != ((16, 64), "dense"):
                assert (tile, form, 1, 0) in seen, (tile, form)
                if tile != (256, 256):
                    assert (tile, form, 0, 1) in seen, (tile, form)


def test_every_shape_has_cases_with_edges():
    """test_gpu_mx_tiles.py's cases, by their sizes: all six shapes of dense products but the
    smallest, all six of experts' products, with both kinds of scales where there are both."""
    def cases(test):
        mark = next(m for m in test.pytestmark if m.name == "parametrize")
        return mark.args[1]

    dense = {t[:3] for t in (tiles_of(*c) for c in cases(edges.test_product))}
    experts = {(swiglu, *tiles_of(routes, n, k, e, swiglu)[:3])
               for swiglu, routes, e, n, k in cases(edges.test_experts)}
    for tile in ((16, 64), (16, 128), (32, 128), (64, 64), (128, 128), (256, 256)):
        for wide in (0, 1) if tile != (256, 256) else (1,):
            assert tile == (16, 64) or (*tile, wide) in dense, (tile, wide)
            for swiglu in (False, True):
                assert (tile, wide) == ((16, 64), 0) or (swiglu, *tile, wide) in experts, (swiglu, tile, wide)
    streamed = {tiles_of(routes, n, k, e, swiglu)[:4]
                for swiglu, routes, e, n, k, _ in cases(edges.test_weights_past_the_caches)}
    assert streamed == {(16, 64, 1, 1), (16, 128, 1, 1), (32, 128, 1, 1)}


def test_no_dense_product_takes_turns_on_the_smallest_tiles():
    for m in (1, 2, 15, 16, 17, 31, 32, 33, 48, 64, 100, 1000, 20000):
        for n in sorted({int(64 * 1.06 ** i) for i in range(170)} | {49152 + 64 * i for i in range(300)}):
            t = tiles_of(m, n, 256)
            assert (t.rows, t.columns) != (16, 64) or t.at_most <= t.workgroups, (m, n, t)


@pytest.mark.gpu
@pytest.mark.parametrize("tile,m,n,k", dense_cases())
def test_product(q38m, tile, m, n, k):
    print(f"product {m} x {n} x {k} on {tile}", flush=True)
    rng = np.random.default_rng(m + n + k)
    check_product(q38m, Encoded(q38m, *encoded(rng, m, k), k), Encoded(q38m, *encoded(rng, n, k), k), k,
                  "f32" if k % 4 else "bf16", spare=3)


@pytest.mark.gpu
@pytest.mark.parametrize("tile,routes,experts,n,swiglu,k", expert_cases())
def test_experts(q38m, tile, routes, experts, n, swiglu, k):
    print(f"experts {routes} of {experts}, {n} x {k} swiglu {swiglu} on {tile}", flush=True)
    rng = np.random.default_rng(routes + n + k)
    offsets, packed, _ = mx.sort_routes(ids_of(routes, experts), experts)
    kept = int(offsets[-1])
    w = Encoded(q38m, *encoded(rng, experts * n, k, 122, 126), k, experts)
    gather = k % 4 == 0
    # two routes a token where rows are gathered
    rows = Encoded(q38m, *encoded(rng, (routes + 1) // 2 if gather else routes, k, 122, 126), k)
    dtype = "f32" if n % 4 else "bf16"
    words, got = run_experts(q38m, w, rows, device(offsets), device(packed) if gather else None, 2, routes, swiglu, dtype)
    want, bound = want_experts(w.values, rows.values, offsets, packed, 2 if gather else 0, experts, k, swiglu)
    assert (words[kept:] == 0x4a4a).all(), "a dropped route's row was written"
    close(got[:kept], want[:kept], bound[:kept], dtype, (tile, routes, experts, n, k))
