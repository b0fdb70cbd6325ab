"""Which kernels the shapes of test_gpu_hidden_tiles.py launch, against a stand-in of the HIP
runtime: every kind of tile is reached in each pass, whole and split, and no kernel of a
hidden block is left out."""
import hostrun
import pytest
import test_gpu_hidden_tiles as tiles
import test_host_hidden as host

SHAPES = {"64x32": "64,32,1,1,4,256,3,false", "64x64": "64,32,1,2,2,128,4,false", "128x128": "64,64,2,2,1,128,3,false",
          "256x256": "128,64,2,4,1,128,2,true"}
F8_SHAPES = {"64x32": "16,32,4,1,1,128,6,false", "64x64": "32,32,2,2,1,128,4,false", "128x128": SHAPES["128x128"],
             "256x256": SHAPES["256x256"]}


def _mangled(numbers):
    """template arguments as a mangled name has them"""
    return "".join(f"Lb{int(v == 'true')}E" if v in ("true", "false") else f"Li{v}E" for v in numbers.split(","))


def _tile(names, kernel, shape):
    """whether one of the names is this tile kernel's, of this shape"""
    return any(kernel in n and any(f in n.replace(" ", "") for f in (f"TileShape<{shape}>", f"TileShapeI{_mangled(shape)}E")) for n in names)


def _launched(calls):
    got = hostrun.call(host._calls, calls)
    assert all(rc == 0 for rc, _, _ in got), got
    return [[k for k, _ in names] for _, _, names in got]


def _gated(shape, dtype, backward):
    rows, k, n = shape
    if backward:
        return host._backward(rows=rows, k=k, n=n, xs=k, wgs=k, us=k, gs=n, dxs=k, dtype=dtype)
    return host._forward(rows=rows, k=k, n=n, xs=k, gs=k, us=k, hs=n, dtype=dtype)


# of a product: the number in its kernel's name
@pytest.mark.parametrize("dtype", [2, 3])
@pytest.mark.parametrize("op,number,shapes", [("forward", 0, tiles.FORWARD), ("dx", 1, tiles.INPUT), ("dw", 2, tiles.WEIGHT)])
def test_gated(op, number, shapes, dtype):
    assert {t for t, _ in shapes} == set(SHAPES) and len(shapes) == 2 * len(SHAPES)
    for ((tile, split), shape), names in zip(shapes.items(), _launched([_gated(s, dtype, op != "forward") for s in shapes.values()])):
        mine = [n for n in names if f">,{number}," in n.replace(" ", "") or f"EELi{number}E" in n]
        assert _tile(mine, "gated_tile_kernel", SHAPES[tile]), (op, tile, split, shape, names)
        joins = [n for n in names if "gated_join_kernel" in n and (f"<{number}," in n.replace(" ", "") or f"ILi{number}E" in n)]
        assert bool(joins) == split, (op, tile, split, names)


@pytest.mark.parametrize("out,shapes", [(2, tiles.F8_16), (3, tiles.F8_16), (1, tiles.F8_32)])
def test_f8(out, shapes):
    calls = [host._f8(rows=r, k=k, xs=k, ws=k, q=q, ys=q, od=out) for r, k, q in shapes.values()]
    for ((tile, split), shape), names in zip(shapes.items(), _launched(calls)):
        assert _tile(names, "f8_tile_kernel", F8_SHAPES[tile]), (tile, split, shape, names)
        assert any("f8_join_kernel" in n for n in names) == split and any("f8_quantise" in n for n in names), (tile, split, names)


@pytest.mark.parametrize("out,shapes", [(2, tiles.F8_LONG_16), (1, tiles.F8_LONG_32)])
def test_f8_long(out, shapes):
    assert set(shapes) == (set(F8_SHAPES) if out == 2 else set(F8_SHAPES) - {"256x256"})
    calls = [host._f8(rows=r, k=k, xs=k, ws=k, q=q, ys=q, od=out) for r, k, q in shapes.values()]
    for (tile, shape), names in zip(shapes.items(), _launched(calls)):
        assert _tile(names, "f8_tile_kernel", F8_SHAPES[tile]) and not any("join" in n for n in names), (tile, shape, names)


def test_rows_quantised_by_the_workgroups():
    calls = [host._f8(rows=r, k=k, xs=k, ws=k, q=q, ys=q, od=out) for r, k, q in ((1, 16384, 70000), (3, 4096, 40000), (8, 2048, 33000), (31, 512, 40000))
             for out in (1, 2)]
    for names in _launched(calls):
        assert len(names) == 1 and "f8_tile_kernel" in names[0], names
