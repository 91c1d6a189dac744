"""Which form of the int8 product takes a shape (CPU): nothing is compiled that no shape reaches."""
import pytest

import mul_forms_util as U

pytestmark = pytest.mark.skipif(not U.there, reason="g++ not available")

ROWS = (1, 2, 5, 9, 16, 17, 24, 32, 33, 48, 49, 64, 70, 99, 100, 130, 200, 256, 300, 400, 700, 1000, 1500, 2000, 4000, 8000)
CHANNELS = (1, 16, 40, 100, 256, 576, 1024, 2112, 4096, 7168, 12000, 16384, 24576)
DEPTHS = (16, 128, 144, 512, 1536, 4096, 7168, 16384, 65536, 131056)


def test_every_form_is_chosen():
    """Each of them whole, and cut where it may be; a workspace where k is cut and then only."""
    forms, seen = U.forms(), set()
    assert sorted(forms) == sorted(U.NAMES)
    for rows in ROWS:
        for n in CHANNELS:
            for k in DEPTHS:
                name, parts, work = U.form_of(rows, n, k)
                bn, bm, cuts = forms[name]
                tiles = -(-n // bn) * -(-rows // bm)
                assert parts == 1 or cuts
                assert work == (tiles * parts * bn * bm * 4 if parts > 1 else 0) <= 1 << 24
                assert U.form_of(rows, n, k, False)[1:] == (1, 0)
                seen |= {(name, parts > 1), (U.form_of(rows, n, k, False)[0], False)}
    assert seen == {(f, cut) for f, (_, _, cuts) in forms.items() for cut in ({False, cuts})}


def test_shapes_of_every_form():
    """The shapes that the GPU tests run are given to the forms that they are listed under: uncut without a workspace, cut with one."""
    assert set(U.SHAPES) == {(f, cut) for f, (_, _, cuts) in U.forms().items() for cut in ({False, cuts})}
    for (form, cut), shapes in U.SHAPES.items():
        for s in shapes:
            name, parts, _ = U.form_of(*s, cut)
            assert (name, parts > 1) == (form, cut), (s, name, parts)
