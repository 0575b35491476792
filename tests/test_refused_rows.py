"""Refusals of tmopt_refused_rows (CPU: they come before any launch)."""


def test_refused_rows_refusals(tm):
    lib, e, P = tm._lib.load(), tm._lib, 16

    def call(reject=P, out=P, st=1024, sh=128, rows=5, heads=8, dim=128,
             lse=P, lsh=5, lheads=8):
        return lib.tmopt_refused_rows(reject, out, st, sh, rows, heads, dim,
                                      lse, lsh, lheads, None)
    assert call(rows=0) == call(rows=0, reject=None, out=None) == e.TMOPT_OK
    for kw in (dict(reject=None), dict(out=None), dict(out=4), dict(st=2),
               dict(sh=2), dict(dim=6), dict(dim=0), dict(heads=0),
               dict(heads=1 << 30), dict(lheads=0), dict(rows=-1)):
        assert call(**kw) == e.TMOPT_EINVAL, kw
    assert call(rows=(1 << 31) + 1) == e.TMOPT_EUNSUPPORTED
