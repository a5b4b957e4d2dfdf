"""The batch operators' refusals, without a device: pagedAppend, pagedAttention and tokenLogprobs check
every argument before any device work (a null context stands in for the device; valid calls then
report DeviceFailure)."""
import ctypes as C

import numpy as np
import pytest

from conftest import ROOT  # noqa: F401  (puts the package on the path)

FAKE = 1 << 20  # never dereferenced: the checks come first


def rc_of(hip, fn, args):
    return getattr(hip.LIB, fn)(None, C.byref(args))


def views(hip, **sizes):
    """Views a MiB apart (`sizes` in bytes)."""
    return {n: hip.Buf(FAKE * (i + 1), 0, b) for i, (n, b) in enumerate(sizes.items())}


SHAPE = dict(q_dtype=0, n_tokens=5, n_seqs=2, n_q_heads=4, n_kv_heads=2, head_dim=64, page_size=16, n_pages=3, max_pages=2,
             max_seq_len=32)
POOL, ROW = 2 * 3 * 16 * 64 * 2, 64 * 4


def append(hip, **kw):
    v = views(hip, q=5 * 4 * ROW, k=5 * 2 * ROW, v=5 * 2 * ROW, q_norm=ROW, k_norm=ROW, q_out=5 * 4 * ROW, k_pool=POOL, v_pool=POOL,
              page_table=16, starts=12, seq_lens=8)
    return hip.PagedAppendArgs(**{**v, **SHAPE, "eps": 1e-6, "theta": 1e6, "freq_scale": 1.0, **kw})


def attention(hip, **kw):
    v = views(hip, q=5 * 4 * ROW, k_pool=POOL, v_pool=POOL, page_table=16, starts=12, seq_lens=8, out=5 * 4 * ROW)
    return hip.PagedAttentionArgs(**{**v, **SHAPE, "scale": 0.125, **kw})


def logprobs(hip, **kw):
    v = views(hip, logits=(2 * 104 + 100) * 4, targets=12, logprobs=12, entropy=12, top_ids=60, top_logprobs=60)
    return hip.TokenLogprobsArgs(**{**v, **dict(n_rows=3, vocab=100, row_stride=104, top_n=5), **kw})


BATCH = [("ds5_hip_paged_append", append), ("ds5_hip_paged_attention", attention)]


@pytest.mark.parametrize("fn,make", BATCH)
def test_batch_refusals(hip, fn, make):
    assert rc_of(hip, fn, make(hip)) == 3  # valid: only the device is missing
    assert getattr(hip.LIB, fn)(None, None) == 1
    for dt in (8, 2, 30):
        assert rc_of(hip, fn, make(hip, q_dtype=dt)) == 2
    big = 2 ** 32 - 1
    for bad in (dict(n_kv_heads=0), dict(n_q_heads=0), dict(head_dim=0), dict(head_dim=96), dict(head_dim=256), dict(page_size=0),
                dict(page_size=24), dict(n_pages=0), dict(max_pages=0), dict(max_seq_len=33), dict(n_pages=4), dict(n_tokens=6),
                dict(n_seqs=3), dict(max_pages=3), dict(n_tokens=big), dict(n_seqs=big), dict(n_pages=big), dict(max_pages=big),
                dict(n_kv_heads=big, n_q_heads=big), dict(page_size=big - 15), dict(n_pages=big, page_size=big - 15)):
        assert rc_of(hip, fn, make(hip, **bad)) == 1, bad
    for name in ("q", "k_pool", "v_pool", "page_table", "starts", "seq_lens"):
        b = getattr(make(hip), name)
        assert rc_of(hip, fn, make(hip, **{name: hip.Buf(b.handle, 0, b.len - 1)})) == 1, name
        assert rc_of(hip, fn, make(hip, **{name: hip.Buf(b.handle, 2, b.len)})) == 1, name
        assert rc_of(hip, fn, make(hip, **{name: hip.Buf(None, 0, b.len)})) == 1, name
    for name in ("q", "k_pool", "v_pool"):
        b = getattr(make(hip), name)
        assert rc_of(hip, fn, make(hip, **{name: hip.Buf(b.handle, 8, b.len)})) == 1, name
    for name in ("page_table", "starts", "seq_lens"):
        b = getattr(make(hip), name)
        assert rc_of(hip, fn, make(hip, **{name: hip.Buf(b.handle, 4, b.len)})) == 3, name
    for nothing in (dict(n_tokens=0), dict(n_seqs=0)):
        assert rc_of(hip, fn, make(hip, **nothing)) == 0


def test_append_refusals(hip):
    fn = "ds5_hip_paged_append"
    none = hip.Buf()
    assert rc_of(hip, fn, append(hip, q=none, q_out=none, n_q_heads=0)) == 3  # k and v alone
    assert rc_of(hip, fn, append(hip, q_norm=none, k_norm=none)) == 3
    assert rc_of(hip, fn, append(hip, n_q_heads=3)) == 3  # q heads need no group here
    a = append(hip)
    for name in ("k", "v", "q_out", "q_norm", "k_norm"):
        b = getattr(a, name)
        assert rc_of(hip, fn, append(hip, **{name: hip.Buf(b.handle, 0, b.len - 4)})) == 1, name
        assert rc_of(hip, fn, append(hip, **{name: hip.Buf(b.handle, 4, b.len)})) == 1, name
    # f16 rows take half the room; in place only where the types agree
    half = hip.Buf(a.q_out.handle, 0, a.q_out.len // 2)
    assert rc_of(hip, fn, append(hip, q_out=half, q_dtype=1)) == 3
    assert rc_of(hip, fn, append(hip, q_out=half)) == 1
    assert rc_of(hip, fn, append(hip, q_out=a.q)) == 3
    assert rc_of(hip, fn, append(hip, q_out=a.q, q_dtype=1)) == 1
    assert rc_of(hip, fn, append(hip, q_out=hip.Buf(a.q.handle, 16, a.q.len))) == 1
    for out, other in (("q_out", "k"), ("k_pool", "v"), ("v_pool", "k_pool"), ("k_pool", "q"), ("v_pool", "q_out"), ("q_out", "seq_lens"),
                       ("k_pool", "page_table"), ("v_pool", "k_norm")):
        assert rc_of(hip, fn, append(hip, **{out: hip.Buf(getattr(a, other).handle, 0, getattr(a, out).len)})) == 1, (out, other)


def test_attention_refusals(hip):
    fn = "ds5_hip_paged_attention"
    a = attention(hip)
    assert rc_of(hip, fn, attention(hip, n_q_heads=3)) == 1
    assert rc_of(hip, fn, attention(hip, out=hip.Buf(a.out.handle, 0, a.out.len - 1))) == 1
    assert rc_of(hip, fn, attention(hip, out=hip.Buf(a.out.handle, 8, a.out.len))) == 1
    for other in ("q", "k_pool", "v_pool", "page_table", "starts", "seq_lens"):
        assert rc_of(hip, fn, attention(hip, out=hip.Buf(getattr(a, other).handle, 0, a.out.len))) == 1, other
    half = hip.Buf(a.q.handle, 0, a.q.len // 2)
    assert rc_of(hip, fn, attention(hip, q=half, q_dtype=1)) == 3
    assert rc_of(hip, fn, attention(hip, q=half)) == 1
    many = dict(n_seqs=1024, starts=hip.Buf(FAKE * 50, 0, 4 * 1026), seq_lens=hip.Buf(FAKE * 51, 0, 4 * 1025),
                page_table=hip.Buf(FAKE * 52, 0, 8 * 1025))
    assert rc_of(hip, fn, attention(hip, **many)) == 3
    assert rc_of(hip, fn, attention(hip, **{**many, "n_seqs": 1025})) == 1
    # (append takes more sequences)
    assert rc_of(hip, "ds5_hip_paged_append", append(hip, **{**many, "n_seqs": 1025})) == 3


def test_logprobs_refusals(hip):
    fn = "ds5_hip_token_logprobs"
    assert rc_of(hip, fn, logprobs(hip)) == 3
    assert getattr(hip.LIB, fn)(None, None) == 1
    none, big = hip.Buf(), 2 ** 32 - 1
    for bad in (dict(vocab=0), dict(vocab=hip.LOGPROBS_MAX_VOCAB + 1, row_stride=big), dict(row_stride=99), dict(row_stride=105),
                dict(n_rows=4), dict(n_rows=big), dict(top_n=33), dict(top_n=6), dict(vocab=4, top_n=5), dict(targets=none),
                dict(logits=none), dict(top_ids=none), dict(top_logprobs=none), dict(n_rows=big, row_stride=big)):
        assert rc_of(hip, fn, logprobs(hip, **bad)) == 1, bad
    for ok in (dict(logprobs=none), dict(logprobs=none, targets=none), dict(entropy=none), dict(top_n=0, top_ids=none, top_logprobs=none),
               dict(vocab=99), dict(row_stride=100)):
        assert rc_of(hip, fn, logprobs(hip, **ok)) == 3, ok
    assert rc_of(hip, fn, logprobs(hip, n_rows=0)) == 0
    assert rc_of(hip, fn, logprobs(hip, logprobs=none, entropy=none, top_n=0)) == 0  # nothing asked for
    a = logprobs(hip)
    for name in ("logits", "targets", "logprobs", "entropy", "top_ids", "top_logprobs"):
        b = getattr(a, name)
        assert rc_of(hip, fn, logprobs(hip, **{name: hip.Buf(b.handle, 0, b.len - 4)})) == 1, name
        assert rc_of(hip, fn, logprobs(hip, **{name: hip.Buf(b.handle, 2, b.len)})) == 1, name
        assert rc_of(hip, fn, logprobs(hip, **{name: hip.Buf(b.handle, 4, b.len)})) == 3, name
    for out, other in (("logprobs", "logits"), ("top_ids", "targets"), ("entropy", "logprobs"), ("top_logprobs", "top_ids")):
        assert rc_of(hip, fn, logprobs(hip, **{out: hip.Buf(getattr(a, other).handle, 0, getattr(a, out).len)})) == 1, (out, other)


def test_more_rows_than_a_launch_takes(hip):
    """2^24 - 1 workgroups of 256 threads at most, whatever the views hold."""
    at = {n: hip.Buf((i + 1) << 44, 0, 1 << 43) for i, n in enumerate(("q", "k", "v", "q_norm", "k_norm", "q_out", "k_pool", "v_pool",
                                                                       "page_table", "starts", "seq_lens"))}
    for n, rc in ((2 ** 24 - 1, 3), (2 ** 24, 1)):
        assert rc_of(hip, "ds5_hip_paged_append", append(hip, **at, n_tokens=n)) == rc
    at = {n: hip.Buf((i + 1) << 44, 0, 1 << 43) for i, n in enumerate(("logits", "targets", "logprobs", "entropy", "top_ids", "top_logprobs"))}
    for n, V, rc in ((2 ** 24 - 1, 8192, 3), (2 ** 24, 100, 1), (2 ** 23 - 1, 8193, 3), (2 ** 23, 8193, 1), (2 ** 32 - 1, 1, 1)):
        assert rc_of(hip, "ds5_hip_token_logprobs", logprobs(hip, **at, n_rows=n, vocab=V, row_stride=V, top_n=0)) == rc, (n, V)


def test_structs_match_c(hip, tmp_path):
    import subprocess
    import test_abi
    names = {"ds5_paged_append_args": "PagedAppendArgs", "ds5_paged_attention_args": "PagedAttentionArgs",
             "ds5_token_logprobs_args": "TokenLogprobsArgs"}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{test_abi.HEADER}"', 'int main(void) {']
    for c, py in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in getattr(hip, py)._fields_]
    lines.append('printf("%u\\n%u\\n%u\\n", DS5_PAGED_MAX_SEQS, DS5_LOGPROBS_MAX_VOCAB, DS5_LOGPROBS_MAX_TOP); return 0; }')
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in names.values():
        t = getattr(hip, py)
        want += [C.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]
    assert got == want + [hip.PAGED_MAX_SEQS, hip.LOGPROBS_MAX_VOCAB, hip.LOGPROBS_MAX_TOP]


def test_score_refusals(hip):
    from qw3_amd import engine as E
    eng = E.Engine.__new__(E.Engine)
    eng.cfg = dict(vocab_size=10)
    for tokens, targets, top in (([1, 2], [3], 0), ([1], [10], 0), ([1], [-1], 0), ([1], [1], 11), ([1], [1], -1)):
        with pytest.raises(ValueError):
            eng.score(tokens, np.array(targets), top)


def test_more_sequences_than_the_rows_can_name(hip):
    """A row's sequence is searched in 32 bits: 2^31 - 1 sequences at most, whatever the views hold."""
    at = {n: hip.Buf((i + 1) << 44, 0, 1 << 43) for i, n in enumerate(("q", "k", "v", "q_norm", "k_norm", "q_out", "k_pool", "v_pool",
                                                                       "page_table", "starts", "seq_lens"))}
    for n, rc in ((2 ** 31 - 1, 3), (2 ** 31, 1), (2 ** 32 - 1, 1)):
        assert rc_of(hip, "ds5_hip_paged_append", append(hip, **at, n_seqs=n)) == rc


def test_score_refuses_before_it_runs(hip):
    """A vocabulary that the scores do not take is refused before the forward moves the engine on."""
    from qw3_amd import engine as E
    eng = E.Engine.__new__(E.Engine)
    eng.cfg, eng.ctx, eng.scores, eng.max_batch, ran = dict(vocab_size=hip.LOGPROBS_MAX_VOCAB + 1), None, [None] * 5, 1, []
    eng.forward = lambda *a, **k: ran.append(a)
    with pytest.raises(ValueError):
        eng.score([1], [1])
    assert not ran
