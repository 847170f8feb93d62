"""Decoding with the KV cache held in 4 bits: the model's steps over a 4-bit pool, its own pages or a
pool shared through kv_resize.

The twin computes each token with the CPU oracle's operators, in float32, but attends the K and V rows
that the GPU holds (read back with kv_q4_read), in 64 bits.  So a code that rounds the other way
because a projection's last bit differs moves both sides, and the logits are held to the decode steps' own
tolerance.  The held rows themselves are held to the rows that the twin computes: half a quantisation step,
and 2 % of one for the projections' rounding (1e-4 of a row's largest value, whose step is a seventh)."""
import numpy as np
import pytest

import oracle
from helpers import DECODE_LOGIT_TOL, max_err_vs_row_max
from test_kv_q4 import attend64, scale_of, status_word

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def held_rows(sess, layer, lane, n):
    from glacier_b200 import ops
    c = sess.dm.cfg
    p = torch.arange(n, device="cuda")
    slots = sess.block_tables[lane].long()[p // 16] * 16 + p % 16
    k, v = ops.kv_q4_read(sess.pages(), slots, c["num_layers"], layer, c["num_kv_heads"], c["head_dim"])
    return k.cpu().numpy().astype(np.float64), v.cpu().numpy().astype(np.float64)


def check_held(held, row):
    for h, x in zip(held.reshape(-1, 32), np.asarray(row, np.float64).reshape(-1, 32)):
        assert np.abs(h - x).max() <= 0.52 * scale_of(np.abs(x).max()) + 1e-12


def twin(m, sess, lane, token, pos, cos, sin):
    """Logits of `token` at `pos`, attending the rows that the session holds for the lane."""
    c = m.cfg
    D, F, H, Hkv, hd = c["dim"], c["hidden"], c["num_heads"], c["num_kv_heads"], c["head_dim"]
    qd, kvd, eps, G = H * hd, Hkv * hd, c["eps"], c["num_heads"] // c["num_kv_heads"]
    x = m.embedding[token].astype(np.float32)
    for i, L in enumerate(m.layers):
        h = oracle.rmsnorm(x, L["input_norm"], eps)
        q = oracle.linear_int4(h, *L["wq"], qd, D, 32)[0] + L["bq"]
        k = oracle.linear_int4(h, *L["wk"], kvd, D, 32)[0] + L["bk"]
        v = oracle.linear_int4(h, *L["wv"], kvd, D, 32)[0] + L["bv"]
        q = oracle.rope_apply(cos, sin, q, pos, H, hd)
        k = oracle.rope_apply(cos, sin, k, pos, Hkv, hd)
        ks, vs = held_rows(sess, i, lane, pos + 1)
        check_held(ks[pos], k)
        check_held(vs[pos], v)
        a = np.concatenate([attend64(q.reshape(H, hd)[j * G:(j + 1) * G], ks[:, j * hd:(j + 1) * hd],
                                     vs[:, j * hd:(j + 1) * hd]).ravel() for j in range(Hkv)]).astype(np.float32)
        x = x + oracle.linear_int4(a, *L["wo"], D, qd, 32)[0]
        h2 = oracle.rmsnorm(x, L["post_attn_norm"], eps)
        g = oracle.linear_int4(h2, *L["wg"], F, D, 32)[0]
        u = oracle.linear_int4(h2, *L["wu"], F, D, 32)[0]
        x = x + oracle.linear_int4(oracle.silu_mul(g, u), *L["wd"], D, F, 32)[0]
    return oracle.linear_int4(oracle.rmsnorm(x, m.final_norm, eps), *m.lm_head, c["vocab"], D, 32)[0]


def make(heads, kv_heads, hd, lanes, max_pages, dim=512, hidden=1024, **session):
    from glacier_b200.model import DecodeSession, DeviceModel, ModelConfig, SyntheticModel
    cfg = ModelConfig(num_layers=2, dim=dim, hidden=hidden, num_heads=heads, num_kv_heads=kv_heads, head_dim=hd,
                      vocab=1000)
    m = SyntheticModel(cfg, seed=5)
    dm = DeviceModel(m, max_positions=16 * max_pages)
    cos, sin = oracle.rope_table(16 * max_pages, hd, cfg.theta)
    return m, dm, DecodeSession(dm, lanes, max_pages, kv_format="q4", **session), cos, sin


@pytest.mark.parametrize("heads,kv_heads,hd,lanes", [(8, 2, 64, 3), (28, 4, 128, 2), (28, 4, 128, 6)])
def test_decode_over_a_4_bit_pool(heads, kv_heads, hd, lanes):
    """Few lanes (GEMV, the cluster attention) and tensor-core mode (split activations)."""
    m, dm, sess, cos, sin = make(heads, kv_heads, hd, lanes, 3)
    logits = torch.empty((lanes, 1000), dtype=torch.float32, device="cuda")
    cur = np.array([(37 * b + 11) % 1000 for b in range(lanes)], np.int32)
    for pos in range(19):
        out = sess.step(tokens=cur, positions=[pos] * lanes, logits=logits).cpu().numpy()
        if pos in (0, 1, 15, 16, 18):
            gl = logits.cpu().numpy()
            for b in range(lanes):
                assert max_err_vs_row_max(gl[b], twin(m, sess, b, int(cur[b]), pos, cos, sin)) <= DECODE_LOGIT_TOL
        cur = out.astype(np.int32)
    assert status_word() == 0
    sess.close()
    dm.close()


def test_prefill_then_decode():
    """A prompt in chunks, then steps behind it."""
    m, dm, sess, cos, sin = make(8, 2, 64, 5, 4, reserve_lanes=8)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (1, 8, 20, 33, 16)]
    logits = torch.empty(1000, dtype=torch.float32, device="cuda")
    first = []
    for b, p in enumerate(prompts):
        first.append(int(sess.prefill(p, lane=b, logits=logits)[0]))
        assert max_err_vs_row_max(logits.cpu().numpy(), twin(m, sess, b, p[-1], len(p) - 1, cos, sin)) <= DECODE_LOGIT_TOL
    step = torch.empty((5, 1000), dtype=torch.float32, device="cuda")
    pos = [len(p) for p in prompts]
    sess.step(tokens=first, positions=pos, logits=step)
    for b in range(5):
        assert max_err_vs_row_max(step[b].cpu().numpy(), twin(m, sess, b, first[b], pos[b], cos, sin)) <= DECODE_LOGIT_TOL
    assert status_word() == 0
    sess.close()
    dm.close()


def test_shared_pool_serves_requests_of_different_lengths():
    """Lanes grow, end and are admitted again from one pool of pages smaller than lanes * max_pages."""
    m, dm, sess, cos, sin = make(8, 2, 64, 3, 4, pool_pages=6)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (15, 31, 2)]  # 1 + 2 + 1 pages
    cur = [int(sess.prefill(p, lane=b)[0]) for b, p in enumerate(prompts)]
    logits = torch.empty((3, 1000), dtype=torch.float32, device="cuda")
    for k in range(3):  # lanes 0 and 1 cross a page border: all six pages are out
        out = sess.step(tokens=cur, logits=logits).cpu().numpy()
        assert sess.grow_status.tolist() == [0, 0, 0]
        assert sess.positions.tolist() == [len(p) + k for p in prompts]
        for b in range(3):
            ref = twin(m, sess, b, int(cur[b]), len(prompts[b]) + k, cos, sin)
            assert max_err_vs_row_max(logits[b].cpu().numpy(), ref) <= DECODE_LOGIT_TOL
        cur = out.tolist()
    assert int(sess.free_count) == 0
    with pytest.raises(MemoryError):
        sess.prefill([1] * 20, lane=2)
    assert sess.lens.tolist() == [18, 34, 5]
    sess.resize([18, 0, 5])  # request 1 ends
    assert int(sess.free_count) == 3
    new = rng.integers(0, 1000, 33).tolist()
    cur[1] = int(sess.prefill(new, lane=1)[0])
    sess.active.copy_(torch.tensor([1, 1, 0]))  # lane 2 waits
    sess.step(tokens=cur, logits=logits)
    assert sess.positions.tolist() == [18, 33, -1] and sess.lens.tolist() == [19, 34, 5]
    for b, pos in ((0, 18), (1, 33)):
        ref = twin(m, sess, b, int(cur[b]), pos, cos, sin)
        assert max_err_vs_row_max(logits[b].cpu().numpy(), ref) <= DECODE_LOGIT_TOL
    tables = sess.block_tables.cpu().numpy()
    used = [t for b, n in enumerate((19, 34, 5)) for t in tables[b, :-(-n // 16)]]
    assert len(set(used)) == len(used) == 6
    assert status_word() == 0  # an idle lane is no error
    sess.close()
    dm.close()


@pytest.mark.parametrize("shared", [False, True])
def test_captured_steps_equal_eager_ones(shared):
    runs = []
    for captured in (False, True):
        more = dict(pool_pages=7) if shared else {}
        m, dm, sess, cos, sin = make(8, 2, 64, 2, 3, **more)
        for b in range(2):
            sess.tokens[b] = int(sess.prefill([3 + b, 9, 27], lane=b)[0])
        if not shared:
            sess.positions.fill_(3)
        toks = []
        if captured:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                sess.capture_greedy_step(stream=s)
                for _ in range(20):
                    toks.append(sess.replay_greedy_step().clone())
            s.synchronize()
        else:
            for _ in range(20):
                out = sess.step()
                toks.append(out.clone())
                sess.tokens.copy_(out)
                if not shared:
                    sess.positions.add_(1)
        runs.append(torch.stack(toks).cpu().numpy())
        assert status_word() == 0
        sess.close()
        dm.close()
    np.testing.assert_array_equal(runs[0], runs[1])


def test_an_fp32_pool_can_be_shared_too():
    """kv_resize under FP32 pages: the tokens of a session with its own pages."""
    from glacier_b200.model import DecodeSession, DeviceModel, ModelConfig, SyntheticModel
    cfg = ModelConfig(num_layers=2, dim=256, hidden=512, num_heads=8, num_kv_heads=2, head_dim=64, vocab=1000)
    dm = DeviceModel(SyntheticModel(cfg, seed=7), max_positions=64)
    got = []
    for more in ({}, dict(pool_pages=5)):
        sess = DecodeSession(dm, 2, 4, **more)
        cur, toks = [int(sess.prefill([5, 6 + b], lane=b)[0]) for b in range(2)], []
        for k in range(18):
            cur = sess.step(tokens=cur, positions=None if more else [2 + k] * 2).tolist()
            toks.append(cur)
        got.append(toks)
        sess.close()
    assert got[0] == got[1]
    dm.close()


def test_a_prompt_that_is_refused_gives_its_pages_back():
    from glacier_b200 import _lib
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 4, pool_pages=6)
    sess.prefill([1, 2, 3], lane=0)
    with pytest.raises(_lib.GlacierCudaError):  # a mask of the wrong width
        sess.prefill([4] * 20, lane=1, eligible=torch.zeros((1, 3), dtype=torch.int64, device="cuda"))
    assert sess.lens.tolist() == [3, 0] and int(sess.free_count) == 5
    with pytest.raises(ValueError):
        sess.resize([5])  # one length for two lanes
    with pytest.raises(IndexError):
        sess.prefill([1], lane=2)
    assert sess.lens.tolist() == [3, 0]
    sess.close()
    dm.close()


def test_a_prompt_on_another_stream_follows_what_that_stream_still_does():
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 4, pool_pages=6)
    ref = int(sess.prefill([1, 2, 3, 4, 5], lane=1)[0])
    sess.resize([0, 0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(50):
            torch.randn((2048, 2048), device="cuda") @ torch.randn((2048, 2048), device="cuda")
    sess.resize([0, 3], stream=side)  # behind that work: the prompt has to go behind these positions
    sess.resize([0, 0], stream=side)
    first = sess.prefill([1, 2, 3], lane=1, stream=side)
    second = sess.prefill([4, 5], lane=1, stream=side)
    side.synchronize()
    assert sess.lens.tolist() == [0, 5] and int(second[0]) == ref
    sess.close()
    dm.close()


def test_refusals():
    from glacier_b200 import _lib
    from glacier_b200.model import DecodeSession, DeviceModel, ModelConfig, SyntheticModel
    cfg = ModelConfig(num_layers=1, dim=256, hidden=512, num_heads=8, num_kv_heads=2, head_dim=32, vocab=100)
    dm = DeviceModel(SyntheticModel(cfg, seed=7), max_positions=64)
    with pytest.raises(_lib.GlacierCudaError):
        DecodeSession(dm, 2, 4, kv_format="q4")  # 32-dim heads
    with pytest.raises(ValueError):
        DecodeSession(dm, 2, 4, kv_format="q8")
    sess = DecodeSession(dm, 2, 4)
    with pytest.raises(ValueError):
        sess.resize([1, 1])
    L = _lib.lib()
    assert not L.glacier_cuda_kv_create_q4(dm.h, 0) and not L.glacier_cuda_kv_create_q4(None, 4)
    assert not L.glacier_cuda_kv_q4_pages(sess.kv) and L.glacier_cuda_kv_page_bytes(sess.kv) == 4 * sess.page_floats
    sess.close()
    dm.close()


def test_a_position_or_page_out_of_range_is_reported():
    m, dm, sess, cos, sin = make(8, 2, 64, 3, 2)
    logits = torch.empty((3, 1000), dtype=torch.float32, device="cuda")
    sess.step(tokens=[1, 2, 3], positions=[0, 32, 0], logits=logits)  # past the table
    assert status_word() == 2
    sess.block_tables[2, 0] = -1
    sess.step(tokens=[1, 2, 3], positions=[1, 0, 0], logits=logits)  # no page
    assert status_word() == 2
    for b, pos in ((0, 1), (1, 0)):
        ref = twin(m, sess, b, b + 1, pos, cos, sin)
        assert max_err_vs_row_max(logits[b].cpu().numpy(), ref) <= DECODE_LOGIT_TOL
    sess.close()
    dm.close()


def captured_tokens(sess, stream, kept, active=None):
    """One replay; the tokens of the lanes that advanced go to `kept`."""
    if active is not None:
        sess.active.copy_(torch.tensor(active, dtype=torch.int32))
    out = sess.replay_greedy_step().tolist()
    for b, p in enumerate(sess.positions.tolist()):
        if p >= 0:
            kept[b].append(out[b])


@pytest.mark.parametrize("kv_format", ["q4", "f32"])
def test_a_captured_loop_keeps_the_token_of_a_lane_that_waits(kv_format):
    """A lane that gets no page, and one that is paused, go on from their own tokens: every lane's tokens are
    those of a session in which nobody waits."""
    from glacier_b200.model import DecodeSession
    prompts = [[3, 9, 27, 81, 243, 729, 5, 15, 45, 135, 405, 2, 6, 18], list(range(40, 55)), [7, 77, 777, 70]]
    m, dm, own, cos, sin = make(8, 2, 64, 3, 3)
    own.close()
    own = DecodeSession(dm, 3, 3, kv_format=kv_format)
    cur = [int(own.prefill(p, lane=b)[0]) for b, p in enumerate(prompts)]
    free_run = [[] for _ in prompts]
    for k in range(9):
        cur = own.step(tokens=cur, positions=[len(p) + k for p in prompts]).tolist()
        for b in range(3):
            free_run[b].append(cur[b])
    own.close()
    sess = DecodeSession(dm, 3, 3, kv_format=kv_format, pool_pages=4)
    for b, p in enumerate(prompts):
        sess.tokens[b] = int(sess.prefill(p, lane=b)[0])
    s, kept = torch.cuda.Stream(), [[], [], []]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sess.capture_greedy_step(stream=s)
        for _ in range(2):
            captured_tokens(sess, s, kept)
        assert sess.lens.tolist() == [16, 17, 6] and int(sess.free_count) == 0
        pending = int(sess.tokens[0])
        captured_tokens(sess, s, kept)  # lane 0 gets no page
        assert sess.grow_status.tolist() == [-3, 0, 0] and sess.positions.tolist() == [-1, 17, 6]
        assert int(sess.tokens[0]) == pending
        captured_tokens(sess, s, kept, active=[1, 0, 1])  # and lane 1 is paused
        assert sess.positions.tolist() == [-1, -1, 7] and int(sess.tokens[0]) == pending
        sess.resize([16, 18, 0], stream=s)  # request 2 ends: its page goes to lane 0
        for _ in range(3):
            captured_tokens(sess, s, kept, active=[1, 0, 0])
        for _ in range(3):
            captured_tokens(sess, s, kept, active=[1, 1, 0])
    s.synchronize()
    assert [len(k) for k in kept] == [8, 6, 4]
    assert kept == [run[:len(k)] for run, k in zip(free_run, kept)]
    status_word()  # an FP32 pool reports the lanes that waited
    sess.close()
    dm.close()


def test_an_idle_lane_of_a_captured_loop_stays_idle():
    """Lanes with their own pages: position -1 is no position that a replay counts on from."""
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 2)
    ref = [int(sess.prefill([3, 9, 27], lane=0)[0])]
    for k in range(4):
        ref.append(int(sess.step(tokens=[ref[-1], 5], positions=[3 + k, -1])[0]))
    sess.tokens.copy_(torch.tensor([ref[0], 5]))
    sess.positions.copy_(torch.tensor([3, -1]))
    before = sess.pages()[2:].clone()
    s, got = torch.cuda.Stream(), []
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sess.capture_greedy_step(stream=s)
        for _ in range(4):
            got.append(int(sess.replay_greedy_step()[0]))
    s.synchronize()
    assert got == ref[1:]
    assert sess.positions.tolist() == [7, -1] and int(sess.tokens[1]) == 5
    assert torch.equal(sess.pages()[2:], before)  # nothing was written for the idle lane
    assert status_word() == 0
    sess.close()
    dm.close()


def test_a_refused_step_leaves_the_session_as_it_was():
    from glacier_b200 import _lib
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 3, pool_pages=4)
    cur = [int(sess.prefill(list(range(b + 1, b + n)), lane=b)[0]) for b, n in ((0, 17), (1, 6))]  # 16 and 5 positions
    sess.active.copy_(torch.tensor([1, 0]))
    sess.tokens.copy_(torch.tensor(cur))
    state = lambda: [t.clone() for t in (sess.lens, sess.free_count, sess.free_pages[:2], sess.block_tables[1],  # noqa: E731
                                         sess.block_tables[0, :1], sess.tokens)]
    before = state()
    with pytest.raises(_lib.GlacierCudaError):  # a mask of the wrong width: lane 0 had taken a page by then
        sess.step(eligible=torch.zeros((2, 3), dtype=torch.int64, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(state(), before))
    with pytest.raises(ValueError):
        sess.step(tokens=[1, 2], positions=[16, 5])
    assert all(torch.equal(a, b) for a, b in zip(state(), before))
    logits = torch.empty((2, 1000), dtype=torch.float32, device="cuda")
    sess.step(logits=logits)
    assert sess.positions.tolist() == [16, -1]
    assert max_err_vs_row_max(logits[0].cpu().numpy(), twin(m, sess, 0, cur[0], 16, cos, sin)) <= DECODE_LOGIT_TOL
    assert status_word() == 0
    sess.close()
    dm.close()


def test_a_prompt_of_a_shared_pool_starts_behind_the_lane():
    """A start that is not the lane's length is refused, not dropped."""
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 4, pool_pages=6)
    whole = int(sess.prefill([1, 2, 3, 4, 5], lane=1)[0])
    sess.resize([0, 0])
    sess.prefill([1, 2, 3], lane=1, start=0)
    for start in (0, 2, 4, -1):
        with pytest.raises(ValueError):
            sess.prefill([4, 5], lane=1, start=start)
    assert sess.lens.tolist() == [0, 3] and int(sess.free_count) == 5
    assert int(sess.prefill([4, 5], lane=1, start=3)[0]) == whole
    assert sess.lens.tolist() == [0, 5]
    sess.close()
    dm.close()


def test_a_prompt_that_no_pages_could_hold_is_not_short_of_memory():
    """MemoryError is for a pool that has no pages now; a prompt longer than the block table never fits."""
    from glacier_b200 import _lib
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 4, pool_pages=6)
    sess.prefill([1] * 20, lane=0)
    for lane, n in ((0, 45), (1, 65), (1, 1000)):
        with pytest.raises(_lib.GlacierCudaError) as e:
            sess.prefill([1] * n, lane=lane)
        assert e.value.code == _lib.EINVAL
    sess.prefill([1] * 33, lane=1)  # three of the four pages that were left
    with pytest.raises(MemoryError):
        sess.prefill([1] * 44, lane=0)
    assert sess.lens.tolist() == [20, 33] and int(sess.free_count) == 1
    sess.close()
    dm.close()


def busy(stream, n=60):
    """Work that keeps `stream` behind the host for a while."""
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a = torch.randn((4096, 4096), device="cuda")
        for _ in range(n):
            a @ a


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("on_device", [False, True])
def test_prompts_on_another_stream_keep_their_tokens(shared, on_device):
    """Two prompts of several chunks, one behind the other on a stream that is busy: neither sees the other's
    tokens, nor what is allocated when the caller has dropped its prompt."""
    more = dict(pool_pages=8) if shared else {}
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 4, reserve_lanes=8, **more)
    rng = np.random.default_rng(9)
    prompts = [rng.integers(0, 1000, 40).tolist() for _ in range(2)]
    ref = [int(sess.prefill(p, lane=b)[0]) for b, p in enumerate(prompts)]
    if shared:
        sess.resize([0, 0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    busy(side)
    first = []
    for b, p in enumerate(prompts):
        p = torch.tensor(p, dtype=torch.int32, device="cuda") if on_device else p
        if on_device:
            torch.cuda.current_stream().synchronize()  # the prompt is there; how long it stays is not the caller's care
        first.append(sess.prefill(p, lane=b, stream=side))
        del p
        junk = [torch.zeros(40, dtype=torch.int32, device="cuda") for _ in range(4)]
    side.synchronize()
    assert [int(t) for t in first] == ref and len(junk) == 4
    assert status_word() == 0
    sess.close()
    dm.close()


def test_steps_on_another_stream_take_their_inputs_there():
    """Tokens, positions and lengths are copied behind the steps that still read the ones before."""
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 4)
    inputs = [([3 + k, 500 + k], [k, k]) for k in range(4)]
    ref = [torch.empty((2, 1000), device="cuda") for _ in inputs]
    for (tokens, positions), logits in zip(inputs, ref):
        sess.step(tokens=tokens, positions=positions, logits=logits)
    sess.pages().zero_()
    got = [torch.empty_like(r) for r in ref]
    side = torch.cuda.Stream()
    busy(side)
    for (tokens, positions), logits in zip(inputs, got):
        sess.step(tokens=torch.tensor(tokens).pin_memory(), positions=torch.tensor(positions).pin_memory(), logits=logits,
                  stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    sess.close()
    m, dm2, sess, cos, sin = make(8, 2, 64, 2, 4, pool_pages=6)
    late = torch.zeros(2, dtype=torch.int64, device="cuda")
    busy(side)
    with torch.cuda.stream(side):
        late.copy_(torch.tensor([20, 7]).pin_memory(), non_blocking=True)
    sess.resize(late, stream=side)
    side.synchronize()
    assert sess.lens.tolist() == [20, 7]
    sess.close()
    dm.close()
    dm2.close()


@pytest.mark.parametrize("kv_format", ["q4", "f32"])
def test_a_pool_of_another_model_is_refused(kv_format):
    """A pool's pages have to be the model's: one of smaller pages would be written past its end."""
    from glacier_b200 import _lib
    from glacier_b200.model import DecodeSession, DeviceModel, ModelConfig, SyntheticModel
    i32 = dict(dtype=torch.int32, device="cuda")
    dms, sess = [], []
    for layers in (1, 3):
        cfg = ModelConfig(num_layers=layers, dim=256, hidden=512, num_heads=8, num_kv_heads=2, head_dim=64, vocab=100)
        dms.append(DeviceModel(SyntheticModel(cfg, seed=7), max_positions=64))
        sess.append(DecodeSession(dms[-1], 2, 4, kv_format=kv_format))
    prompt, out = torch.ones(3, **i32), torch.zeros(1, **i32)
    for a in (0, 1):
        s, kv = sess[a], sess[1 - a].kv
        for name, args in (("glacier_cuda_decode_step",
                            (2, s.tokens.data_ptr(), s.positions.data_ptr(), s.block_tables.data_ptr(), 4, None, 0,
                             s.out.data_ptr(), None, None, None)),
                           ("glacier_cuda_prefill", (prompt.data_ptr(), 3, 0, s.block_tables.data_ptr(), 4, None, 0,
                                                     out.data_ptr(), None, None, None))):
            with pytest.raises(_lib.GlacierCudaError) as e:
                _lib.call(name, dms[a].h, kv, *args)
            assert e.value.code == _lib.EINVAL
        assert int(s.prefill([1, 2, 3])[0]) >= 0 and len(s.step(positions=[3, 0]).tolist()) == 2
    assert status_word() == 0
    for x in sess + dms:
        x.close()


def test_a_mask_that_is_no_tensor_leaves_the_session_as_it_was():
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 3, pool_pages=4)
    sess.prefill([1] * 16, lane=0)
    with pytest.raises(AttributeError):
        sess.step(tokens=[1, 2], eligible=[1, 2])
    with pytest.raises(AttributeError):
        sess.prefill([1, 2], lane=1, eligible=[1, 2])
    assert sess.lens.tolist() == [16, 0] and int(sess.free_count) == 3
    sess.close()
    dm.close()


def test_masks_and_logits_on_another_stream_are_kept():
    """A mask that the caller drops, and logits memory that nobody else may get, while the step is still to come."""
    m, dm, sess, cos, sin = make(8, 2, 64, 2, 4, reserve_lanes=8)
    words = torch.zeros((2, 16), dtype=torch.int64, device="cuda")
    words[:, 3] = 1 << 7  # token 199 alone
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy(side)
    mask, logits = words.clone(), torch.empty((2, 1000), device="cuda")
    torch.cuda.current_stream().synchronize()
    out = sess.step(positions=torch.zeros(2, dtype=torch.int32, device="cuda"), eligible=mask, logits=logits, stream=side)
    del mask, logits
    junk = [torch.full((2, 16), -1, dtype=torch.int64, device="cuda") for _ in range(4)]
    rows = [torch.full((2, 1000), 3.0, device="cuda") for _ in range(4)]
    side.synchronize()
    assert out.tolist() == [199, 199] and len(junk) == 4 and all((r == 3).all() for r in rows)
    busy(side)
    prompt = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    mask = words[:1].clone()
    torch.cuda.current_stream().synchronize()
    first = sess.prefill(prompt, lane=1, eligible=mask, stream=side)
    del mask
    junk = [torch.full((1, 16), -1, dtype=torch.int64, device="cuda") for _ in range(4)]
    side.synchronize()
    assert int(first) == 199
    sess.close()
    dm.close()
