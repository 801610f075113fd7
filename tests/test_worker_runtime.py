"""Worker runtime: poison jobs fail on their own and
oversized batches are split to the engine's capacity.  CPU-only, in-proc
fake Redis, the mock CPU engine."""
import os

import pytest

from kiosk_autoscaler_amd.models import mlp
from kiosk_autoscaler_amd.worker import runtime as rt


class _Channel(object):
    def __init__(self):
        self.events = []
        self.direct = {}

    def emit(self, ev, **fields):
        self.events.append((ev, fields))


def _runtime(redis_client, batch=1, rows=64, kind='deployment'):
    env = {'ROWS_PER_KEY': str(rows), 'WORKER_BATCH': str(batch),
           'MOCK_WORK_MS': '0', 'QUEUES': 'predict'}
    cfg = rt.WorkerConfig(env, {'worker_id': 'w-g0-x-1', 'kind': kind})
    run = rt.WorkerRuntime(cfg, None, _Channel(), lambda: redis_client)
    run.redis = redis_client
    run.engine = mlp.CpuMlpEngine(cfg)
    return run


def _push(client, name, **fields):
    client.hset(name, mapping=dict({'status': 'new'}, **fields))
    client.lpush('predict', name)


def test_oversized_job_fails_alone_and_worker_keeps_serving(redis_client):
    run = _runtime(redis_client)
    consumer = rt.QueueConsumer(redis_client, 'w-g0-x-1', ['predict'])
    _push(redis_client, 'predict:bad', rows=10 ** 9)
    _push(redis_client, 'predict:good', rows=8)
    for _ in range(2):
        run._process(consumer, consumer.pull(limit=1, block=False))
    bad = redis_client.hgetall('predict:bad')
    assert bad['status'] == 'failed' and 'rows=' in bad['reason']
    assert redis_client.hget('predict:good', 'status') == 'done'
    # the poison job is not requeued: no processing key is left behind
    assert not list(redis_client.scan_iter(match='processing-predict:*'))
    assert run.keys_done == 1


@pytest.mark.parametrize('field,value', [('rows', '0'), ('passes', '-3'),
                                         ('service_ms', '99999999'),
                                         ('rows', 'many')])
def test_invalid_fields_rejected(redis_client, field, value):
    run = _runtime(redis_client)
    redis_client.hset('predict:j', mapping={'status': 'new', field: value})
    with pytest.raises(rt.JobError):
        run._job_params('predict:j')


def test_engine_rejection_marks_batch_failed(redis_client):
    run = _runtime(redis_client)

    def reject(rows, passes, seed):
        raise ValueError('rows must be in [1, max_rows]')
    run.engine.forward = reject
    consumer = rt.QueueConsumer(redis_client, 'w-g0-x-1', ['predict'])
    _push(redis_client, 'predict:a', rows=8)
    run._process(consumer, consumer.pull(limit=1, block=False))
    assert redis_client.hget('predict:a', 'status') == 'failed'
    assert not list(redis_client.scan_iter(match='processing-predict:*'))


def test_batch_split_to_engine_capacity(redis_client):
    run = _runtime(redis_client, batch=4, rows=64, kind='job')
    calls = []
    real = run.engine.forward

    def forward(rows, passes, seed):
        calls.append(rows)
        return real(rows, passes, seed)
    run.engine.forward = forward
    limit = run.max_rows()             # max(64 * 4, 256) = 256
    for i in range(4):
        _push(redis_client, 'predict:j%d' % i, rows=100)
    consumer = rt.QueueConsumer(redis_client, 'w-g0-x-1', ['predict'])
    run._process(consumer, consumer.pull(limit=4, block=False))
    assert all(r <= limit for r in calls) and sum(calls) == 400
    assert len(calls) == 2
    assert all(redis_client.hget('predict:j%d' % i, 'status') == 'done'
               for i in range(4))


def test_cold_spawn_opens_the_device_on_a_helper_thread(monkeypatch):
    """Cold spawn: ``preinit_device`` runs on a helper thread while the main
    thread imports and connects; the engine joins it and records its
    stamps.  A failing open is left to the engine's own init to report."""
    import threading
    from kiosk_autoscaler_amd.ops import native
    from kiosk_autoscaler_amd.worker import main as worker_main
    release = threading.Event()

    class FakeMod(object):
        fail = False

        def preinit_device(self, device):
            release.wait(10)
            if self.fail:
                raise RuntimeError('no device')
            return {'preinit_enter': 1, 'preinit_done': 2}
    mod = FakeMod()
    monkeypatch.setattr(native, 'load', lambda **kw: mod)
    worker_main._open_device_async()
    assert worker_main._DEVICE_OPEN['thread'].is_alive()   # not joined yet
    release.set()
    stages = []
    worker_main._join_device_open(lambda name, t=None: stages.append(name))
    assert stages == ['preinit_enter', 'preinit_done', 'device_open_joined']
    worker_main._join_device_open()          # idempotent
    mod.fail = True
    worker_main._DEVICE_OPEN.clear()
    worker_main._open_device_async()
    worker_main._join_device_open()
    assert 'no device' in worker_main._DEVICE_OPEN['error']
    worker_main._DEVICE_OPEN.clear()


COLD = """
import os, sys, threading
from kiosk_autoscaler_amd.ops import native
from kiosk_autoscaler_amd.worker import main as worker_main


class Mod(object):
    def preinit_device(self, device):
        print('opened on', threading.current_thread().name, flush=True)
        return {'preinit_done': 1}

    def release_kept_stream(self):
        pass


class Runtime(object):
    recycle, keys_done = False, 0


def serve(assignment, backend, channel, node_agent=None):
    print('serving', flush=True)
    if sys.argv[2] == 'engine':
        worker_main._join_device_open(
            lambda name, t=None: print(name, flush=True))
    return 0, Runtime()


native.load = lambda **kw: Mod()
worker_main._serve = serve
worker_main.main(['--backend', 'hip', '--assign', '{"gpu": "0"}'],
                 **eval(sys.argv[1]))
"""


@pytest.mark.parametrize('how,engine,want', [
    ({'forked': True}, 'engine',
     ['opened on device-open', 'serving', 'preinit_done',
      'device_open_joined']),
    ({}, 'engine', ['serving', 'opened on MainThread', 'preinit_done',
                    'device_open_joined']),
    # an assignment that ends before its engine opens nothing
    ({}, 'none', ['serving'])])
def test_only_a_forked_worker_opens_the_device_on_a_helper_thread(
        how, engine, want):
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run(
        [sys.executable, '-c', COLD, repr(how), engine], text=True,
        capture_output=True, timeout=60, cwd=root,
        env=dict(os.environ, FENCE='none', PYTHONPATH=root))
    lines = done.stdout.split('\n')[:-1]
    # (beside the main thread's own steps the helper thread may be late)
    assert (sorted(lines) if how else lines) == \
        (sorted(want) if how else want), (lines, done.stderr)


def test_zygote_tells_the_worker_that_it_is_forked(monkeypatch):
    import socket
    from kiosk_autoscaler_amd.worker import main as worker_main
    from kiosk_autoscaler_amd.worker import zygote
    calls = []

    class Ended(Exception):
        pass

    def end(code):
        raise Ended
    monkeypatch.setattr(worker_main, 'main',
                        lambda argv, **kw: calls.append((argv, kw)) or 0)
    monkeypatch.setattr(os, '_exit', end)
    monkeypatch.setattr(os, 'setsid', lambda: None)
    monkeypatch.setattr(os, 'close', lambda fd: None)
    monkeypatch.setattr(zygote.signal, 'signal', lambda *a: None)
    monkeypatch.setattr(os, 'environ', dict(os.environ))
    monkeypatch.setattr('sys.argv', ['x'])
    ours, theirs = socket.socketpair()
    with pytest.raises(Ended):
        zygote._child({'env': {}, 'argv': ['--backend', 'hip']}, (7, 8),
                      theirs)
    ours.close()
    assert calls == [(['--backend', 'hip'], {'forked': True})]


class _FenceAgent(object):
    def __init__(self):
        self.calls = []

    def submit(self, message):
        self.calls.append(('submit', message.get('cmd')))

    def close(self):
        self.calls.append(('close',))
        return True

    def abandon(self):
        self.calls.append(('abandon',))


@pytest.mark.parametrize('recycle', [True, False])
def test_exiting_worker_leaves_the_communicator_to_process_exit(
        redis_client, recycle):
    """A drained worker that goes back to the pool releases its fence
    communicator gracefully; one that exits abandons it (its process exit
    frees it: a graceful RCCL finalize only kept the GPU alive longer)."""
    import queue
    channel = _Channel()
    channel.commands = queue.Queue()
    channel.start_reader = lambda: None
    channel.commands.put({'cmd': 'drain', 'recycle': recycle})
    env = {'ROWS_PER_KEY': '64', 'MOCK_WORK_MS': '0', 'QUEUES': 'predict',
           'WARM_START': '1'}
    cfg = rt.WorkerConfig(env, {'worker_id': 'w-g0-x-2', 'recycle': True})
    agent = _FenceAgent()
    run = rt.WorkerRuntime(cfg, lambda c, stage: mlp.CpuMlpEngine(c),
                           channel, lambda: redis_client,
                           fence_factory=lambda runtime: agent)
    assert run.run() == 0
    assert run.recycle is recycle
    assert agent.calls == [('close',) if recycle else ('abandon',)]
    assert 'fence' not in channel.direct      # unhooked either way


def test_multi_queue_pull_is_round_robin(redis_client):
    """QUEUES=predict,track: a backlog on the first queue does not starve
    the second (each sweep starts one queue further)."""
    for i in range(4):
        redis_client.lpush('predict', 'predict:%d' % i)
        redis_client.lpush('track', 'track:%d' % i)
    consumer = rt.QueueConsumer(redis_client, 'w-g0-x-3',
                                ['predict', 'track'])
    order = []
    for _ in range(4):
        for queue, item, pkey in consumer.pull(limit=1, block=False):
            order.append(queue)
            consumer.complete(pkey)
    assert order == ['predict', 'track', 'predict', 'track']


class _Agreement(object):
    """Stands in for NodeFenceAgent.agreement (the rank's own result)."""

    def __init__(self):
        self.by_group = {}

    def agreement(self, group):
        return self.by_group.get(group)


def test_worker_fenced_out_stops_pulling(redis_client):
    """A worker serves ungated until a fence includes it; once a newer
    agreed membership excludes its slot it takes no more keys, and a later
    fence that includes it again resumes it."""
    agent = _Agreement()
    group = 'default/w'
    agent.by_group[group] = {'seq': 3, 'epoch': 2, 'slots': []}   # stale
    env = {'ROWS_PER_KEY': '8', 'MOCK_WORK_MS': '0', 'QUEUES': 'predict'}
    cfg = rt.WorkerConfig(env, {'worker_id': 'w-g1-x-1', 'slot': 1,
                                'namespace': 'default', 'resource': 'w'})
    run = rt.WorkerRuntime(cfg, None, _Channel(), lambda: redis_client,
                           node_agent=agent)
    run._gate_base = agent.agreement(group)['seq']
    assert not run.excluded()                 # nothing newer: ungated
    agent.by_group[group] = {'seq': 4, 'epoch': 3, 'slots': [0]}
    assert not run.excluded()                 # never included yet
    agent.by_group[group] = {'seq': 5, 'epoch': 4, 'slots': [0, 1]}
    assert not run.excluded()
    agent.by_group[group] = {'seq': 6, 'epoch': 5, 'slots': [0]}
    assert run.excluded() and run.fenced_out
    assert ('fenced_out', {'seq': 6}) in run.channel.events
    agent.by_group[group] = {'seq': 7, 'epoch': 6, 'slots': [1]}
    assert not run.excluded()
    assert ('fenced_in', {'seq': 7}) in run.channel.events


class _Emits(object):
    def __init__(self):
        self.out = []

    def emit(self, ev, **fields):
        self.out.append(dict(fields, ev=ev))


def test_standby_prebuild_builds_the_engine_the_assignment_reuses(
        monkeypatch):
    """An arrival-woken standby (pin ``prebuild``) builds the engine for the
    resource's shape before any assignment: the assignment with the same
    model gets it from the cache; a failed prebuild leaves nothing cached
    and reports the error."""
    from kiosk_autoscaler_amd.worker import main as wm
    monkeypatch.setenv('MODEL_DIM', '64')
    monkeypatch.setenv('MODEL_HIDDEN', '128')
    monkeypatch.setenv('MODEL_LAYERS', '1')
    monkeypatch.setenv('ROWS_PER_KEY', '16')
    monkeypatch.delenv('WORKER_ENGINE', raising=False)
    wm._ENGINES.clear()
    chan = _Emits()
    try:
        wm._prebuild_engine('cpu', {'slot': 0, 'gpu': '', 'prebuild': {
            'kind': 'deployment', 'keys_per_pod': 1}}, chan)
        built = [e for e in chan.out if e['ev'] == 'prebuilt']
        assert built and 'error' not in built[0] and len(wm._ENGINES) == 1
        cfg = rt.WorkerConfig(os.environ, {'worker_id': 'w', 'slot': 0})
        engine = wm._cached_engine('cpu', cfg, None)
        assert engine.reused is True
        # a failure is contained: nothing stays cached
        chan = _Emits()

        def boom(*args):
            raise RuntimeError('no device')
        monkeypatch.setattr(wm, '_cached_engine', boom)
        wm._prebuild_engine('cpu', {'prebuild': {}}, chan)
        assert 'no device' in chan.out[-1]['error'] and not wm._ENGINES
    finally:
        wm._drop_cached_engines()


def test_worker_config_reads_model_and_prefers_the_parsed_sizes():
    """A standalone worker reads the autoscaler's MODEL knob; the
    manager's parsed MODEL_DIM / MODEL_HIDDEN / MODEL_LAYERS win."""
    cfg = rt.WorkerConfig({'MODEL': '512x2048x2'}, {'worker_id': 'w'})
    assert (cfg.dim, cfg.hidden, cfg.layers) == (512, 2048, 2)
    cfg = rt.WorkerConfig({'MODEL': '512x2048x2', 'MODEL_DIM': '1024'},
                          {'worker_id': 'w'})
    assert (cfg.dim, cfg.hidden, cfg.layers) == (1024, 2048, 2)
    cfg = rt.WorkerConfig({}, {'worker_id': 'w'})
    assert (cfg.dim, cfg.hidden, cfg.layers) == (4096, 16384, 4)


class _FakeHsa(object):
    def __init__(self):
        self.calls = []

    def hsa_init(self):
        self.calls.append('init')
        return 0

    def hsa_shut_down(self):
        self.calls.append('shut_down')
        return 0


def _settled(monkeypatch, zygote_rocr, argv, env, delay=0.0, gpu=None):
    """An embryo's ROCr init under the zygote's environment, then its
    hand-off of a request whose env is the manager's (the zygote's, as
    ``_spawn`` passes it) with ``env`` on top."""
    from kiosk_autoscaler_amd.worker import zygote
    lib = _FakeHsa()
    monkeypatch.setattr('ctypes.CDLL', lambda *a, **k: lib)
    if zygote_rocr is None:
        monkeypatch.delenv('ROCR_VISIBLE_DEVICES', raising=False)
    else:
        monkeypatch.setenv('ROCR_VISIBLE_DEVICES', zygote_rocr)
    request_env = {k: v for k, v in os.environ.items()
                   if k != 'ROCR_VISIBLE_DEVICES'}
    request_env.update(env)
    pre = zygote._HsaPreinit()
    pre.DELAY_S = delay
    pre.start(gpu)
    if gpu is not None:
        # (the embryo process binds itself: undo it for the next test)
        monkeypatch.setenv('ROCR_VISIBLE_DEVICES', str(gpu))
    if delay == 0.0:
        pre.thread.join()
    request = {'argv': argv, 'env': request_env}
    stamp = pre.settle(request)
    return stamp, lib.calls, request


def test_embryo_keeps_rocr_when_the_pin_matches(monkeypatch):
    """The 1-GPU box: ROCR_VISIBLE_DEVICES=0 and the worker pins GPU 0."""
    stamp, calls, _ = _settled(monkeypatch, '0',
                               ['--pin', '{"gpu": 0}'],
                               {'ROCR_VISIBLE_DEVICES': '0'})
    assert calls == ['init'] and isinstance(stamp, int)


def test_embryo_keeps_rocr_under_hip_level_pinning(monkeypatch):
    # ROCR unset: the pin is HIP_VISIBLE_DEVICES, applied at hipInit
    stamp, calls, _ = _settled(monkeypatch, None,
                               ['--pin', '{"gpu": 5}'], {})
    assert calls == ['init'] and stamp is not None


def test_embryo_shuts_rocr_down_when_the_pin_differs(monkeypatch):
    """A node filtering at the ROCr level: the worker's GPU 3 re-filters
    ROCR_VISIBLE_DEVICES, which the early init would have missed."""
    stamp, calls, _ = _settled(monkeypatch, '0,1,2,3',
                               ['--pin', '{"gpu": 1}', '--assign',
                                '{"gpu": 3}'],
                               {'ROCR_VISIBLE_DEVICES': '0,1,2,3'})
    assert calls == ['init', 'shut_down'] and stamp is None


def test_embryo_request_before_the_delay_skips_the_init(monkeypatch):
    stamp, calls, _ = _settled(monkeypatch, None, [], {}, delay=30.0)
    assert calls == [] and stamp is None


def test_slot_bound_embryo_keeps_rocr_for_its_gpu(monkeypatch):
    """an embryo bound to GPU 6 initialises ROCr with
    ROCR_VISIBLE_DEVICES=6 (that device alone); a worker for GPU 6 keeps
    the init and pins at the ROCr level too."""
    stamp, calls, request = _settled(monkeypatch, None,
                                     ['--pin', '{"gpu": "6"}'], {}, gpu='6')
    assert calls == ['init'] and stamp is not None
    assert request['env']['ROCR_VISIBLE_DEVICES'] == '6'
    from kiosk_autoscaler_amd.worker.zygote import _worker_env
    worker = _worker_env(request)
    assert worker['ROCR_VISIBLE_DEVICES'] == '6'
    assert 'HIP_VISIBLE_DEVICES' not in worker


def test_slot_bound_embryo_of_another_gpu_is_shut_down(monkeypatch):
    """A slot-bound embryo handed a request for another GPU shuts its
    ROCr down instead of keeping a runtime that opened the wrong device."""
    stamp, calls, request = _settled(monkeypatch, None,
                                     ['--pin', '{"gpu": "2"}'], {}, gpu='6')
    assert calls == ['init', 'shut_down'] and stamp is None
    assert 'ROCR_VISIBLE_DEVICES' not in request['env']


def test_slot_bound_embryo_under_the_visible_pin_is_shut_down(monkeypatch):
    """WORKER_PIN=visible: the worker keeps every managed GPU visible, so an
    init bound to its GPU alone cannot be kept -- shut down, and the
    request's environment is left as the manager sent it."""
    import json
    pin = {'gpu': '6', 'visible': ['4', '5', '6', '7']}
    stamp, calls, request = _settled(monkeypatch, None,
                                     ['--pin', json.dumps(pin)], {}, gpu='6')
    assert calls == ['init', 'shut_down'] and stamp is None
    assert 'ROCR_VISIBLE_DEVICES' not in request['env']


def test_embryo_of_another_template_shuts_rocr_down(monkeypatch):
    """an HSA_* setting the assignment's template env changes
    (SDMA off here) was silently ignored by a kept init."""
    import json
    assign = {'gpu': '6', 'template': {'env': {'HSA_ENABLE_SDMA': '0'}}}
    stamp, calls, _ = _settled(monkeypatch, None,
                               ['--assign', json.dumps(assign)], {},
                               gpu='6')
    assert calls == ['init', 'shut_down'] and stamp is None


def test_requests_go_to_the_embryo_bound_to_their_gpu(monkeypatch):
    import json
    from kiosk_autoscaler_amd.worker import zygote
    made = []
    monkeypatch.setattr(zygote, '_double_fork',
                        lambda body: made.append(len(made) + 200) or made[-1])
    stock = zygote._Embryos(4, rocr=2, gpus=['0', '1'])
    for _ in range(4):
        assert stock.make()
    assert [r for _, _, r in stock.ready] == ['0', '1', False, False]
    monkeypatch.setattr('socket.send_fds', lambda sock, bufs, fds: None)

    def req(gpu):
        return json.dumps({'argv': ['--pin', json.dumps({'gpu': gpu})],
                           'env': {}}).encode()
    assert stock.hand(req('1'), []) == 201      # bound to GPU 1
    assert stock.hand(req('5'), []) == 202      # no GPU 5 embryo: a plain one
    stock.make()                                 # GPU 1's replacement
    assert [r for _, _, r in stock.ready] == ['0', False, '1']
    assert stock.hand(req('1'), []) == 204


def test_rocr_embryos_are_made_up_to_the_cap_and_handed_first(monkeypatch):
    from kiosk_autoscaler_amd.worker import zygote
    made = []

    def fake_fork(body):
        made.append(len(made) + 100)
        return made[-1]
    monkeypatch.setattr(zygote, '_double_fork', fake_fork)
    stock = zygote._Embryos(4, rocr=2)
    for _ in range(4):
        assert stock.make()
    assert [r for _, _, r in stock.ready] == [True, True, False, False]
    sent = []
    monkeypatch.setattr('socket.send_fds',
                        lambda sock, bufs, fds: sent.append(sock))
    assert stock.hand(b'{}', []) == 100
    # the replacement for a handed-out ROCr embryo initialises ROCr too
    stock.make()
    assert [r for _, _, r in stock.ready] == [True, False, False, True]
    assert stock.hand(b'{}', []) == 101
    assert stock.hand(b'{}', []) == 104
    assert stock.hand(b'{}', []) == 102


def _legacy_client(version):
    from kiosk_autoscaler_amd.fakes import FakeRedis, RedisEngine
    return FakeRedis(engine=RedisEngine(version=version))


@pytest.mark.parametrize('version,block_mode', [
    ('7.2.0', 'blmove'), ('6.0.16', 'brpoplpush'), ('5.0.14', 'poll')])
def test_consumer_adapts_to_the_server_version(version, block_mode):
    """against Redis < 6.2 (no LMOVE/BLMOVE) the
    consumer switches once to RPOPLPUSH/BRPOPLPUSH, and below 6.0 (integer
    blocking timeouts) to a non-blocking poll.  FIFO order and the
    processing-key convention are unchanged."""
    client = _legacy_client(version)
    consumer = rt.QueueConsumer(client, 'w-g0-x-4', ['predict'],
                                poll_block=0.005)
    assert consumer.pull(limit=1) == []          # empty: the blocking path
    assert consumer.block_mode == block_mode
    for i in range(3):
        client.lpush('predict', 'predict:%d' % i)
    got = []
    for _ in range(3):
        (queue, item, pkey), = consumer.pull(limit=1)
        assert pkey == 'processing-predict:w-g0-x-4'
        assert client.lrange(pkey, 0, -1) == [item]
        consumer.complete(pkey)
        got.append(item)
    assert got == ['predict:0', 'predict:1', 'predict:2']
    assert consumer.move_mode == ('lmove' if version >= '6.2' else
                                  'rpoplpush')
    # a key that lands while the consumer waits is taken by the wait itself
    client.lpush('predict', 'predict:late')
    assert consumer.pull(limit=1, block=True)[0][1] == 'predict:late'


def test_pull_error_does_not_crash_the_worker(redis_client, monkeypatch):
    """A protocol error the consumer cannot adapt to is reported and
    retried; the worker keeps running until it is drained."""
    import queue
    channel = _Channel()
    channel.commands = queue.Queue()
    channel.start_reader = lambda: None
    env = {'ROWS_PER_KEY': '8', 'MOCK_WORK_MS': '0', 'QUEUES': 'predict'}
    cfg = rt.WorkerConfig(env, {'worker_id': 'w-g0-x-5'})
    run = rt.WorkerRuntime(cfg, lambda c, stage: mlp.CpuMlpEngine(c),
                           channel, lambda: redis_client)
    calls = []

    def broken(self, limit=1, block=True):
        calls.append(1)
        if len(calls) == 2:
            channel.commands.put({'cmd': 'drain'})
        raise rt.redis_errors.ResponseError('ERR something odd')
    monkeypatch.setattr(rt.QueueConsumer, 'pull', broken)
    monkeypatch.setattr(rt.time, 'sleep', lambda s: None)
    assert run.run() == 0
    assert len(calls) == 2
    assert [e for e, _ in channel.events].count('pull_error') == 2


def test_channel_cap_is_decided_without_importing_the_plugin(monkeypatch,
                                                              tmp_path):
    """deciding the RCCL channel cap must not import a user
    plug-in (its module-level imports would run before the GPU pin)."""
    import sys
    from kiosk_autoscaler_amd.worker import main as worker_main
    mod = tmp_path / 'sideeffect_plugin.py'
    mod.write_text('import os\nos.environ["PLUGIN_IMPORTED"] = "1"\n'
                   'def factory(cfg, stage=None):\n    return None\n')
    monkeypatch.syspath_prepend(str(tmp_path))
    monkeypatch.delenv('PLUGIN_IMPORTED', raising=False)
    monkeypatch.setenv('WORKER_ENGINE', 'sideeffect_plugin:factory')
    assert worker_main._engine_collectives() is True
    assert 'PLUGIN_IMPORTED' not in os.environ
    assert 'sideeffect_plugin' not in sys.modules
    monkeypatch.setenv('WORKER_ENGINE', 'kiosk_autoscaler_amd.models.'
                       'torch_kiosk:TorchKioskEngine')
    assert worker_main._engine_collectives() is False
    monkeypatch.delenv('WORKER_ENGINE')
    assert worker_main._engine_collectives() is False


def test_recycled_worker_retired_at_once_skips_the_collection(monkeypatch):
    """A recycled worker runs ``gc.collect`` only once no command came
    within ``COLLECT_AFTER_S``: one the manager retires on that pass exits
    without it (a PyTorch process's full collection is standby GPU time)."""
    from kiosk_autoscaler_amd.worker import main as wmain
    from kiosk_autoscaler_amd.worker.channel import TIMEOUT
    collected = []
    monkeypatch.setattr(wmain.gc, 'collect', lambda: collected.append(1))

    class FakeChannel(object):
        def __init__(self, replies):
            self.replies = list(replies)
            self.timeouts = []
            self.emitted = []
            self.device_reported = False

        def emit(self, ev, **fields):
            self.emitted.append(ev)

        def read_command(self, timeout=None):
            self.timeouts.append(timeout)
            return self.replies.pop(0)

    exit_now = FakeChannel([{'cmd': 'exit'}])
    assert wmain._wait_for_assignment(exit_now, None, 0, 'cpu', {},
                                      collect=True) is None
    assert collected == [] and exit_now.emitted == ['standby']
    assert exit_now.timeouts == [wmain.COLLECT_AFTER_S]
    # kept as a standby: collected once, then it blocks as before
    kept = FakeChannel([TIMEOUT, {'cmd': 'assign', 'gpu': None}])
    assert wmain._wait_for_assignment(kept, None, 0, 'cpu', {},
                                      collect=True)['cmd'] == 'assign'
    assert collected == [1]
    assert kept.timeouts == [wmain.COLLECT_AFTER_S, None]
