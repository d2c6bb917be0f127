"""PyTorch-tensor front end of the native ops (device memory and streams come from torch; the
work is done by libb200ops.so on the current CUDA stream).

`reference(task, inp)` mirrors the reference's per-task `reference(inp) -> dict`
(tasks/<task>/reference.py): the same input dict keys (the C argument names), the same output
names and shapes, so a caller of the reference's PyTorch entry can switch to this one unchanged.
Every function raises on a non-CUDA tensor, a wrong dtype or a non-contiguous input, and on a
non-zero native status; there is no CPU fallback.
"""
import ctypes
import functools
import threading

import torch
from torch.autograd.function import once_differentiable

from . import _native

_WS = {}


def _lib():
    return _native.load()


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _opt_ptr(t, stand_in):
    """Pointer of an optional input stream: NULL when absent.  torch gives an empty tensor a NULL
    data pointer, which the C ABI would read as "absent"; a present but empty stream passes a
    valid stand-in address instead (never dereferenced: there are no elements)."""
    if t is None:
        return ctypes.c_void_p(0)
    return ctypes.c_void_p(t.data_ptr() or stand_in.data_ptr())


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _need(t, name, dtype, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")
    return t


def workspace(op, nbytes, device):
    """Zero-initialised scratch for `op` on `device` and the current stream, grown on demand.

    The reduction kernels leave their control words ready for the next call, so one buffer serves
    every later call issued on the same stream (never two streams at once)."""
    key = (op, device.index, torch.cuda.current_stream(device).cuda_stream)
    buf = _WS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(int(nbytes), 4096), dtype=torch.uint8, device=device)
        _WS[key] = buf
    return buf


# ----------------------------------------------------------------------------------- robust-L1
def robust_l1(inp, target, out=None):
    """mean(sqrt((inp - target)^2 + 1e-6)) as a 0-d fp32 tensor."""
    _need(inp, "inp", torch.float32)
    _need(target, "target", torch.float32, inp.device)
    if inp.numel() != target.numel():
        raise ValueError("inp and target differ in size")
    n = inp.numel()
    out = torch.empty((), dtype=torch.float32, device=inp.device) if out is None else out
    lib = _lib()
    ws = workspace("robust_l1", lib.b200_robust_l1_workspace_bytes(n), inp.device)
    _native.check(lib.b200_robust_l1_async(_ptr(inp), _ptr(target), n, _ptr(out), _ptr(ws), ws.numel(),
                                           _stream(inp.device)), "robust_l1")
    return out


def robust_l1_partials(inp, target):
    """Chunk partials (fp64, one per b200_robust_l1_chunk_elems() elements) of one shard."""
    _need(inp, "inp", torch.float32)
    _need(target, "target", torch.float32, inp.device)
    lib = _lib()
    n = inp.numel()
    chunk = lib.b200_robust_l1_chunk_elems()
    parts = torch.empty((n + chunk - 1) // chunk, dtype=torch.float64, device=inp.device)
    _native.check(lib.b200_robust_l1_shard_partials(_ptr(inp), _ptr(target), n, _ptr(parts),
                                                    _stream(inp.device)), "robust_l1_partials")
    return parts


def robust_l1_finish(partials, n_total, out=None):
    _need(partials, "partials", torch.float64)
    out = torch.empty((), dtype=torch.float32, device=partials.device) if out is None else out
    _native.check(_lib().b200_robust_l1_finish(_ptr(partials), partials.numel(), int(n_total), _ptr(out),
                                               _stream(partials.device)), "robust_l1_finish")
    return out


# ----------------------------------------------------------------------------------------- PPO
def ppo_clip(cur, old, adv, clip_epsilon, entropy=None, out=None):
    """[loss, clip_fraction, approx_kl, ess, max_ratio, mean_ratio] (+ mean entropy)."""
    _need(cur, "current_log_prob", torch.float32)
    _need(old, "old_log_prob", torch.float32, cur.device)
    _need(adv, "advantage", torch.float32, cur.device)
    if entropy is not None:
        _need(entropy, "entropy", torch.float32, cur.device)
    n = cur.numel()
    if old.numel() != n or adv.numel() != n or (entropy is not None and entropy.numel() != n):
        raise ValueError("PPO inputs differ in size")
    k = 7 if entropy is not None else 6
    out = torch.empty(k, dtype=torch.float32, device=cur.device) if out is None else out
    lib = _lib()
    ws = workspace("ppo", lib.b200_ppo_workspace_bytes(n), cur.device)
    _native.check(lib.b200_ppo_async(_ptr(cur), _ptr(old), _ptr(adv), _opt_ptr(entropy, out), n,
                                     float(clip_epsilon), _ptr(out), _ptr(ws), ws.numel(), _stream(cur.device)),
                  "ppo_clip")
    return out


def ppo_partials(cur, old, adv, clip_epsilon, entropy=None):
    """Per-chunk partial records (uint8 rows of b200_ppo_partial_bytes()) of one shard."""
    lib = _lib()
    n = cur.numel()
    chunk = lib.b200_ppo_chunk_elems()
    rec = lib.b200_ppo_partial_bytes()
    parts = torch.empty(((n + chunk - 1) // chunk, rec), dtype=torch.uint8, device=cur.device)
    _native.check(lib.b200_ppo_shard_partials(_ptr(cur), _ptr(old), _ptr(adv), _opt_ptr(entropy, parts), n,
                                              float(clip_epsilon), _ptr(parts), _stream(cur.device)),
                  "ppo_partials")
    return parts


def ppo_finish(partials, n_total, with_entropy, out=None):
    k = 7 if with_entropy else 6
    out = torch.empty(k, dtype=torch.float32, device=partials.device) if out is None else out
    _native.check(_lib().b200_ppo_finish(_ptr(partials), partials.shape[0], int(n_total), int(bool(with_entropy)),
                                         _ptr(out), _stream(partials.device)), "ppo_finish")
    return out


# -------------------------------------------------------------------------------- reward-to-go
def reward_to_go(reward, done, gamma, out=None):
    _need(reward, "reward", torch.float32)
    _need(done, "done", torch.bool, reward.device)
    if reward.dim() != 2 or done.shape != reward.shape:
        raise ValueError("reward and done must both be (B, T)")
    B, T = reward.shape
    out = torch.empty_like(reward) if out is None else out
    _native.check(_lib().b200_reward_to_go_async(_ptr(reward), _ptr(done), float(gamma), B, T, _ptr(out),
                                                 _stream(reward.device)), "reward_to_go")
    return out


def pack_done(done, out=None):
    """Done flags bool [B, T] -> bits int32 [B, ceil(T/32)]: bit t % 32 of word [b, t // 32] is
    done[b, t], bits past T zero."""
    _need(done, "done", torch.bool)
    if done.dim() != 2:
        raise ValueError("done must be (B, T)")
    B, T = done.shape
    out = torch.empty((B, (T + 31) // 32), dtype=torch.int32, device=done.device) if out is None else out
    _native.check(_lib().b200_pack_done_async(_ptr(done), B, T, _ptr(out), _stream(done.device)), "pack_done")
    return out


def reward_to_go_bits(reward, done_bits, gamma, out=None):
    """reward_to_go with the done flags as bits (pack_done): the same output bits."""
    _need(reward, "reward", torch.float32)
    if reward.dim() != 2:
        raise ValueError("reward must be (B, T)")
    B, T = reward.shape
    _need(done_bits, "done_bits", torch.int32, reward.device)
    if done_bits.shape != (B, (T + 31) // 32):
        raise ValueError("done_bits must be (B, ceil(T/32))")
    out = torch.empty_like(reward) if out is None else out
    _native.check(_lib().b200_reward_to_go_bits_async(_ptr(reward), _ptr(done_bits), float(gamma), B, T, _ptr(out),
                                                      _stream(reward.device)), "reward_to_go_bits")
    return out


def _done_layout(reward, done):
    """(is_bits, T) for a done tensor: bool [B, T] or int32 bits [B, ceil(T/32)]."""
    B, T = reward.shape
    if done.dtype == torch.int32:
        _need(done, "done_bits", torch.int32, reward.device)
        if done.shape != (B, (T + 31) // 32):
            raise ValueError("done bits must be (B, ceil(T/32))")
        return 1
    _need(done, "done", torch.bool, reward.device)
    if done.shape != reward.shape:
        raise ValueError("reward and done must both be (B, T)")
    return 0


def reward_to_go_chunked(reward, done, gamma, out=None):
    """reward_to_go parallel along T (for few, long rows); done: bool [B, T] or pack_done bits."""
    _need(reward, "reward", torch.float32)
    if reward.dim() != 2:
        raise ValueError("reward must be (B, T)")
    bits = _done_layout(reward, done)
    B, T = reward.shape
    out = torch.empty_like(reward) if out is None else out
    lib = _lib()
    ws = workspace("rtg_chunked", lib.b200_reward_to_go_chunked_workspace_bytes(B, T), reward.device)
    _native.check(lib.b200_reward_to_go_chunked_async(_ptr(reward), _ptr(done), bits, float(gamma), B, T, _ptr(out),
                                                      _ptr(ws), ws.numel(), _stream(reward.device)),
                  "reward_to_go_chunked")
    return out


def reward_to_go_slice_maps(reward, done, gamma, maps_out=None):
    """First half of reward-to-go sharded over time: this rank's [B, 2] fp64 slice maps (a, b)."""
    _need(reward, "reward", torch.float32)
    bits = _done_layout(reward, done)
    B, T = reward.shape
    maps_out = torch.empty((B, 2), dtype=torch.float64, device=reward.device) if maps_out is None else maps_out
    lib = _lib()
    ws = workspace("rtg_slice", lib.b200_reward_to_go_chunked_workspace_bytes(B, T), reward.device)
    _native.check(lib.b200_reward_to_go_slice_maps_async(_ptr(reward), _ptr(done), bits, float(gamma), B, T,
                                                         _ptr(maps_out), _ptr(ws), ws.numel(),
                                                         _stream(reward.device)), "reward_to_go_slice_maps")
    return maps_out


def reward_to_go_slice_scan(reward, done, gamma, all_maps, rank, out=None):
    """Second half: this rank's outputs from every rank's slice maps all_maps [world, B, 2] (rank
    order).  Uses the workspace reward_to_go_slice_maps filled on this stream."""
    _need(reward, "reward", torch.float32)
    bits = _done_layout(reward, done)
    B, T = reward.shape
    _need(all_maps, "all_maps", torch.float64, reward.device)
    world = all_maps.shape[0]
    if all_maps.shape != (world, B, 2):
        raise ValueError("all_maps must be (world, B, 2)")
    out = torch.empty_like(reward) if out is None else out
    lib = _lib()
    ws = workspace("rtg_slice", lib.b200_reward_to_go_chunked_workspace_bytes(B, T), reward.device)
    _native.check(lib.b200_reward_to_go_slice_scan_async(_ptr(reward), _ptr(done), bits, float(gamma), B, T,
                                                         _ptr(all_maps), int(world), int(rank), _ptr(out), _ptr(ws),
                                                         ws.numel(), _stream(reward.device)),
                  "reward_to_go_slice_scan")
    return out


def reward_to_go_time_sharded(reward, done, gamma, group=None, out=None):
    """reward_to_go over rows whose steps are sharded across the ranks of `group` in rank order
    (this rank holds steps [offset, offset + T_local) of every row): slice maps, one all-gather of
    16 bytes per row per rank, then this rank's outputs."""
    import torch.distributed as dist
    maps = reward_to_go_slice_maps(reward, done, gamma)
    world = dist.get_world_size(group)
    all_maps = torch.empty((world * maps.shape[0], 2), dtype=maps.dtype, device=maps.device)  # rank-major
    dist.all_gather_into_tensor(all_maps, maps, group=group)
    return reward_to_go_slice_scan(reward, done, gamma, all_maps.view(world, -1, 2), dist.get_rank(group), out=out)


# ---------------------------------------------------------------------------- fused RL loss step
STEP_INPUTS_READY = 1  # B200_STEP_INPUTS_READY
STEP_DONE_BITS = 2     # B200_STEP_DONE_BITS


def _step_done_flags(reward, done, dev):
    """The step's done argument: bool [B, T], or bits int32 [B, ceil(T/32)] (flag STEP_DONE_BITS)."""
    if reward.dim() != 2:
        raise ValueError("reward must be (B, T)")
    B, T = reward.shape
    if isinstance(done, torch.Tensor) and done.dtype == torch.int32:
        _need(done, "done", torch.int32, dev)
        if done.shape != (B, (T + 31) // 32):
            raise ValueError("done bits must be (B, ceil(T/32))")
        return STEP_DONE_BITS
    _need(done, "done", torch.bool, dev)
    if done.shape != reward.shape:
        raise ValueError("reward and done must both be (B, T)")
    return 0


def rl_step(reward, done, gamma, cur, old, adv, clip_epsilon, entropy=None, rtg_out=None, ppo_out=None,
            inputs_ready=False):
    """reward_to_go and ppo_clip on independent inputs in one launch; the same bits as the two
    separate calls.  Returns (returns [B, T], PPO outputs [6] or [7]).

    inputs_ready=True declares that the kernel launched just before on the stream writes none of
    the inputs, so the step reads them while that kernel finishes (programmatic dependent launch).
    done: bool [B, T], or the flags as bits (pack_done)."""
    _need(reward, "reward", torch.float32)
    dev = reward.device
    flags = _step_done_flags(reward, done, dev)
    for t, nm in ((cur, "current_log_prob"), (old, "old_log_prob"), (adv, "advantage")):
        _need(t, nm, torch.float32, dev)
    if entropy is not None:
        _need(entropy, "entropy", torch.float32, dev)
    n = cur.numel()
    if old.numel() != n or adv.numel() != n or (entropy is not None and entropy.numel() != n):
        raise ValueError("PPO inputs differ in size")
    B, T = reward.shape
    rtg_out = torch.empty_like(reward) if rtg_out is None else rtg_out
    k = 7 if entropy is not None else 6
    ppo_out = torch.empty(k, dtype=torch.float32, device=dev) if ppo_out is None else ppo_out
    lib = _lib()
    ws = workspace("ppo", lib.b200_ppo_workspace_bytes(n), dev)
    _native.check(lib.b200_rl_step_ex_async(_ptr(reward), _ptr(done), float(gamma), B, T, _ptr(rtg_out), _ptr(cur),
                                            _ptr(old), _ptr(adv), _opt_ptr(entropy, ppo_out), n, float(clip_epsilon),
                                            _ptr(ppo_out), _ptr(ws), ws.numel(),
                                            flags | (STEP_INPUTS_READY if inputs_ready else 0), _stream(dev)),
                  "rl_step")
    return rtg_out, ppo_out


def rl_step_shard(reward, done, gamma, cur, old, adv, clip_epsilon, entropy=None, rtg_out=None, partials_out=None):
    """The fused step of one shard: returns and the PPO per-chunk partial records (as
    ppo_partials), for a cross-GPU gather and ppo_finish."""
    _need(reward, "reward", torch.float32)
    dev = reward.device
    _need(done, "done", torch.bool, dev)
    if reward.dim() != 2 or done.shape != reward.shape:
        raise ValueError("reward and done must both be (B, T)")
    for t, nm in ((cur, "current_log_prob"), (old, "old_log_prob"), (adv, "advantage")):
        _need(t, nm, torch.float32, dev)
    if entropy is not None:
        _need(entropy, "entropy", torch.float32, dev)
    n = cur.numel()
    if old.numel() != n or adv.numel() != n or (entropy is not None and entropy.numel() != n):
        raise ValueError("PPO inputs differ in size")
    lib = _lib()
    chunk = lib.b200_ppo_chunk_elems()
    shape = ((n + chunk - 1) // chunk, lib.b200_ppo_partial_bytes())
    if partials_out is None:
        partials_out = torch.empty(shape, dtype=torch.uint8, device=dev)
    elif tuple(partials_out.shape) != shape or partials_out.dtype != torch.uint8:
        raise ValueError(f"partials_out must be uint8 {shape}")
    B, T = reward.shape
    rtg_out = torch.empty_like(reward) if rtg_out is None else rtg_out
    _native.check(lib.b200_rl_step_shard_async(_ptr(reward), _ptr(done), float(gamma), B, T, _ptr(rtg_out),
                                               _ptr(cur), _ptr(old), _ptr(adv), _opt_ptr(entropy, rtg_out), n,
                                               float(clip_epsilon), _ptr(partials_out), _stream(dev)),
                  "rl_step_shard")
    return rtg_out, partials_out


# ------------------------------------------------------- multi-GPU RL step over NVLink peer memory
class PeerExchange:
    """The per-rank exchange buffer of the fused multi-GPU RL step (one process per GPU).

    `swap(handle) -> list of handles` must return every rank's 64-byte handle in rank order; with
    torch.distributed initialised, the default does that with all_gather_object."""

    def __init__(self, world, rank, n, swap=None, slots=None, record_bytes=None):
        """An exchange for the RL step over n samples per rank (the default), or, with `slots` and
        `record_bytes`, for another op's records (e.g. RobustL1Exchange)."""
        lib = _lib()
        self._ptr = ctypes.c_void_p()
        handle = (ctypes.c_char * lib.b200_peer_handle_bytes())()
        slots = 1 if slots is None else int(slots)
        rec = lib.b200_rl_step_exchange_record_bytes() if record_bytes is None else int(record_bytes)
        _native.check(lib.b200_peer_exchange_create(int(world), int(rank), slots, rec, ctypes.byref(self._ptr),
                                                    handle), "peer_exchange_create")
        if swap is None:
            import torch.distributed as dist

            def swap(h):
                out = [None] * world
                dist.all_gather_object(out, h)
                return out
        handles = swap(bytes(handle))
        if len(handles) != world:
            raise ValueError("swap() must return one handle per rank")
        blob = b"".join(handles)
        _native.check(lib.b200_peer_exchange_open(self._ptr, blob), "peer_exchange_open")
        self.world, self.rank, self.n, self.epoch = world, rank, int(n), 0

    @property
    def handle(self):
        return self._ptr

    def close(self):
        if self._ptr:
            _native.check(_lib().b200_peer_exchange_destroy(self._ptr), "peer_exchange_destroy")
            self._ptr = ctypes.c_void_p()


class RobustL1Exchange(PeerExchange):
    """The NVLink exchange of the multi-GPU robust-L1 mean over n_total elements (one process per
    GPU; every rank builds one with the same n_total, collectively)."""

    def __init__(self, world, rank, n_total, swap=None):
        lib = _lib()
        super().__init__(world, rank, n_total, swap=swap, slots=lib.b200_robust_l1_exchange_slots(int(n_total), world),
                         record_bytes=lib.b200_robust_l1_exchange_record_bytes())

    def shard_range(self):
        """[lo, hi) global element range this rank holds (whole chunks, as dist.shard_range)."""
        lib = _lib()
        chunk = lib.b200_robust_l1_chunk_elems()
        n_chunks = (self.n + chunk - 1) // chunk
        c0, c1 = (n_chunks * self.rank) // self.world, (n_chunks * (self.rank + 1)) // self.world
        return min(c0 * chunk, self.n), min(c1 * chunk, self.n)


def robust_l1_exchange(exchange, inp_shard, tgt_shard, out=None):
    """The robust-L1 mean over every rank's elements, from this rank's shard (its
    exchange.shard_range() elements); every rank gets the same bits, those of robust_l1 over the
    whole range on one GPU.  Every rank must call it the same number of times."""
    _need(inp_shard, "inp", torch.float32)
    _need(tgt_shard, "target", torch.float32, inp_shard.device)
    lo, hi = exchange.shard_range()
    if inp_shard.numel() != hi - lo or tgt_shard.numel() != hi - lo:
        raise ValueError(f"this rank holds elements [{lo}, {hi}); got {inp_shard.numel()}")
    dev = inp_shard.device
    out = torch.empty((), dtype=torch.float32, device=dev) if out is None else out
    lib = _lib()
    ws = workspace("robust_l1_exchange", 256, dev)
    exchange.epoch = lib.b200_peer_next_epoch(exchange.epoch)
    _native.check(lib.b200_robust_l1_exchange_async(_opt_ptr(inp_shard, out), _opt_ptr(tgt_shard, out), exchange.n,
                                                    _ptr(out), _ptr(ws), ws.numel(), exchange.handle, exchange.epoch,
                                                    _stream(dev)), "robust_l1_exchange")
    return out


def rl_step_exchange(exchange, reward, done, gamma, cur, old, adv, clip_epsilon, entropy=None, rtg_out=None,
                     ppo_out=None, inputs_ready=False):
    """One rank's fused multi-GPU RL step: this rank's returns, and the PPO outputs over every
    rank's samples (the same bits on every rank).  Every rank must call it the same number of
    times.  inputs_ready and done as for rl_step."""
    _need(reward, "reward", torch.float32)
    dev = reward.device
    flags = _step_done_flags(reward, done, dev)
    for t, nm in ((cur, "current_log_prob"), (old, "old_log_prob"), (adv, "advantage")):
        _need(t, nm, torch.float32, dev)
    if entropy is not None:
        _need(entropy, "entropy", torch.float32, dev)
    n = cur.numel()
    if n != exchange.n:
        raise ValueError("the exchange was created for a different sample count")
    B, T = reward.shape
    rtg_out = torch.empty_like(reward) if rtg_out is None else rtg_out
    k = 7 if entropy is not None else 6
    ppo_out = torch.empty(k, dtype=torch.float32, device=dev) if ppo_out is None else ppo_out
    lib = _lib()
    ws = workspace("ppo", lib.b200_ppo_workspace_bytes(n), dev)
    exchange.epoch = lib.b200_peer_next_epoch(exchange.epoch)
    _native.check(lib.b200_rl_step_exchange_async(_ptr(reward), _ptr(done), float(gamma), B, T, _ptr(rtg_out),
                                                  _ptr(cur), _ptr(old), _ptr(adv), _opt_ptr(entropy, ppo_out), n,
                                                  float(clip_epsilon), _ptr(ppo_out), _ptr(ws), ws.numel(),
                                                  exchange.handle, exchange.epoch,
                                                  flags | (STEP_INPUTS_READY if inputs_ready else 0), _stream(dev)),
                  "rl_step_exchange")
    return rtg_out, ppo_out


# ----------------------------------------------------------------------------------------- GAE
def gae(reward, value, next_value, done, terminated, gamma, lmbda, advantage=None, value_target=None):
    """Generalised advantage estimation over [B, T] rows: returns (advantage, value_target)."""
    _need(reward, "reward", torch.float32)
    dev = reward.device
    for t, nm in ((value, "value"), (next_value, "next_value")):
        _need(t, nm, torch.float32, dev)
    for t, nm in ((done, "done"), (terminated, "terminated")):
        _need(t, nm, torch.bool, dev)
    if reward.dim() != 2 or any(t.shape != reward.shape for t in (value, next_value, done, terminated)):
        raise ValueError("gae: all inputs must be (B, T)")
    B, T = reward.shape
    advantage = torch.empty_like(reward) if advantage is None else advantage
    value_target = torch.empty_like(reward) if value_target is None else value_target
    _native.check(_lib().b200_gae_async(_ptr(reward), _ptr(value), _ptr(next_value), _ptr(done), _ptr(terminated),
                                        float(gamma), float(lmbda), B, T, _ptr(advantage), _ptr(value_target),
                                        _stream(dev)), "gae")
    return advantage, value_target


# ----------------------------------------------------------------------------------------- LIF
def leaky_packed(input_current, mem0, beta, threshold, spike_bits=None, final_mem=None):
    """The LIF layer with bit-packed spikes: returns (spike_bits int32 [ceil(T/32), B, H], bit t % 32
    of word [t // 32] being the spike at step t; final_mem [B, H])."""
    _need(input_current, "input_current", torch.float32)
    dev = input_current.device
    for t, nm in ((mem0, "mem0"), (beta, "beta"), (threshold, "threshold")):
        _need(t, nm, torch.float32, dev)
    T, B, H = input_current.shape
    if spike_bits is None:
        spike_bits = torch.empty(((T + 31) // 32, B, H), dtype=torch.int32, device=dev)
    final_mem = torch.empty((B, H), dtype=torch.float32, device=dev) if final_mem is None else final_mem
    _native.check(_lib().b200_leaky_packed_async(_ptr(input_current), _ptr(mem0), _ptr(beta), _ptr(threshold), T, B,
                                                 H, _ptr(spike_bits), _ptr(final_mem), _stream(dev)), "leaky_packed")
    return spike_bits, final_mem


def leaky(input_current, mem0, beta, threshold, spikes=None, final_mem=None):
    _need(input_current, "input_current", torch.float32)
    dev = input_current.device
    for t, nm in ((mem0, "mem0"), (beta, "beta"), (threshold, "threshold")):
        _need(t, nm, torch.float32, dev)
    T, B, H = input_current.shape
    spikes = torch.empty_like(input_current) if spikes is None else spikes
    final_mem = torch.empty((B, H), dtype=torch.float32, device=dev) if final_mem is None else final_mem
    _native.check(_lib().b200_leaky_async(_ptr(input_current), _ptr(mem0), _ptr(beta), _ptr(threshold), T, B, H,
                                          _ptr(spikes), _ptr(final_mem), _stream(dev)), "leaky")
    return spikes, final_mem


def _leaky_args(input_current, mem0, beta, threshold):
    _need(input_current, "input_current", torch.float32)
    dev = input_current.device
    for t, nm in ((mem0, "mem0"), (beta, "beta"), (threshold, "threshold")):
        _need(t, nm, torch.float32, dev)
    T, B, H = input_current.shape
    return dev, T, B, H


def _checkpoint_buffer(T, B, H, dev):
    return torch.empty(((T + 15) // 16, B, H), dtype=torch.float32, device=dev)


def leaky_train(input_current, mem0, beta, threshold):
    """The LIF forward for training: (spikes, final_mem, checkpoints), spikes and final_mem as leaky();
    checkpoints [ceil(T/16), B, H] are the membrane state before every 16th step, what
    leaky_backward recomputes the trajectory from."""
    dev, T, B, H = _leaky_args(input_current, mem0, beta, threshold)
    spikes = torch.empty_like(input_current)
    final_mem = torch.empty((B, H), dtype=torch.float32, device=dev)
    ckpt = _checkpoint_buffer(T, B, H, dev)
    _native.check(_lib().b200_leaky_train_async(_ptr(input_current), _ptr(mem0), _ptr(beta), _ptr(threshold), T, B,
                                                H, _ptr(spikes), _ptr(final_mem), _ptr(ckpt), _stream(dev)),
                  "leaky_train")
    return spikes, final_mem, ckpt


def leaky_checkpoints(input_current, mem0, beta, threshold):
    """The membrane checkpoints alone, for a forward that ran through leaky()."""
    dev, T, B, H = _leaky_args(input_current, mem0, beta, threshold)
    ckpt = _checkpoint_buffer(T, B, H, dev)
    _native.check(_lib().b200_leaky_checkpoints_async(_ptr(input_current), _ptr(mem0), _ptr(beta), _ptr(threshold),
                                                      T, B, H, _ptr(ckpt), _stream(dev)), "leaky_checkpoints")
    return ckpt


def leaky_backward(input_current, checkpoints, beta, threshold, grad_spikes, grad_final_mem=None, alpha=2.0,
                   need_params=True):
    """Surrogate-gradient backward (arctangent surrogate, reset detached): returns (grad_input,
    grad_mem0, grad_beta, grad_threshold); the last two are None unless need_params."""
    _need(input_current, "input_current", torch.float32)
    dev = input_current.device
    T, B, H = input_current.shape
    for t, nm in ((checkpoints, "checkpoints"), (beta, "beta"), (threshold, "threshold"),
                  (grad_spikes, "grad_spikes")):
        _need(t, nm, torch.float32, dev)
    if grad_final_mem is not None:
        _need(grad_final_mem, "grad_final_mem", torch.float32, dev)
    if checkpoints.numel() != ((T + 15) // 16) * B * H or grad_spikes.shape != input_current.shape:
        raise ValueError("leaky_backward: inconsistent shapes")
    lib = _lib()
    gx = torch.empty_like(input_current)
    gm = torch.empty((B, H), dtype=torch.float32, device=dev)
    gb = torch.empty(H, dtype=torch.float32, device=dev) if need_params else None
    gt = torch.empty(H, dtype=torch.float32, device=dev) if need_params else None
    ws = workspace("leaky_backward", lib.b200_leaky_backward_workspace_bytes(B, H), dev) if need_params else None
    _native.check(lib.b200_leaky_backward_async(_ptr(input_current), _ptr(checkpoints), _ptr(beta), _ptr(threshold),
                                                T, B, H, _ptr(grad_spikes),
                                                None if grad_final_mem is None else _ptr(grad_final_mem),
                                                float(alpha), _ptr(gx), _ptr(gm), _ptr(gb), _ptr(gt),
                                                None if ws is None else _ptr(ws), 0 if ws is None else ws.numel(),
                                                _stream(dev)), "leaky_backward")
    return gx, gm, gb, gt


class LeakyFunction(torch.autograd.Function):
    """torch.autograd form of the layer: forward through leaky_train (keeps the 1/4-byte-per-step
    checkpoints, not the trajectory), backward through leaky_backward."""

    @staticmethod
    def forward(ctx, input_current, mem0, beta, threshold, alpha=2.0):
        spikes, final_mem, ckpt = leaky_train(input_current, mem0, beta, threshold)
        ctx.save_for_backward(input_current, ckpt, beta, threshold)
        ctx.alpha = float(alpha)
        return spikes, final_mem

    @staticmethod
    def backward(ctx, grad_spikes, grad_final_mem):
        x, ckpt, beta, threshold = ctx.saved_tensors
        if grad_spikes is None:
            grad_spikes = torch.zeros_like(x)
        gs = grad_spikes.contiguous()
        gf = None if grad_final_mem is None else grad_final_mem.contiguous()
        need = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        gx, gm, gb, gt = leaky_backward(x, ckpt, beta, threshold, gs, gf, ctx.alpha, need_params=need)
        return gx, gm, gb, gt, None


# --------------------------------------------------------------- gated linear recurrence
DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # B200_F32, B200_BF16, B200_F16
RECURRENCE_FORMS = {"decay": 0, "sigmoid": 1}
_I32_MAX = 2**31 - 1


_current_device = torch.cuda.current_device
# The handle of a device's current stream, without a Stream object around it where torch offers that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


@functools.lru_cache(maxsize=1024)
def _strides(*values):
    """A host array of element strides for the C ABI, which only reads it."""
    return (ctypes.c_int64 * len(values))(*values)


def _needs(ctx, k):
    """Whether apply()'s argument k (which may have been left out) requires a gradient."""
    return k < len(ctx.needs_input_grad) and ctx.needs_input_grad[k]


# A call may be more than one launch over the scratch of its stream, so threads take turns.
_LAUNCH = threading.Lock()


def _run(what, fn, index, *args):
    """A stream form on the current stream of device `index`, which is made the current device for it (a
    launch goes to the current device)."""
    with _LAUNCH:
        if _current_device() == index:
            status = fn(*args, _raw_stream(index))
        else:
            with torch.cuda.device(index):
                status = fn(*args, _raw_stream(index))
    if status:
        _native.check(status, what)


def _call(name, *args):
    """An operator's outputs by the short way (csrc/python/calls.cpp), which takes its ordinary calls; None where the
    call has to go the long way, through the checks below and ctypes."""
    calls = _native.calls()
    if calls is None:
        return None
    with _LAUNCH:
        return getattr(calls, name)(*args)


def _address(t):
    return None if t is None else t.data_ptr()


def _scratch(op, nbytes, device):
    """workspace(), except that a call being captured into a CUDA graph gets scratch of its own (its
    zero-fill is captured with it): graphs may be replayed at the same time as one another and as
    calls outside them."""
    index = device.index
    if _current_device() == index:
        capturing = torch.cuda.is_current_stream_capturing()
    else:
        with torch.cuda.device(index):
            capturing = torch.cuda.is_current_stream_capturing()
    if capturing:
        return torch.zeros(max(int(nbytes), 16), dtype=torch.uint8, device=device)
    buf = _WS.get((op, index, _raw_stream(index)))
    return buf if buf is not None and buf.numel() >= nbytes else workspace(op, nbytes, device)


def _float_tensor(t, name, device=None, dtype=None, dims=None):
    """A CUDA tensor of a model (fp32, bf16 or fp16, or `dtype`) whose last axis is contiguous."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor (no CPU path)")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")
    if dtype is None:
        if t.dtype not in DTYPE_CODES:
            raise ValueError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    elif t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got {t.dim()}")
    if t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel():
        raise ValueError(f"{name}: expected a contiguous last dimension")
    if t.numel() > _I32_MAX and any(n > _I32_MAX for n in t.shape):
        raise ValueError(f"{name}: a dimension is larger than 2^31 - 1")
    return t


def _bth(gate, x, form):
    """Checks gate and x [B, T, H] of a recurrence: (device, dtype code, form code, shape)."""
    if form not in RECURRENCE_FORMS:
        raise ValueError(f"form must be one of {sorted(RECURRENCE_FORMS)}, got {form!r}")
    _float_tensor(x, "x", dims=3)
    device, shape = x.device, x.shape
    _float_tensor(gate, "gate", device, x.dtype, 3)
    if gate.shape != shape:
        raise ValueError("gate and x must have the same shape (B, T, H)")
    return device, DTYPE_CODES[x.dtype], RECURRENCE_FORMS[form], shape


def _dense_like(t):
    """A contiguous output of t's shape and dtype."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _like_bth(x):
    """An output of x's shape and dtype: dense, time first in memory when x is."""
    B, T, H = x.shape
    if B > 1 and T > 1 and x.stride(0) < x.stride(1):
        return x.new_empty((T, B, H)).transpose(0, 1)
    return _dense_like(x)


def _writable(t, like, name):
    """A caller's output for `like`'s shape: own memory per element."""
    _float_tensor(t, name, like.device, like.dtype, like.dim())
    if t.shape != like.shape:
        raise ValueError(f"{name}: expected shape {tuple(like.shape)}, got {tuple(t.shape)}")
    if t.numel():
        dims = sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1)
        reach = 1
        for s, n in dims:
            if s < reach:
                raise ValueError(f"{name}: elements share memory")
            reach = s * (n - 1) + reach
    return t


def _reach(t):
    """[first, last) byte of the memory that t spans."""
    if t.numel() == 0:
        return 0, 0
    n = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _apart(out, name, **inputs):
    """Refuses an output in the memory of an input."""
    lo, hi = _reach(out)
    for other, t in inputs.items():
        if t is None:
            continue
        a, b = _reach(t)
        if lo < b and a < hi:
            raise ValueError(f"{name} overlaps {other}")
    return out


def _state_arg(state, name, B, H, device):
    if state is None:
        return None
    _need(state, name, torch.float32, device)
    if state.shape != (B, H):
        raise ValueError(f"{name} must be ({B}, {H})")
    return state


def _reset_arg(reset, B, T, device):
    if reset is None:
        return None
    if not isinstance(reset, torch.Tensor) or not reset.is_cuda or reset.dtype != torch.bool:
        raise ValueError("reset: expected a CUDA bool tensor")
    if reset.device != device or reset.shape != (B, T):
        raise ValueError(f"reset must be ({B}, {T}) on {device}")
    return reset


def _bt(t):
    return (0, 0) if t is None else t.stride()[:2]


@functools.lru_cache(maxsize=256)
def _recurrence_sizes(B, T, H):
    """(fp32 values of the checkpoints, bytes of the workspace)."""
    lib = _lib()
    return (lib.b200_linear_recurrence_checkpoint_bytes(B, T, H) // 4,
            lib.b200_linear_recurrence_workspace_bytes(B, T, H))


def _recurrence_scratch(nbytes, device):
    """(workspace, its address, its bytes); sequences of one tile need none."""
    if nbytes == 0:
        return None, None, 0
    ws = _scratch("linear_recurrence", nbytes, device)
    return ws, ws.data_ptr(), ws.numel()


def _form_code(forms, form):
    """The C ABI's number of a form, -1 for none."""
    return forms.get(form, -1) if isinstance(form, str) else -1


def _recurrence_forward(gate, x, state, reset, form, out, train):
    if out is None:
        r = _call("recurrence", gate, x, state, reset, _form_code(RECURRENCE_FORMS, form), train)
        if r is not None:
            return r
    dev, dt, fm, (B, T, H) = _bth(gate, x, form)
    state = _state_arg(state, "state", B, H, dev)
    reset = _reset_arg(reset, B, T, dev)
    h = _like_bth(x) if out is None else _apart(_writable(out, x, "out"), "out", gate=gate, x=x, state=state,
                                                        reset=reset)
    n_ckpt, n_ws = _recurrence_sizes(B, T, H)
    final = torch.empty((B, H), dtype=torch.float32, device=dev)
    ckpt = torch.empty(n_ckpt, dtype=torch.float32, device=dev) if train else None
    ws, ws_at, ws_bytes = _recurrence_scratch(n_ws, dev)
    _run("linear_recurrence", _lib().b200_linear_recurrence_async, dev.index, gate.data_ptr(), x.data_ptr(), dt, fm,
         _strides(*_bt(gate), *_bt(x), *_bt(h), *_bt(reset)), _address(state), _address(reset), B, T, H, h.data_ptr(),
         final.data_ptr(), _address(ckpt), ws_at, ws_bytes)
    return h, final, ckpt


def linear_recurrence(gate, x, state=None, reset=None, form="decay", out=None):
    """Gated linear recurrence over x [B, T, H]: h[t] = a[t] h[t-1] + v[t] per channel, with a = gate,
    v = x ("decay", |gate| <= 1 expected) or a = sigmoid(gate), v = (1 - a) x ("sigmoid").

    gate and x: fp32, bf16 or fp16 with a contiguous channel axis and any other strides (halves of one
    projection, time-first layouts).  state: fp32 [B, H] before the first step (None: 0).  reset: bool
    [B, T], True where a step starts a new document (the state before it is dropped).  out: x's shape and
    dtype, in memory of its own.  Returns (h of x's dtype, the fp32 state [B, H] after the last step)."""
    h, final, _ = _recurrence_forward(gate, x, state, reset, form, out, False)
    return h, final


def linear_recurrence_train(gate, x, state=None, reset=None, form="decay"):
    """linear_recurrence for training: (h, final state, checkpoints); the checkpoints (fp32 states at
    fixed steps) are what linear_recurrence_backward recomputes h from."""
    return _recurrence_forward(gate, x, state, reset, form, None, True)


def linear_recurrence_backward(gate, x, checkpoints, grad_h, grad_final=None, reset=None, form="decay"):
    """Gradients of linear_recurrence: (grad_gate, grad_x, grad_state) for grad_h [B, T, H] (x's dtype) and
    grad_final (fp32 [B, H] or None)."""
    r = _call("recurrence_backward", gate, x, checkpoints, grad_h, grad_final, reset,
              _form_code(RECURRENCE_FORMS, form))
    if r is not None:
        return r
    dev, dt, fm, (B, T, H) = _bth(gate, x, form)
    _float_tensor(grad_h, "grad_h", dev, x.dtype, 3)
    if grad_h.shape != x.shape:
        raise ValueError("grad_h must have x's shape")
    grad_final = _state_arg(grad_final, "grad_final", B, H, dev)
    reset = _reset_arg(reset, B, T, dev)
    n_ckpt, n_ws = _recurrence_sizes(B, T, H)
    _need(checkpoints, "checkpoints", torch.float32, dev)
    if checkpoints.numel() != n_ckpt:
        raise ValueError("checkpoints do not belong to inputs of this shape")
    gg, gx = _like_bth(gate), _like_bth(x)
    gs = torch.empty((B, H), dtype=torch.float32, device=dev)
    ws, ws_at, ws_bytes = _recurrence_scratch(n_ws, dev)
    _run("linear_recurrence_backward", _lib().b200_linear_recurrence_backward_async, dev.index, gate.data_ptr(),
         x.data_ptr(), dt, fm, _strides(*_bt(gate), *_bt(x), *_bt(grad_h), *_bt(gg), *_bt(gx), *_bt(reset)),
         checkpoints.data_ptr(), _address(reset), grad_h.data_ptr(), _address(grad_final), B, T, H, gg.data_ptr(),
         gx.data_ptr(), gs.data_ptr(), ws_at, ws_bytes)
    return gg, gx, gs


def linear_recurrence_step(gate, x, state, slots=None, form="decay", out=None, state_out=None):
    """One token per row: h [B, H] from gate and x [B, H] and a pool of states fp32 [S, H], updated in place
    (or written to state_out, whose other rows stay as they are).  slots (int32 [B]) names each row's state, row b its own without it.  Rows
    with the same slot are consecutive tokens of one sequence, in row order; a row whose slot is outside
    [0, S) is skipped (its h row is left as it was, so pass `out` to know what it holds)."""
    if out is None:
        r = _call("recurrence_step", gate, x, state, slots, _form_code(RECURRENCE_FORMS, form), state_out)
        if r is not None:
            return r[0]
    if form not in RECURRENCE_FORMS:
        raise ValueError(f"form must be one of {sorted(RECURRENCE_FORMS)}, got {form!r}")
    _float_tensor(x, "x", dims=2)
    dev, shape = x.device, x.shape
    _float_tensor(gate, "gate", dev, x.dtype, 2)
    if gate.shape != shape:
        raise ValueError("gate and x must have the same shape (B, H)")
    B, H = shape
    _need(state, "state", torch.float32, dev)
    if state.dim() != 2 or state.shape[1] != H:
        raise ValueError(f"state must be (slots, {H})")
    S = state.shape[0]
    if S > _I32_MAX:
        raise ValueError("state has more than 2^31 - 1 rows")
    if state_out is None:
        state_out = state
    else:
        _need(state_out, "state_out", torch.float32, dev)
        if state_out.shape != state.shape:
            raise ValueError("state_out must have state's shape")
        if state_out.data_ptr() != state.data_ptr():
            _apart(state_out, "state_out", state=state)
    if slots is None:
        if S < B:
            raise ValueError("state has fewer rows than x and no slots are given")
    else:
        _need(slots, "slots", torch.int32, dev)
        if slots.shape != (B,):
            raise ValueError(f"slots must be ({B},)")
    _apart(state_out, "the written state", gate=gate, x=x, slots=slots)
    h = _dense_like(x) if out is None else _apart(_writable(out, x, "out"), "out", gate=gate, x=x, state=state,
                                                       state_out=state_out)
    _run("linear_recurrence_step", _lib().b200_linear_recurrence_step_async, dev.index, gate.data_ptr(), x.data_ptr(),
         DTYPE_CODES[x.dtype], RECURRENCE_FORMS[form], _strides(gate.stride(0), x.stride(0), h.stride(0)),
         state.data_ptr(), state_out.data_ptr(), _address(slots), S, B, H, h.data_ptr())
    return h


class LinearRecurrenceFunction(torch.autograd.Function):
    """torch.autograd form of the recurrence: apply(gate, x, state, reset, form) -> (h, final state), forward
    through linear_recurrence_train, backward through linear_recurrence_backward."""

    @staticmethod
    def forward(ctx, gate, x, state=None, reset=None, form="decay"):
        h, final, ckpt = linear_recurrence_train(gate, x, state, reset, form)
        ctx.save_for_backward(gate, x, ckpt, reset)
        ctx.form = form
        return h, final

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_final):
        gate, x, ckpt, reset = ctx.saved_tensors
        if grad_h is None:
            grad_h = torch.zeros_like(x)
        elif grad_h.shape[-1] > 1 and grad_h.stride(-1) != 1:
            grad_h = grad_h.contiguous()
        gf = None if grad_final is None else grad_final.contiguous()
        gg, gx, gs = linear_recurrence_backward(gate, x, ckpt, grad_h, gf, reset, ctx.form)
        return gg, gx, gs if _needs(ctx, 2) else None, None, None


# ------------------------------------------------------------------------------ token log-probs
def _token_args(logits, token):
    """(device, dtype code, B, T, V, strides) of logits [..., V] and token [...] with 1 or 2 leading axes."""
    _float_tensor(logits, "logits")
    shape, device = logits.shape, logits.device
    if len(shape) not in (2, 3):
        raise ValueError("logits must be (N, V) or (B, T, V)")
    if not isinstance(token, torch.Tensor) or token.dtype != torch.int64:
        raise ValueError("token: expected an int64 tensor")
    if token.device != device:
        raise ValueError(f"token: on {token.device}, expected {device}")
    if token.shape != shape[:-1]:
        raise ValueError("token must have the shape of logits without the last axis")
    V = shape[-1]
    if V < 1:
        raise ValueError("logits: the vocabulary is empty")
    if len(shape) == 2:
        B, T = 1, shape[0]
        st = _strides(0, logits.stride(0), 0, token.stride(0))
    else:
        B, T = shape[:2]
        st = _strides(logits.stride(0), logits.stride(1), token.stride(0), token.stride(1))
    if B * T > _I32_MAX:
        raise ValueError("logits: more than 2^31 - 1 rows")
    return device, DTYPE_CODES[logits.dtype], B, T, V, st


def _check_over(out, logits):
    """out is memory of its own, or exactly the logits (contiguous)."""
    if out.numel() == 0 or (out.data_ptr() == logits.data_ptr() and logits.is_contiguous()):
        return
    _apart(out, "out", logits=logits)


def _temperature(temperature):
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError("temperature must be positive (between 1e-30 and 1e30)")
    return temperature


def _token_logprob(logits, token, temperature, entropy, train):
    r = _call("logprob", logits, token, temperature, bool(entropy), train)
    if r is not None:
        return r
    dev, dt, B, T, V, st = _token_args(logits, token)
    temperature = _temperature(temperature)
    lp = torch.empty(token.shape, dtype=torch.float32, device=dev)
    ent = _dense_like(lp) if entropy else None
    stats = torch.empty((*token.shape, 3), dtype=torch.float32, device=dev) if train else None
    _run("token_logprob", _lib().b200_token_logprob_async, dev.index, logits.data_ptr(), dt, st, token.data_ptr(), B, T,
         V, temperature, lp.data_ptr(), _address(ent), _address(stats))
    return lp, ent, stats


def token_logprob(logits, token, temperature=1.0, entropy=True):
    """Log-probability (fp32) of each position's token under softmax(logits / temperature), and that
    distribution's entropy (fp32, None unless `entropy`).

    logits: fp32, bf16 or fp16 [N, V] or [B, T, V] with a contiguous vocabulary axis (views such as
    logits[:, :-1] are taken as they are); token: int64 of the leading shape.  A negative token masks its
    position (outputs 0); a token >= V gives NaN, and so does a position whose logits are all -inf or hold a
    NaN or +inf."""
    lp, ent, _ = _token_logprob(logits, token, temperature, entropy, False)
    return lp, ent


def token_logprob_train(logits, token, temperature=1.0, entropy=True):
    """token_logprob for training: (log_prob, entropy, stats), stats (fp32 [..., 3]) for
    token_logprob_backward (with grad_entropy only if `entropy`)."""
    return _token_logprob(logits, token, temperature, entropy, True)


def token_logprob_backward(logits, token, stats, grad_log_prob, grad_entropy=None, temperature=1.0, out=None):
    """grad_logits (contiguous, of logits' dtype) for the gradients of token_logprob's outputs (fp32).  out may
    be the logits themselves when these are contiguous (they are overwritten)."""
    if out is None:
        r = _call("logprob_backward", logits, token, stats, grad_log_prob, grad_entropy, temperature)
        if r is not None:
            return r[0]
    dev, dt, B, T, V, st = _token_args(logits, token)
    temperature = _temperature(temperature)
    for t, nm, shape in ((stats, "stats", (*token.shape, 3)), (grad_log_prob, "grad_log_prob", token.shape),
                         (grad_entropy, "grad_entropy", token.shape)):
        if t is None and nm == "grad_entropy":
            continue
        _need(t, nm, torch.float32, dev)
        if t.shape != shape:
            raise ValueError(f"{nm} must be {tuple(shape)}")
    if out is None:
        out = _dense_like(logits)
    else:
        _need(out, "out", logits.dtype, dev)
        if out.shape != logits.shape:
            raise ValueError("out must have logits' shape")
        _check_over(out, logits)
        _apart(out, "out", token=token, stats=stats, grad_log_prob=grad_log_prob, grad_entropy=grad_entropy)
    _run("token_logprob_backward", _lib().b200_token_logprob_backward_async, dev.index, logits.data_ptr(), dt, st,
         token.data_ptr(), stats.data_ptr(), grad_log_prob.data_ptr(), _address(grad_entropy), B, T, V, temperature,
         out.data_ptr())
    return out


class TokenLogProbFunction(torch.autograd.Function):
    """torch.autograd form: apply(logits, token, temperature) -> (log_prob, entropy)."""

    @staticmethod
    def forward(ctx, logits, token, temperature=1.0):
        lp, ent, stats = token_logprob_train(logits, token, temperature)
        ctx.save_for_backward(logits, token, stats)
        ctx.temperature = float(temperature)
        ctx.set_materialize_grads(False)
        return lp, ent

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_lp, grad_ent):
        logits, token, stats = ctx.saved_tensors
        if grad_lp is None and grad_ent is None:
            return None, None, None
        gl = torch.zeros(token.shape, device=logits.device) if grad_lp is None else grad_lp.contiguous()
        ge = None if grad_ent is None else grad_ent.contiguous()
        return token_logprob_backward(logits, token, stats, gl, ge, ctx.temperature), None, None


# ----------------------------------------------------------------- policy and preference losses
KL_FORMS = {"k1": 0, "k2": 1, "k3": 2}
LOSS_REDUCTIONS = {"token_mean": 0, "sequence_mean": 1, "sum": 2}
PREFERENCE_FORMS = {"sigmoid": 0, "hinge": 1, "ipo": 2}
POLICY_OUTPUTS = ("loss", "policy", "kl", "entropy", "clip_fraction", "approx_kl", "max_ratio", "mean_ratio")
PREFERENCE_OUTPUTS = ("loss", "accuracy", "margin")


def _token_stream(t, name, B, T, device, dtype=torch.float32):
    """A [B, T] per-token tensor with a contiguous token axis."""
    if isinstance(t, torch.Tensor) and t.shape == (B, T) and t.dtype == dtype and t.stride(1) == 1 \
            and t.device == device:
        return t
    _float_tensor(t, name, device, dtype, 2)
    if t.shape != (B, T):
        raise ValueError(f"{name} must be ({B}, {T}), got {tuple(t.shape)}")
    return t


def _row_stride(t):
    return 0 if t is None else t.stride(0)


def _number(v, name):
    v = float(v)
    if v != v or v in (float("inf"), float("-inf")):
        raise ValueError(f"{name} must be finite")
    return v


def _policy_options(clip_low, clip_high, dual_clip, kl_coef, kl_form, entropy_coef, reduction, scale, has_ref,
                    has_entropy):
    """The loss's options checked, as the C ABI takes them.  They are made Python's numbers first, so that a tensor is
    read in every call."""
    return _checked_policy_options(float(clip_low), float(clip_high), None if dual_clip is None else float(dual_clip),
                                   float(kl_coef), kl_form, float(entropy_coef), reduction, float(scale), has_ref,
                                   has_entropy)


@functools.lru_cache(maxsize=256)
def _checked_policy_options(clip_low, clip_high, dual_clip, kl_coef, kl_form, entropy_coef, reduction, scale, has_ref,
                            has_entropy):
    if kl_form not in KL_FORMS:
        raise ValueError(f"kl_form must be one of {sorted(KL_FORMS)}, got {kl_form!r}")
    if reduction not in LOSS_REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(LOSS_REDUCTIONS)}, got {reduction!r}")
    clip_low, clip_high = _number(clip_low, "clip_low"), _number(clip_high, "clip_high")
    if not 0.0 <= clip_low < 1.0 or clip_high < 0.0:
        raise ValueError("clip_low must be in [0, 1) and clip_high >= 0")
    dual = 0.0 if dual_clip is None else _number(dual_clip, "dual_clip")
    if dual_clip is not None and dual <= 1.0:
        raise ValueError("dual_clip must be larger than 1")
    kl_coef, entropy_coef = _number(kl_coef, "kl_coef"), _number(entropy_coef, "entropy_coef")
    if kl_coef != 0.0 and not has_ref:
        raise ValueError("kl_coef needs ref_log_prob")
    if entropy_coef != 0.0 and not has_entropy:
        raise ValueError("entropy_coef needs entropy")
    return (clip_low, clip_high, dual, kl_coef, KL_FORMS[kl_form], entropy_coef, LOSS_REDUCTIONS[reduction],
            _number(scale, "scale"))


@functools.lru_cache(maxsize=256)
def _policy_scratch_bytes(B, T):
    return _lib().b200_policy_loss_workspace_bytes(B, T)


def _policy_loss(log_prob, old_log_prob, advantage, mask, ref_log_prob, entropy, clip_low, clip_high, dual_clip,
                 kl_coef, kl_form, entropy_coef, reduction, scale, want_grad, want_grad_entropy):
    options = _policy_options(clip_low, clip_high, dual_clip, kl_coef, kl_form, entropy_coef, reduction, scale,
                              ref_log_prob is not None, entropy is not None)
    r = _call("policy", log_prob, old_log_prob, advantage, mask, ref_log_prob, entropy, options, want_grad,
              want_grad_entropy)
    if r is not None:
        return r
    _float_tensor(log_prob, "log_prob", dtype=torch.float32, dims=2)
    dev = log_prob.device
    B, T = log_prob.shape
    old = log_prob if old_log_prob is None else _token_stream(old_log_prob, "old_log_prob", B, T, dev)
    if isinstance(advantage, torch.Tensor) and advantage.dim() == 1:
        _float_tensor(advantage.unsqueeze(1), "advantage", dev, torch.float32)
        if advantage.shape != (B,):
            raise ValueError(f"advantage must be ({B},) or ({B}, {T})")
        adv_e = 0
    else:
        _token_stream(advantage, "advantage", B, T, dev)
        adv_e = 1
    if mask is not None:
        _token_stream(mask, "mask", B, T, dev, torch.bool)
    if ref_log_prob is not None:
        _token_stream(ref_log_prob, "ref_log_prob", B, T, dev)
    if entropy is not None:
        _token_stream(entropy, "entropy", B, T, dev)
    out = torch.empty(8, dtype=torch.float32, device=dev)
    grad = _dense_like(log_prob) if want_grad else None
    ge = _dense_like(log_prob) if want_grad_entropy else None
    n_ws = _policy_scratch_bytes(B, T)
    ws = _scratch("policy_loss", n_ws, dev) if n_ws else None
    _run("policy_loss", _lib().b200_policy_loss_async, dev.index, log_prob.data_ptr(), old.data_ptr(),
         advantage.data_ptr(), _address(ref_log_prob), _address(entropy), _address(mask),
         _strides(log_prob.stride(0), old.stride(0), advantage.stride(0), adv_e, _row_stride(ref_log_prob),
                  _row_stride(entropy), _row_stride(mask)),
         B, T, *options, out.data_ptr(), _address(grad), _address(ge), _address(ws), ws.numel() if n_ws else 0)
    return out, grad, ge


def policy_loss(log_prob, old_log_prob, advantage, mask=None, ref_log_prob=None, entropy=None, clip_low=0.2,
                clip_high=0.2, dual_clip=None, kl_coef=0.0, kl_form="k3", entropy_coef=0.0, reduction="token_mean",
                scale=1.0):
    """Clipped policy loss of token log-probs fp32 [B, T] with a KL term to ref_log_prob and an entropy
    term: a tensor of POLICY_OUTPUTS.

    old_log_prob: [B, T], or None for an update on the policy's own samples (ratio 1).  advantage: [B, T],
    or [B] for one per sequence.  mask: bool [B, T], True where a token counts; what masked-out tokens
    hold is never looked at.  The token axis of each is contiguous, rows may be strided.  kl_form: "k1", "k2" or "k3";
    reduction: "token_mean", "sequence_mean" (mean over the non-empty sequences of their means) or
    "sum"; scale multiplies the loss."""
    return _policy_loss(log_prob, old_log_prob, advantage, mask, ref_log_prob, entropy, clip_low, clip_high,
                        dual_clip, kl_coef, kl_form, entropy_coef, reduction, scale, False, False)[0]


def policy_loss_grad(log_prob, old_log_prob, advantage, mask=None, ref_log_prob=None, entropy=None, clip_low=0.2,
                     clip_high=0.2, dual_clip=None, kl_coef=0.0, kl_form="k3", entropy_coef=0.0,
                     reduction="token_mean", scale=1.0):
    """policy_loss with its gradients: (outputs, d loss / d log_prob [B, T], d loss / d entropy [B, T] or None
    without an entropy)."""
    return _policy_loss(log_prob, old_log_prob, advantage, mask, ref_log_prob, entropy, clip_low, clip_high,
                        dual_clip, kl_coef, kl_form, entropy_coef, reduction, scale, True, entropy is not None)


class PolicyLossFunction(torch.autograd.Function):
    """torch.autograd form: apply(log_prob, entropy, old_log_prob, advantage, mask, ref_log_prob, options) ->
    (loss, outputs), options a dict of policy_loss's other arguments.  The forward computes the gradients
    with the loss; the backward scales them.  outputs (POLICY_OUTPUTS) carries no gradient."""

    @staticmethod
    def forward(ctx, log_prob, entropy, old_log_prob, advantage, mask=None, ref_log_prob=None, options=None):
        if any(_needs(ctx, k) for k in (2, 3, 5)):
            raise ValueError("PolicyLossFunction: old_log_prob, advantage and ref_log_prob are constants; detach them")
        o = dict(clip_low=0.2, clip_high=0.2, dual_clip=None, kl_coef=0.0, kl_form="k3", entropy_coef=0.0,
                 reduction="token_mean", scale=1.0)
        unknown = set(options or {}) - set(o)
        if unknown:
            raise TypeError(f"PolicyLossFunction: unknown options {sorted(unknown)}")
        o.update(options or {})
        out, grad, ge = _policy_loss(log_prob, old_log_prob, advantage, mask, ref_log_prob, entropy, **o,
                                     want_grad=ctx.needs_input_grad[0], want_grad_entropy=ctx.needs_input_grad[1])
        ctx.save_for_backward(grad, ge)
        ctx.mark_non_differentiable(out)
        return out[0].clone(), out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        grad, ge = ctx.saved_tensors
        return (None if grad is None else grad * grad_loss, None if ge is None else ge * grad_loss, None, None, None,
                None, None)


def _preference_options(beta, form, label_smoothing, margin):
    """The loss's options checked, as the C ABI takes them (as in _policy_options)."""
    return _checked_preference_options(float(beta), form, float(label_smoothing), float(margin))


@functools.lru_cache(maxsize=256)
def _checked_preference_options(beta, form, label_smoothing, margin):
    if form not in PREFERENCE_FORMS:
        raise ValueError(f"form must be one of {sorted(PREFERENCE_FORMS)}, got {form!r}")
    beta, margin = _number(beta, "beta"), _number(margin, "margin")
    label_smoothing = _number(label_smoothing, "label_smoothing")
    if beta <= 0.0:
        raise ValueError("beta must be positive")
    if not 0.0 <= label_smoothing <= 0.5 or (label_smoothing and form != "sigmoid"):
        raise ValueError("label_smoothing must be in [0, 0.5], and 0 unless form is 'sigmoid'")
    return beta, PREFERENCE_FORMS[form], label_smoothing, margin


@functools.lru_cache(maxsize=256)
def _preference_scratch_bytes(B):
    return _lib().b200_preference_loss_workspace_bytes(B)


def _preference_loss(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta, form,
                     label_smoothing, margin, average, want_chosen, want_rejected):
    options = _preference_options(beta, form, label_smoothing, margin)
    r = _call("preference", chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, options,
              bool(average), want_chosen, want_rejected)
    if r is not None:
        return r
    _float_tensor(chosen, "chosen", dtype=torch.float32, dims=2)
    dev = chosen.device
    _float_tensor(rejected, "rejected", dev, torch.float32, 2)
    (B, Tc), Tr = chosen.shape, rejected.shape[1]
    if rejected.shape[0] != B:
        raise ValueError("chosen and rejected must have the same number of rows")
    if (ref_chosen is None) != (ref_rejected is None):
        raise ValueError("ref_chosen and ref_rejected go together")
    if ref_chosen is not None:
        _token_stream(ref_chosen, "ref_chosen", B, Tc, dev)
        _token_stream(ref_rejected, "ref_rejected", B, Tr, dev)
    if chosen_mask is not None:
        _token_stream(chosen_mask, "chosen_mask", B, Tc, dev, torch.bool)
    if rejected_mask is not None:
        _token_stream(rejected_mask, "rejected_mask", B, Tr, dev, torch.bool)
    out = torch.empty(3, dtype=torch.float32, device=dev)
    rc = torch.empty(B, dtype=torch.float32, device=dev)
    rr = torch.empty(B, dtype=torch.float32, device=dev)
    gc = _dense_like(chosen) if want_chosen else None
    gr = _dense_like(rejected) if want_rejected else None
    ws = _scratch("preference_loss", _preference_scratch_bytes(B), dev)
    _run("preference_loss", _lib().b200_preference_loss_async, dev.index, chosen.data_ptr(), rejected.data_ptr(),
         _address(ref_chosen), _address(ref_rejected), _address(chosen_mask), _address(rejected_mask),
         _strides(chosen.stride(0), rejected.stride(0), _row_stride(ref_chosen), _row_stride(ref_rejected),
                  _row_stride(chosen_mask), _row_stride(rejected_mask)),
         B, Tc, Tr, *options, 1 if average else 0, out.data_ptr(), rc.data_ptr(), rr.data_ptr(), _address(gc),
         _address(gr), ws.data_ptr(), ws.numel())
    return out, rc, rr, gc, gr


def preference_loss(chosen, rejected, ref_chosen=None, ref_rejected=None, chosen_mask=None, rejected_mask=None,
                    beta=0.1, form="sigmoid", label_smoothing=0.0, margin=0.0, average=False):
    """Preference loss over pairs of answers given as token log-probs fp32 [B, Tc] and [B, Tr]: (a tensor of
    PREFERENCE_OUTPUTS, reward_chosen [B], reward_rejected [B]).

    Each answer counts with the sum (the mean with `average`) of its masked tokens' log_prob - ref_log_prob;
    z = beta * (chosen - rejected) - margin goes through form "sigmoid" (with label_smoothing),
    "hinge" or "ipo".  Without the references the log-probs count alone.  masks: bool, True where a token
    counts.  Rows may be strided (halves of one concatenated batch)."""
    return _preference_loss(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta, form,
                            label_smoothing, margin, average, False, False)[:3]


def preference_loss_grad(chosen, rejected, ref_chosen=None, ref_rejected=None, chosen_mask=None, rejected_mask=None,
                         beta=0.1, form="sigmoid", label_smoothing=0.0, margin=0.0, average=False):
    """preference_loss with its gradients: (outputs, reward_chosen, reward_rejected, d loss / d chosen [B, Tc],
    d loss / d rejected [B, Tr])."""
    return _preference_loss(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, beta, form,
                            label_smoothing, margin, average, True, True)


class PreferenceLossFunction(torch.autograd.Function):
    """torch.autograd form: apply(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, options)
    -> (loss, outputs, reward_chosen, reward_rejected), options a dict of preference_loss's other arguments.
    Only the loss carries a gradient."""

    @staticmethod
    def forward(ctx, chosen, rejected, ref_chosen=None, ref_rejected=None, chosen_mask=None, rejected_mask=None,
                options=None):
        if _needs(ctx, 2) or _needs(ctx, 3):
            raise ValueError("PreferenceLossFunction: the reference log-probs are constants; detach them")
        o = dict(beta=0.1, form="sigmoid", label_smoothing=0.0, margin=0.0, average=False)
        unknown = set(options or {}) - set(o)
        if unknown:
            raise TypeError(f"PreferenceLossFunction: unknown options {sorted(unknown)}")
        o.update(options or {})
        out, rc, rr, gc, gr = _preference_loss(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask,
                                               **o, want_chosen=ctx.needs_input_grad[0],
                                               want_rejected=ctx.needs_input_grad[1])
        ctx.save_for_backward(gc, gr)
        ctx.mark_non_differentiable(out, rc, rr)
        return out[0].clone(), out, rc, rr

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, *_):
        gc, gr = ctx.saved_tensors
        return (None if gc is None else gc * grad_loss, None if gr is None else gr * grad_loss, None, None, None, None,
                None)


# ----------------------------------------------------------------------------------------- KAN
def efficient_kan(x, grid, base_weight, spline_weight, spline_scaler, grid_size, spline_order, out=None):
    """KANLinear forward: out[B, O] = silu(x) base_weight^T + bases(x) (spline_weight * scaler)^T."""
    _need(x, "x", torch.float32)
    dev = x.device
    for t, nm in ((grid, "grid"), (base_weight, "base_weight"), (spline_weight, "spline_weight"),
                  (spline_scaler, "spline_scaler")):
        _need(t, nm, torch.float32, dev)
    B, I = x.shape
    O = base_weight.shape[0]
    G, K = int(grid_size), int(spline_order)
    if grid.shape != (I, G + 2 * K + 1) or base_weight.shape != (O, I) or spline_weight.shape != (O, I, G + K) \
            or spline_scaler.shape != (O, I):
        raise ValueError("efficient_kan: inconsistent shapes")
    out = torch.empty((B, O), dtype=torch.float32, device=dev) if out is None else out
    lib = _lib()
    ws = workspace("kan", lib.b200_efficient_kan_workspace_bytes(G, K, B, I, O), dev)
    _native.check(lib.b200_efficient_kan_async(_ptr(x), _ptr(grid), _ptr(base_weight), _ptr(spline_weight),
                                               _ptr(spline_scaler), G, K, B, I, O, _ptr(out), _ptr(ws),
                                               ws.numel(), _stream(dev)), "efficient_kan")
    return out


def efficient_kan_backward(x, grid, base_weight, spline_weight, spline_scaler, grid_size, spline_order, grad_out,
                           need_x=True, need_weights=True):
    """Gradients of efficient_kan for grad_out [B, O]: (grad_x, grad_base_weight, grad_spline_weight,
    grad_spline_scaler); the input gradient is None unless need_x, the weight gradients None
    unless need_weights."""
    _need(x, "x", torch.float32)
    dev = x.device
    for t, nm in ((grid, "grid"), (base_weight, "base_weight"), (spline_weight, "spline_weight"),
                  (spline_scaler, "spline_scaler"), (grad_out, "grad_out")):
        _need(t, nm, torch.float32, dev)
    B, I = x.shape
    O = base_weight.shape[0]
    G, K = int(grid_size), int(spline_order)
    if grid.shape != (I, G + 2 * K + 1) or base_weight.shape != (O, I) or spline_weight.shape != (O, I, G + K) \
            or spline_scaler.shape != (O, I) or grad_out.shape != (B, O):
        raise ValueError("efficient_kan_backward: inconsistent shapes")
    gx = torch.empty_like(x) if need_x else None
    gwb = torch.empty_like(base_weight) if need_weights else None
    gsw = torch.empty_like(spline_weight) if need_weights else None
    gsc = torch.empty_like(spline_scaler) if need_weights else None
    lib = _lib()
    ws = workspace("kan_backward", lib.b200_efficient_kan_backward_workspace_bytes(G, K, B, I, O), dev)
    _native.check(lib.b200_efficient_kan_backward_async(_ptr(x), _ptr(grid), _ptr(base_weight), _ptr(spline_weight),
                                                        _ptr(spline_scaler), G, K, B, I, O, _ptr(grad_out), _ptr(gx),
                                                        _ptr(gwb), _ptr(gsw), _ptr(gsc), _ptr(ws), ws.numel(),
                                                        _stream(dev)), "efficient_kan_backward")
    return gx, gwb, gsw, gsc


class KANLinearFunction(torch.autograd.Function):
    """torch.autograd form of the KAN layer: forward through efficient_kan, backward through
    efficient_kan_backward (the knot grid gets no gradient, as a KANLinear buffer)."""

    @staticmethod
    def forward(ctx, x, grid, base_weight, spline_weight, spline_scaler, grid_size, spline_order):
        ctx.save_for_backward(x, grid, base_weight, spline_weight, spline_scaler)
        ctx.gk = (int(grid_size), int(spline_order))
        return efficient_kan(x, grid, base_weight, spline_weight, spline_scaler, grid_size, spline_order)

    @staticmethod
    def backward(ctx, grad_out):
        x, grid, wb, sw, sc = ctx.saved_tensors
        need_x = ctx.needs_input_grad[0]
        need_w = any(ctx.needs_input_grad[2:5])
        gx, gwb, gsw, gsc = efficient_kan_backward(x, grid, wb, sw, sc, *ctx.gk, grad_out.contiguous(), need_x, need_w)
        return gx, None, gwb, gsw, gsc, None, None


# ---------------------------------------------------------------------------------- FP8 linear
def fp8_quantize(x, q=None, scale=None):
    """Per-tensor E4M3 quantisation of an fp32 or bf16 tensor (tasks/fp8_linear/reference.py:15-18):
    returns (q as float8_e4m3fn with x's shape, scale as a 1-element fp32 device tensor)."""
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("fp8_quantize: x must be float32 or bfloat16")
    _need(x, "x", x.dtype)
    dev = x.device
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev) if q is None else q
    scale = torch.empty(1, dtype=torch.float32, device=dev) if scale is None else scale
    lib = _lib()
    ws = workspace("fp8q", lib.b200_fp8_quantize_workspace_bytes(), dev)
    _native.check(lib.b200_fp8_quantize_async(_ptr(x), 1 if x.dtype == torch.bfloat16 else 0, x.numel(), _ptr(q),
                                              _ptr(scale), _ptr(ws), ws.numel(), _stream(dev)), "fp8_quantize")
    return q, scale


def fp8_linear_bf16(x, w_fp8, scale_w, bias, out=None, scale_x=None):
    """The linear layer from a bf16 activation x [M, K]: quantise x on the device, then the E4M3
    GEMM; the same bits as fp8_quantize followed by fp8_linear with the computed scale."""
    _need(x, "x", torch.bfloat16)
    dev = x.device
    _need(w_fp8, "w_fp8", torch.float8_e4m3fn, dev)
    _need(bias, "bias", torch.bfloat16, dev)
    M, K = x.shape
    N = w_fp8.shape[0]
    if w_fp8.shape[1] != K or bias.numel() != N:
        raise ValueError("fp8_linear_bf16: inconsistent shapes")
    out = torch.empty((M, N), dtype=torch.bfloat16, device=dev) if out is None else out
    lib = _lib()
    ws = workspace("fp8lin", lib.b200_fp8_linear_bf16_workspace_bytes(M, K), dev)
    _native.check(lib.b200_fp8_linear_bf16_async(M, K, N, _ptr(x), _ptr(w_fp8), float(scale_w), _ptr(bias),
                                                 _ptr(out), _opt_ptr(scale_x, None), _ptr(ws), ws.numel(),
                                                 _stream(dev)), "fp8_linear_bf16")
    return out


def fp8_linear(x_fp8, scale_x, w_fp8, scale_w, bias, out=None):
    """bf16 (x_fp8 / scale_x) (w_fp8 / scale_w)^T + bias with E4M3 operands [M, K] and [N, K]."""
    _need(x_fp8, "x_fp8", torch.float8_e4m3fn)
    dev = x_fp8.device
    _need(w_fp8, "w_fp8", torch.float8_e4m3fn, dev)
    _need(bias, "bias", torch.bfloat16, dev)
    M, K = x_fp8.shape
    N = w_fp8.shape[0]
    if w_fp8.shape[1] != K or bias.numel() != N:
        raise ValueError("fp8_linear: inconsistent shapes")
    out = torch.empty((M, N), dtype=torch.bfloat16, device=dev) if out is None else out
    _native.check(_lib().b200_fp8_linear_async(M, K, N, _ptr(x_fp8), float(scale_x), _ptr(w_fp8), float(scale_w),
                                               _ptr(bias), _ptr(out), _stream(dev)), "fp8_linear")
    return out


# ------------------------------------------------------------------- reference-interface mirror
def reference(task, inp):
    """Drop-in for tasks/<task>/reference.py:reference(inp): same keys in, same keys out."""
    if task == "pow_abs_sqrt_mean":
        return {"output": robust_l1(inp["inp"], inp["target"])}
    if task == "ppo_clip":
        return {"output": ppo_clip(inp["current_log_prob"], inp["old_log_prob"], inp["advantage"],
                                   inp["clip_epsilon"], inp.get("entropy"))}
    if task == "reward_to_go":
        return {"output": reward_to_go(inp["reward"], inp["done"], inp["gamma"])}
    if task == "leaky":
        s, m = leaky(inp["input_current"], inp["mem0"], inp["beta"], inp["threshold"])
        return {"spikes": s, "final_mem": m}
    if task == "efficient_kan":
        return {"out": efficient_kan(inp["x"], inp["grid"], inp["base_weight"], inp["spline_weight"],
                                     inp["spline_scaler"], inp["grid_size"], inp["spline_order"])}
    if task == "fp8_linear":
        return {"output": fp8_linear(inp["x_fp8"], inp["scale_x"], inp["w_fp8"], inp["scale_w"], inp["bias"])}
    raise KeyError(f"unknown or not yet built task: {task}")
