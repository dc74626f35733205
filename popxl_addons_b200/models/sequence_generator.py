"""Serving of models with per-sequence state (recurrent state, caches): portions of prompts, decoding, logits on request and
greedy generation for a batch of unequal prompts.

A model object (see `models/dunelix.py`) describes its weights, its state and the ops of one portion; everything else is here
and does not know the architecture:

* **slots**: the batch axis of all state tensors. A request takes a slot (`admit`), its tokens advance the slot's position,
  `release` gives it back. A slot needs no clearing: a sequence at position 0 starts from the empty state.
* **portions**: `step` runs the next tokens of any of the live requests, of unequal lengths, cut anywhere. Portion lengths are
  rounded up to a ladder of sizes; padded rows touch neither caches nor recurrent state. One `Program` per size, captured
  into a CUDA graph at its second use.
* **decoding**: tokens, positions and the output buffer stay on the device, so a decoding step is one graph replay.
* **requests of their own kind**: a request may bring an adapter of the model (`load_adapter`), and what shapes its logits before a token
  is chosen (`LogitShaping`). Both are looked up by slot on the device: a batch of unlike requests is one step like any other.
"""
import math
from dataclasses import dataclass
from typing import Dict, List, Mapping, Optional, Sequence, Union

import numpy as np
import torch

from .. import xl
from ..xl import ops

__all__ = ["LogitShaping", "SequenceGenerator", "portion_size"]


@dataclass(frozen=True)
class LogitShaping:
    """What changes the logits of a request, in this order. `repetition`: logits of tokens that occurred are divided by it where
    positive, else multiplied; `frequency` is subtracted for every time a token occurred since the prompt, `presence` once; `biases`
    (token -> value) are added; tokens that are not `allowed` (token ids, or a truth value for every token; None: all are) cannot be
    chosen."""
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    biases: Optional[Mapping[int, float]] = None
    allowed: Optional[Sequence[int]] = None


def mask_words(allowed, vocab: int) -> torch.Tensor:
    """Token ids, or a truth value for every token, as words of 32 bits; None allows everything."""
    bits = torch.ones(vocab, dtype=torch.bool)
    if allowed is not None:
        t = torch.as_tensor(np.asarray(allowed.cpu() if isinstance(allowed, torch.Tensor) else allowed))
        if t.dtype == torch.bool:
            if t.shape != (vocab,):
                raise ValueError(f"a mask has {vocab} truth values, not {tuple(t.shape)}")
            bits = t.clone()
        else:
            if t.dim() != 1 or t.numel() == 0 or t.is_floating_point() or int(t.min()) < 0 or int(t.max()) >= vocab:
                raise ValueError(f"allowed tokens are ids below {vocab}")
            bits = torch.zeros(vocab, dtype=torch.bool)
            bits[t.long()] = True
    if not bits.any():
        raise ValueError("a mask has to allow at least one token")
    words = torch.nn.functional.pad(bits.long(), (0, -vocab % 32)).reshape(-1, 32)
    words = (words << torch.arange(32)).sum(1)
    return torch.where(words > 0x7fffffff, words - (1 << 32), words).to(torch.int32)


def portion_size(n: int) -> int:
    """Smallest ladder size >= n: 1, 2, 4, 8, 16, then eight steps per power of two (at most an eighth of the rows are
    padding), never finer than 16."""
    if n <= 16:
        return 1 << (n - 1).bit_length()
    step = max(16, 1 << ((n - 1).bit_length() - 4))
    return (n + step - 1) // step * step


class SequenceGenerator:
    def __init__(self, model, batch: int = 1, max_seq: int = 2048, max_portion: int = 4096, max_new_tokens: int = 256,
                 device: str = "auto", cuda_graphs: bool = True, use_native: Optional[bool] = None, shaping: bool = False,
                 max_biases: int = 64):
        """`max_seq`: positions a slot can hold; `max_portion`: tokens per sequence of one step's graph (longer portions are
        run in several); `max_new_tokens`: rows of the device buffer that collects generated tokens. `shaping`: requests may bring a
        `LogitShaping` with up to `max_biases` biases; the slots' tokens are then kept on the device."""
        if batch < 1 or max_seq < 1:
            raise ValueError("batch and max_seq must be positive")
        if shaping and not (1 <= max_biases <= ops.MAX_BIASES and max_seq <= ops.MAX_HISTORY):
            raise ValueError(f"shaping takes between 1 and {ops.MAX_BIASES} biases and max_seq up to {ops.MAX_HISTORY}")
        self.shaping, self.max_biases = shaping, max_biases
        self.adapters = getattr(model, "adapters", 0)
        self.model, self.batch, self.max_seq = model, batch, max_seq
        self.max_portion = portion_size(min(max_portion, max_seq))
        self.max_new = max_new_tokens
        self.ir = xl.Ir()
        self.ir.options.cuda_graphs = self.ir.options.cuda_graphs and cuda_graphs
        self._vars: Dict[str, xl.Variable] = {}
        self._mutable = set()
        with self.ir.main_graph:
            for name, (shape, dt) in model.weights().items():
                self._vars[name] = xl.variable(xl.LazyInit(shape, np.float32, "zeros"), dt, name)
            for name, arr in model.tables(max_seq).items():
                self._vars[name] = xl.variable(arr, xl.float32, name)
            state = dict(model.state(batch, max_seq))
            state["stream"] = ((batch * self.max_portion, model.width), xl.float32)
            state.update(pos=((batch,), xl.int32), count=((batch,), xl.int32), current=((batch,), xl.int32),
                         step=((1,), xl.int32), generated=((max_new_tokens, batch), xl.int32))
            if self.adapters:
                state.update(model.adapter_weights(), adapter=((batch,), xl.int32))
            if shaping:
                state.update(history=((batch, max_seq), xl.int32), start=((batch,), xl.int32), penalties=((batch, 3), xl.float32),
                             bias_tokens=((batch, max_biases), xl.int32), bias_values=((batch, max_biases), xl.float32),
                             allowed=((batch, -(-model.vocab // 32)), xl.int32))
            for name, (shape, dt) in state.items():
                self._vars[name] = xl.variable(xl.LazyInit(shape, np.float32, "zeros"), dt, name)
                self._mutable.add(name)
            self._ctrl_in = xl.h2d_stream((2, batch), xl.int32, "slot_positions")
            self._tokens_out = xl.d2h_stream((max_new_tokens, batch), xl.int32, "generated")
        self.session = xl.Session(self.ir, device, use_native=use_native)
        self._programs: Dict[tuple, dict] = {}
        self.lengths = [0] * batch          # positions held by every slot (host mirror of the device-side `pos`)
        self.slots: Dict[object, int] = {}  # live request -> slot
        self._free = list(range(batch))[::-1]
        if self.adapters:
            self._set_device("adapter", -1)
        if shaping:
            for slot in range(batch):
                self._write_shaping(slot, LogitShaping(), 0)

    # -- weights -------------------------------------------------------------------------------------------------------
    def load(self, tensors: Mapping[str, torch.Tensor]):
        """Copy program tensors (`model.convert(...)` or `model.random_weights(...)`) into the session's variables."""
        names = set(self.model.weights())
        if set(tensors) != names:
            raise ValueError(f"weights do not fit: missing {sorted(names - set(tensors))[:8]}, unexpected "
                             f"{sorted(set(tensors) - names)[:8]}")
        for name, value in tensors.items():
            dst = self.session._vars[self._vars[name]][0]
            if tuple(dst.shape) != tuple(value.shape):
                raise ValueError(f"weight {name!r} has shape {tuple(value.shape)}, expected {tuple(dst.shape)}")
            dst.copy_(value)
        return self

    def load_checkpoint(self, ckpt: Mapping[str, torch.Tensor]):
        return self.load(self.model.convert(ckpt, self.session.device))

    def load_adapter(self, index: int, tensors: Mapping[str, torch.Tensor], scale: float = 1.0):
        """Make adapter `index` of `tensors` (see the model's `convert_adapter`); its contributions are multiplied by `scale`."""
        if not 0 <= index < self.adapters:
            raise ValueError(f"this program holds adapters 0 to {self.adapters - 1}, not {index}" if self.adapters else
                             "the model was made without adapters")
        ready = self.model.convert_adapter(tensors)
        for name, value in ready.items():
            self.session.device_tensor(self._vars[name])[index].copy_(value)
        for name in self.model.adapter_weights():
            if name.endswith(".scale"):
                self.session.device_tensor(self._vars[name])[index] = float(scale)
        return self

    # -- slots ---------------------------------------------------------------------------------------------------------
    def admit(self, request, adapter: Optional[int] = None, shaping: Optional[LogitShaping] = None, prompt: int = 0) -> int:
        """Give a request a slot; its first token will be at position 0. `adapter`: which adapter it uses (None: the model alone);
        `shaping`: what changes its logits, of which the first `prompt` tokens count as its prompt."""
        if request in self.slots:
            raise ValueError(f"request {request!r} already holds a slot")
        if not self._free:
            raise RuntimeError(f"all {self.batch} slots are in use")
        if adapter is not None and not 0 <= adapter < self.adapters:
            raise ValueError(f"request {request!r} asks for adapter {adapter} of {self.adapters}")
        if shaping is not None and not self.shaping:
            raise ValueError("this program was made without shaping=True")
        slot = self._free[-1]
        if self.shaping:
            self._write_shaping(slot, shaping or LogitShaping(), prompt)
        if self.adapters:
            self.session.device_tensor(self._vars["adapter"])[slot] = -1 if adapter is None else adapter
        self._free.pop()
        self.slots[request] = slot
        self.lengths[slot] = 0
        return slot

    def release(self, request) -> None:
        slot = self.slots.pop(request)
        self.lengths[slot] = 0
        self._free.append(slot)

    def _write_shaping(self, slot: int, s: LogitShaping, prompt: int) -> None:
        biases = dict(s.biases or {})
        if not (s.repetition > 0 and all(math.isfinite(v) for v in (s.repetition, s.frequency, s.presence))):
            raise ValueError(f"penalties must be finite and repetition positive, not {s.repetition}, {s.frequency}, {s.presence}")
        if len(biases) > self.max_biases or any(not 0 <= k < self.model.vocab for k in biases):
            raise ValueError(f"at most {self.max_biases} biases of tokens below {self.model.vocab}")
        if prompt < 0:
            raise ValueError(f"a prompt has no {prompt} tokens")
        words = mask_words(s.allowed, self.model.vocab)
        tokens, values = torch.full((self.max_biases,), -1, dtype=torch.int32), torch.zeros(self.max_biases)
        tokens[:len(biases)], values[:len(biases)] = torch.tensor(list(biases), dtype=torch.int32), torch.tensor(list(biases.values()))
        for name, value in (("start", torch.tensor(prompt, dtype=torch.int32)), ("bias_tokens", tokens), ("bias_values", values), ("allowed", words),
                            ("penalties", torch.tensor([s.repetition, s.frequency, s.presence]))):
            self.session.device_tensor(self._vars[name])[slot].copy_(value)

    def set_allowed(self, request, allowed) -> None:
        """The tokens that a live request may choose from now on, as in `LogitShaping` (a grammar's next state)."""
        if not self.shaping:
            raise ValueError("this program was made without shaping=True")
        self.session.device_tensor(self._vars["allowed"])[self.slots[request]].copy_(mask_words(allowed, self.model.vocab))

    # -- programs --------------------------------------------------------------------------------------------------------
    def _program(self, key, build):
        entry = self._programs.get(key)
        if entry is None:
            entry = {"program": xl.Program(self.ir, "_".join(str(k) for k in key))}
            with entry["program"] as p:
                build(entry, lambda name: p.use(self._vars[name], by_ref=name in self._mutable))
            self._programs[key] = entry
        return entry

    def _sample(self, t, h):
        """Greedy choice for every slot: becomes the current token and a row of the output buffer."""
        if self.shaping:  # positions have moved on: they are the numbers of tokens that the choice goes by
            ops.take_shaped_(t("current"), self.model.logits(t, h), t("generated"), t("step"), t("pos"), t("count"), self._rules(t),
                             self.model.vocab)
        else:
            ops.take_greedy_(t("current"), self.model.logits(t, h), t("generated"), t("step"), self.model.vocab)

    @staticmethod
    def _rules(t) -> ops.LogitRules:
        return ops.LogitRules(*(t(k) for k in ops.LogitRules._fields))

    def _portion_program(self, T: int, sample: bool):
        def build(entry, t):
            entry["tokens"] = xl.h2d_stream((self.batch * T,), xl.int32, f"tokens_{T}")
            ctrl = ops.host_load(self._ctrl_in)
            tokens = ops.host_load(entry["tokens"])
            ops.var_updates.copy_var_update_(t("pos"), ctrl[0])
            ops.var_updates.copy_var_update_(t("count"), ctrl[1])
            self.model.portion(T, t, tokens, t("pos"), t("count"), final_norm=False)
            if self.shaping:
                ops.append_tokens_(t("history"), tokens, t("pos"), t("count"), T)
                ops.advance_by_(t("pos"), t("count"))
            if sample:
                self._sample(t, self.model.select(t, t("count"), stride=T, offset=1))
            if not self.shaping:
                ops.advance_by_(t("pos"), t("count"))

        return self._program(("portion", T, "sample") if sample else ("portion", T), build)

    def _decode_program(self):
        def build(entry, t):
            h = self.model.portion(1, t, t("current"), t("pos"), t("count"), final_norm=True)
            if self.shaping:
                ops.advance_by_(t("pos"), t("count"))
            self._sample(t, h)
            if not self.shaping:
                ops.advance_by_(t("pos"), t("count"))

        return self._program(("decode",), build)

    def _logits_program(self, n: int, shaped: bool = False):
        def build(entry, t):
            entry["rows"] = xl.h2d_stream((3, n) if shaped else (n,), xl.int32, f"rows_{n}")
            entry["logits"] = xl.d2h_stream((n, self.model.vocab), xl.float32, f"logits_{n}")
            rows = ops.host_load(entry["rows"])
            logits = self.model.logits(t, self.model.select(t, rows[0] if shaped else rows))
            ops.host_store(entry["logits"], ops.shape_logits(logits, rows[1], rows[2], self._rules(t)) if shaped else logits)

        return self._program(("logits", n, "shaped") if shaped else ("logits", n), build)

    # -- steps -----------------------------------------------------------------------------------------------------------
    def _run_portion(self, part: Mapping[int, Sequence[int]], sample: bool = False) -> int:
        """`part`: slot -> its next tokens (at most `max_portion`). Returns the rows per sequence of the program."""
        T = portion_size(max(len(v) for v in part.values()))
        entry = self._portion_program(T, sample)
        tokens = np.zeros((self.batch, T), np.int32)
        ctrl = np.zeros((2, self.batch), np.int32)
        ctrl[0] = self.lengths
        for slot, toks in part.items():
            tokens[slot, :len(toks)] = toks
            ctrl[1, slot] = len(toks)
        self.session.run_program(entry["program"], {self._ctrl_in: ctrl, entry["tokens"]: tokens.reshape(-1)}, fetch=False)
        for slot, toks in part.items():
            self.lengths[slot] += len(toks)
        return T

    def _read_logits(self, rows: Sequence[tuple], shaped: bool = False) -> np.ndarray:
        """`rows`: (row of the stream, slot, tokens up to and with it)."""
        n = portion_size(len(rows))
        entry = self._logits_program(n, shaped)
        padded = np.zeros((3, n), np.int32)
        padded[:, :len(rows)] = np.array(rows, np.int32).T
        out = self.session.run_program(entry["program"], {entry["rows"]: padded if shaped else padded[0]})[entry["logits"]]
        return np.asarray(out).reshape(n, -1)[:len(rows)]

    def step(self, entries: Mapping[object, Sequence[int]], want: Optional[Mapping[object, Sequence[int]]] = None,
             shaped: bool = False) -> Dict[object, np.ndarray]:
        """Advance live requests by their next tokens. `want[request]`: places among these tokens whose logits are returned,
        `{request: (len(want), vocab) float32}` in the given order; `shaped`: as the requests' `LogitShaping` leaves them after the
        tokens up to each place."""
        if shaped and not self.shaping:
            raise ValueError("this program was made without shaping=True")
        want = {r: list(w) for r, w in (want or {}).items() if len(w)}
        todo = {}
        for req, toks in entries.items():
            slot, n = self.slots[req], len(toks)
            if self.lengths[slot] + n > self.max_seq:
                raise ValueError(f"request {req!r} would hold {self.lengths[slot] + n} positions, a slot has {self.max_seq}")
            if n and not (0 <= min(toks) and max(toks) < self.model.vocab):
                raise ValueError(f"request {req!r} has a token outside the vocabulary of {self.model.vocab}")
            if any(not 0 <= w < n for w in want.get(req, ())):
                raise ValueError(f"request {req!r} asks for logits outside its {n} tokens")
            if n:
                todo[req] = list(toks)
        out = {r: np.empty((len(w), self.model.vocab), np.float32) for r, w in want.items()}
        done, before = 0, {r: self.lengths[self.slots[r]] for r in todo}
        while todo:
            part = {self.slots[r]: toks[done:done + self.max_portion] for r, toks in todo.items()}
            T = self._run_portion(part)
            picks = [(r, k, (self.slots[r] * T + w - done, self.slots[r], before[r] + w + 1)) for r in todo
                     for k, w in enumerate(want.get(r, ())) if done <= w < done + self.max_portion]
            if picks:
                for (r, k, _), row in zip(picks, self._read_logits([row for _, _, row in picks], shaped)):
                    out[r][k] = row
            done += self.max_portion
            todo = {r: toks for r, toks in todo.items() if len(toks) > done}
        return out

    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int,
                 shaping: Union[None, LogitShaping, Sequence[Optional[LogitShaping]]] = None,
                 adapters: Optional[Sequence[Optional[int]]] = None) -> List[np.ndarray]:
        """Greedy continuation of every prompt; prompts beyond the number of slots run in further batches. `shaping`: one for all
        prompts or one for each; `adapters`: the adapter of every prompt."""
        if max_new_tokens < 1 or max_new_tokens > self.max_new:
            raise ValueError(f"max_new_tokens must be in [1, {self.max_new}]")
        if self.slots:
            raise RuntimeError("generate() needs all slots: release the live requests first")
        shaping = [shaping] * len(prompts) if shaping is None or isinstance(shaping, LogitShaping) else list(shaping)
        adapters = [None] * len(prompts) if adapters is None else list(adapters)
        if not len(shaping) == len(adapters) == len(prompts):
            raise ValueError(f"{len(prompts)} prompts need as many shapings and adapters")
        out: List[np.ndarray] = []
        for lo in range(0, len(prompts), self.batch):
            hi = lo + self.batch
            out += self._generate_batch(prompts[lo:hi], max_new_tokens, shaping[lo:hi], adapters[lo:hi])
        return out

    def _generate_batch(self, prompts, n_new: int, shaping, adapters) -> List[np.ndarray]:
        if any(len(p) < 1 or len(p) + n_new - 1 > self.max_seq for p in prompts):
            raise ValueError(f"prompts must hold between 1 and {self.max_seq - n_new + 1} tokens")
        reqs, slot = list(range(len(prompts))), {}
        try:
            for r in reqs:
                slot[r] = self.admit(r, adapters[r], shaping[r], len(prompts[r]))
            # all but the last portion of every prompt, then the last ones together: they end in the first sampled token
            last = {r: prompts[r][(len(prompts[r]) - 1) // self.max_portion * self.max_portion:] for r in reqs}
            head = {r: prompts[r][:len(prompts[r]) - len(last[r])] for r in reqs}
            self.step({r: h for r, h in head.items() if len(h)})
            self._set_device("step", 0)
            self.session.record_timestamp("start")
            self._run_portion({slot[r]: last[r] for r in reqs}, sample=True)
            self.session.record_timestamp("prefill_done")
            self._set_device("count", [1 if s in slot.values() else 0 for s in range(self.batch)])
            decode = self._decode_program()["program"]
            for _ in range(n_new - 1):
                self.session.run_program(decode, fetch=False)
            self.session.record_timestamp("decode_done")
            got = self.session.get_tensor_data(self._vars["generated"])
            if self.session.use_native:
                from ..ops import native

                native.check_gemm_errors()
        finally:
            for r in slot:
                self.release(r)
        return [np.array(got[:n_new, slot[r]], np.int32) for r in reqs]

    def _set_device(self, name: str, value):
        v = self.session._vars[self._vars[name]][0]
        v.copy_(torch.as_tensor(value, dtype=v.dtype).reshape(-1).expand_as(v))

    def decode_ms(self) -> float:
        return self.session.elapsed_ms("prefill_done", "decode_done")

    def prefill_ms(self) -> float:
        return self.session.elapsed_ms("start", "prefill_done")
