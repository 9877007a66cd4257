"""Per-request state that drives the index arithmetic of the KV path.

Mirrors the names and semantics of the reference's deserve_worker/task.py
(TaskData 26-65, TaskManager 68-115, SamplingParams 18-23) without its
import-time side effects (the reference switches torch's default dtype to fp16
and binds a global CUDA device when the module is imported, task.py:7-9).
"""
from __future__ import annotations

from dataclasses import dataclass, field


@dataclass
class SamplingParams:
    temperature: float = 0.0
    top_p: float = 1.0
    max_seq_len: int = 4096
    max_new_tokens: int = 4096
    dump_probs_num: int = 0


@dataclass
class TaskData:
    """start_pos = tokens already in the cache; seqlen = tokens fed this step
    (0 while a chunked prefill waits for its next chunk); initial_seqlen = prompt
    length."""

    task_id: str
    start_pos: int
    round: int
    seqlen: int
    initial_seqlen: int
    sampling_params: SamplingParams = field(default_factory=SamplingParams)

    @staticmethod
    def empty(task_id: str, initial_seqlen: int, sampling_params: SamplingParams | None = None) -> "TaskData":
        return TaskData(task_id, 0, 0, 0, initial_seqlen, sampling_params or SamplingParams())

    def init(self, seqlen: int) -> None:
        self.seqlen = seqlen

    def is_prefill(self) -> bool:
        # name kept from the reference, where it is true once the prompt is consumed
        return self.start_pos >= self.initial_seqlen

    def finished_prefill(self) -> bool:
        return self.start_pos + self.seqlen >= self.initial_seqlen

    def step(self) -> None:
        assert self.seqlen > 0
        self.start_pos += self.seqlen
        self.seqlen = 1 if self.start_pos >= self.initial_seqlen else 0
        self.round += 1

    def step_verified(self, accepted: int) -> None:
        """A speculative step is over: the last token and `accepted` of the drafts fed with it are in the cache for
        good (the next step writes over the rejected ones), and one token drawn by the target is fed next."""
        assert self.is_prefill() and 0 <= accepted < self.seqlen
        self.start_pos += accepted + 1
        self.seqlen = 1
        self.round += 1


class TaskManager:
    """Registry of TaskData plus the page arithmetic the schedulers use."""

    def __init__(self, num_pages: int, page_size: int) -> None:
        self.task_datas: dict[str, TaskData] = {}
        self.page_size = page_size

    def add(self, task_data: TaskData) -> None:
        self.task_datas[task_data.task_id] = task_data

    def get(self, task_id: str) -> TaskData:
        return self.task_datas[task_id]

    def calc_space(self, size: int) -> int:
        return -(-size // self.page_size)

    def calc_occupied_space(self, task_ids: list[str]) -> int:
        return sum(self.calc_space(self.get(t).start_pos) for t in task_ids)

    def calc_initial_space(self, task_ids: list[str]) -> int:
        return sum(self.calc_space(self.get(t).initial_seqlen) for t in task_ids)

    def calc_extended_space(self, task_ids: list[str]) -> int:
        datas = [self.get(t) for t in task_ids]
        assert all(d.seqlen > 0 for d in datas)
        return sum(self.calc_space(d.start_pos + d.seqlen) - self.calc_space(d.start_pos) for d in datas)

    def calc_seqlens(self, task_ids: list[str]) -> int:
        return sum(self.get(t).seqlen for t in task_ids)

    def calc_delta_space(self, task_id: str, seqlen: int) -> int:
        d = self.get(task_id)
        return self.calc_space(d.start_pos + seqlen) - self.calc_space(d.start_pos)

    def calc_rest_space(self, task_id: str) -> int:
        d = self.get(task_id)
        return self.calc_space(d.initial_seqlen) - self.calc_space(d.start_pos)
