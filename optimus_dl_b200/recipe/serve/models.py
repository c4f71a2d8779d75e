"""OpenAI-style request / response schemas of the serve recipe
(field names as in optimus_dl/recipe/serve/models.py:9-209)."""

from __future__ import annotations

from typing import Literal

from pydantic import BaseModel, Field, model_validator

DEFAULT_MODEL_NAME = "optimus-dl-model"


class _Sampling(BaseModel):
    model: str = DEFAULT_MODEL_NAME
    max_tokens: int = Field(default=50, ge=1)
    temperature: float = Field(default=1.0, ge=0.0)
    top_k: int | None = Field(default=None, ge=1)
    top_p: float | None = Field(default=None, gt=0.0, le=1.0)
    stream: bool = False

    def alternatives(self) -> int | None:
        """Alternatives per token that the answer lists, None without log probabilities."""
        raise NotImplementedError


class ChatCompletionRequest(_Sampling):
    """Clients send ``logprobs`` as null and with streams as well: a stream is answered, without log probabilities."""

    messages: list[dict]
    logprobs: bool | None = None
    top_logprobs: int | None = Field(default=None, ge=0, le=20)

    def alternatives(self) -> int | None:
        return (self.top_logprobs or 0) if self.logprobs and not self.stream else None


class CompletionRequest(_Sampling):
    prompt: str | list[str]
    logprobs: int | None = Field(default=None, ge=0, le=20)

    def alternatives(self) -> int | None:
        return self.logprobs

    @model_validator(mode="after")
    def _no_streamed_logprobs(self):
        if self.stream and self.logprobs is not None:
            raise ValueError("log probabilities are not streamed: use stream=false")
        return self


class ChatMessage(BaseModel):
    role: str | None = None
    content: str | None = None


class Choice(BaseModel):
    index: int
    text: str
    logprobs: dict | None = None
    finish_reason: str | None = None


class CompletionResponse(BaseModel):
    id: str
    object: Literal["text_completion"]
    created: int
    model: str
    choices: list[Choice]
    usage: dict | None = None


class ChatChoice(BaseModel):
    index: int
    message: ChatMessage
    logprobs: dict | None = None
    finish_reason: str | None = None


class ChatCompletionResponse(BaseModel):
    id: str
    object: Literal["chat.completion"]
    created: int
    model: str
    choices: list[ChatChoice]
    usage: dict | None = None


class Delta(BaseModel):
    role: str | None = None
    content: str | None = None


class ChatChunkChoice(BaseModel):
    index: int
    delta: Delta
    finish_reason: str | None = None


class ChatCompletionChunk(BaseModel):
    id: str
    object: Literal["chat.completion.chunk"]
    created: int
    model: str
    choices: list[ChatChunkChoice]


class CompletionChunkChoice(BaseModel):
    index: int
    text: str
    logprobs: dict | None = None
    finish_reason: str | None = None


class CompletionChunk(BaseModel):
    id: str
    object: Literal["text_completion"]
    created: int
    model: str
    choices: list[CompletionChunkChoice]
