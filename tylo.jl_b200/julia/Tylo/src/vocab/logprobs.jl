export token_logprobs!, token_logprobs, ∇token_logprobs!, ∇token_logprobs, token_logprobs_with_grad!, allocate_top

# No counterpart in the reference: what a model's logits are turned into, beside `softmax!`.
# Token ids are 0-based `Int32`; an id outside `0:M-1` stands for "no token" (padding).

"Elements between the rows (columns in Julia's order) of logits `X (M,N)`, which may be a view of a wider buffer."
function logits_stride(X)
    M, N = size(X)
    ld = N == 1 ? max(stride(X, 2), M) : stride(X, 2)
    (stride(X, 1) == 1 && ld >= M) || throw(ArgumentError("rows of logits must be contiguous and must not overlap"))
    return ld
end

"Checks that the gradient has the size, element type and row stride of the logits (it may be the same memory)."
function require_logits_grad(X, X̄)
    (size(X) == size(X̄) && eltype(X) === eltype(X̄) && logits_stride(X) == logits_stride(X̄)) ||
        throw(ArgumentError("the gradient must have the size, element type and row stride of the logits"))
end

"An uninitialised gradient of `X` with its row stride."
like_logits(X) = view(similar(X, logits_stride(X), size(X, 2)), 1:size(X, 1), :)

function require_row_array(a, T, dims...)
    a === nothing && return
    @assert size(a) == dims
    eltype(a) === T || throw(ArgumentError("expected elements of type $T, got $(eltype(a))"))
    require_dense(a)
end

allocate_checkpoints(::typeof(token_logprobs!), X) = (; M = similar(X, Float32, size(X, 2)), L = similar(X, Float32, size(X, 2)))

"Buffers of the `K` largest alternatives of every row of `X`: `(; logp, index)`."
allocate_top(X, K) = (; logp = similar(X, Float32, K, size(X, 2)), index = similar(X, Int32, K, size(X, 2)))

"""
    token_logprobs!(logp, X, targets; temperature = 1, entropy = nothing, top = nothing, checkpoints = nothing) -> logp

Log probabilities of `targets (N,)` under `softmax(X / temperature)` per column of `X (M,N)`, and, where a buffer is given, the
`entropy (N,)` and the largest alternatives `top = allocate_top(X, K)`.  `logp` and `targets` may both be `nothing`.  The alternatives
are a report: no gradient runs through them, and the rule of `token_logprobs` refuses a cotangent of theirs.
"""
function token_logprobs!(logp, X, targets; temperature = 1, entropy = nothing, top = nothing, checkpoints = nothing)
    px, pl, pe = primal(X), primal(logp), primal(entropy)
    M, N = size(px)
    ld = logits_stride(px)
    K = top === nothing ? 0 : size(top.logp, 1)
    tl, ti = K == 0 ? (nothing, nothing) : (top.logp, top.index)
    cm, cl = checkpoints === nothing ? (nothing, nothing) : (checkpoints.M, checkpoints.L)
    foreach(a -> require_row_array(a, Float32, N), (pl, pe, cm, cl))
    require_row_array(targets, Int32, N)
    require_row_array(tl, Float32, K, N)
    require_row_array(ti, Int32, K, N)
    check(ccall((:tylo_b200_token_logprobs_fwd, libtylo), Int32,
                (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Int32, Int64, Int64,
                 Int64, Float32, Int32, Ptr{Cvoid}),
                devptr(pl), devptr(pe), devptr(tl), devptr(ti), devptr(cm), devptr(cl), devptr(px), devptr(targets), Int32(K), M, N, ld,
                Float32(temperature), tylo_dtype(eltype(px)), current_stream()))
    return logp
end

function token_logprobs(X, targets = nothing; temperature = 1, entropy = false, top = 0, checkpoints = nothing)
    N = size(X, 2)
    logp = targets === nothing ? nothing : similar(X, Float32, N)
    H = entropy ? similar(X, Float32, N) : nothing
    alternatives = top > 0 ? allocate_top(X, top) : nothing
    token_logprobs!(logp, X, targets; temperature, entropy = H, top = alternatives, checkpoints)
    return (; logp, entropy = H, top = alternatives)
end

weights(d) = d === nothing ? nothing : shadow(d)

"""
    ∇token_logprobs!(logp, X, targets; checkpoints, entropy = nothing, temperature = 1)

Overwrites `X.shadow` with the gradient of `sum(logp .* logp.shadow) + sum(entropy .* entropy.shadow)`; `entropy.primal` and
`checkpoints` are the forward's.  `X.shadow` has the row stride of `X` and may be `X` itself.  Returns `nothing`.
"""
function ∇token_logprobs!(logp, X::Duplicated, targets; checkpoints, entropy = nothing, temperature = 1)
    px, l̄, ē = primal(X), weights(logp), weights(entropy)
    M, N = size(px)
    require_logits_grad(px, shadow(X))
    foreach(a -> require_row_array(a, Float32, N), (l̄, ē, primal(entropy), checkpoints.M, checkpoints.L))
    require_row_array(targets, Int32, N)
    check(ccall((:tylo_b200_token_logprobs_bwd, libtylo), Int32,
                (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Int64, Int64, Int64,
                 Float32, Int32, Ptr{Cvoid}),
                devptr(shadow(X)), devptr(l̄), devptr(ē), devptr(px), devptr(targets), devptr(primal(entropy)), devptr(checkpoints.M),
                devptr(checkpoints.L), M, N, logits_stride(px), Float32(temperature), tylo_dtype(eltype(px)), current_stream()))
    return
end

function ∇token_logprobs(l̄, X, targets; checkpoints, entropy = nothing, ē = nothing, temperature = 1)
    Xd = Duplicated(X, like_logits(X))
    ∇token_logprobs!(l̄ === nothing ? nothing : Duplicated(l̄, l̄), Xd, targets; checkpoints,
                     entropy = ē === nothing ? nothing : Duplicated(entropy, ē), temperature)
    return shadow(Xd)
end

"""
    token_logprobs_with_grad!(logp, X, targets; entropy = nothing, temperature = 1)

`token_logprobs!` and `∇token_logprobs!` in one launch, for weights (`logp.shadow`, `entropy.shadow`) that are known before the
forward, as in next-token training.  Returns `nothing`.
"""
function token_logprobs_with_grad!(logp, X::Duplicated, targets; entropy = nothing, temperature = 1)
    px, l̄, ē = primal(X), weights(logp), weights(entropy)
    M, N = size(px)
    require_logits_grad(px, shadow(X))
    foreach(a -> require_row_array(a, Float32, N), (primal(logp), primal(entropy), l̄, ē))
    require_row_array(targets, Int32, N)
    check(ccall((:tylo_b200_token_logprobs_fwd_bwd, libtylo), Int32,
                (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Int64, Int64, Int64, Float32, Int32,
                 Ptr{Cvoid}),
                devptr(primal(logp)), devptr(primal(entropy)), devptr(shadow(X)), devptr(l̄), devptr(ē), devptr(px), devptr(targets), M, N,
                logits_stride(px), Float32(temperature), tylo_dtype(eltype(px)), current_stream()))
    return
end
