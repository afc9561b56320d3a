export distill!, distill, ∇distill!, ∇distill, distill_with_grad!

# No counterpart in the reference.  `teacher (K,N)` Float32 and `index (K,N)` Int32 (0-based ids) hold a teacher's K entries per row.

allocate_checkpoints(::typeof(distill!), X) = allocate_checkpoints(token_logprobs!, X)

function require_teacher(X, teacher, index)
    require_row_array(teacher, Float32, size(teacher, 1), size(X, 2))
    require_row_array(index, Int32, size(teacher, 1), size(X, 2))
end

"""
    distill!(loss, X, teacher, index; temperature = 1, teacher_temperature = temperature, renormalize = true, checkpoints = nothing) -> loss

`loss (N,) = Σₖ Pₖ (log Pₖ − log softmax(X / temperature)[indexₖ])`.  With `renormalize`, `P` is the softmax of
`teacher / teacher_temperature` over the row's entries, otherwise its exponential as it is.  The alternatives of `token_logprobs!`
already have their temperature in them: they go with `teacher_temperature = 1`.  Entries with an id outside `0:M-1` are left out.
The teacher's entries are constants: no gradient runs into them.
"""
function distill!(loss, X, teacher, index; temperature = 1, teacher_temperature = temperature, renormalize = true, checkpoints = nothing)
    px, pl = primal(X), primal(loss)
    M, N = size(px)
    cm, cl = checkpoints === nothing ? (nothing, nothing) : (checkpoints.M, checkpoints.L)
    foreach(a -> require_row_array(a, Float32, N), (pl, cm, cl))
    require_teacher(px, teacher, index)
    check(ccall((:tylo_b200_distill_fwd, libtylo), Int32,
                (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Int32, Int64, Int64, Int64, Float32, Float32,
                 Int32, Int32, Ptr{Cvoid}),
                devptr(pl), devptr(cm), devptr(cl), devptr(px), devptr(teacher), devptr(index), Int32(size(teacher, 1)), M, N,
                logits_stride(px), Float32(temperature), Float32(teacher_temperature), Int32(renormalize), tylo_dtype(eltype(px)),
                current_stream()))
    return loss
end

function distill(X, teacher, index; kwargs...)
    loss = similar(X, Float32, size(X, 2))
    return distill!(loss, X, teacher, index; kwargs...)
end

"""
    ∇distill!(loss, X, teacher, index; checkpoints, temperature, teacher_temperature, renormalize)

Overwrites `X.shadow` with the gradient of `sum(loss .* loss.shadow)`; `checkpoints` are the forward's.  `X.shadow` has the row stride
of `X` and may be `X` itself.  The teacher's entries are constants.  Returns `nothing`.
"""
function ∇distill!(loss::Duplicated, X::Duplicated, teacher, index; checkpoints, temperature = 1, teacher_temperature = temperature,
                   renormalize = true)
    px = primal(X)
    M, N = size(px)
    require_logits_grad(px, shadow(X))
    foreach(a -> require_row_array(a, Float32, N), (shadow(loss), checkpoints.M, checkpoints.L))
    require_teacher(px, teacher, index)
    check(ccall((:tylo_b200_distill_bwd, libtylo), Int32,
                (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Int32, Int64, Int64, Int64, Float32,
                 Float32, Int32, Int32, Ptr{Cvoid}),
                devptr(shadow(X)), devptr(shadow(loss)), devptr(px), devptr(teacher), devptr(index), devptr(checkpoints.M),
                devptr(checkpoints.L), Int32(size(teacher, 1)), M, N, logits_stride(px), Float32(temperature),
                Float32(teacher_temperature), Int32(renormalize), tylo_dtype(eltype(px)), current_stream()))
    return
end

function ∇distill(loss̄, X, teacher, index; kwargs...)
    Xd = Duplicated(X, like_logits(X))
    ∇distill!(Duplicated(loss̄, loss̄), Xd, teacher, index; kwargs...)
    return shadow(Xd)
end

"`distill!` and `∇distill!` in one launch, for weights (`loss.shadow`) that are known before the forward.  Returns `nothing`."
function distill_with_grad!(loss::Duplicated, X::Duplicated, teacher, index; temperature = 1, teacher_temperature = temperature,
                            renormalize = true)
    px = primal(X)
    M, N = size(px)
    require_logits_grad(px, shadow(X))
    foreach(a -> require_row_array(a, Float32, N), (primal(loss), shadow(loss)))
    require_teacher(px, teacher, index)
    check(ccall((:tylo_b200_distill_fwd_bwd, libtylo), Int32,
                (Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Ptr{Cvoid}, Int32, Int64, Int64, Int64, Float32, Float32,
                 Int32, Int32, Ptr{Cvoid}),
                devptr(primal(loss)), devptr(shadow(X)), devptr(shadow(loss)), devptr(px), devptr(teacher), devptr(index),
                Int32(size(teacher, 1)), M, N, logits_stride(px), Float32(temperature), Float32(teacher_temperature),
                Int32(renormalize), tylo_dtype(eltype(px)), current_stream()))
    return
end
